// Teams of lanes on the columns of a matrix: sums over a team, and columns as 16-byte groups at any 4-byte boundary.
#pragma once
#include "common.h"

// Sums or maxima over the 16 lanes of a row, or over a wavefront, by the cross-lane paths of the vector unit (a shuffle through LDS takes
// some 60 cycles a step, these 8).  Every lane gets the same bits: each step combines the same two numbers on both sides.
template <int CTRL>
__device__ __forceinline__ float lane_move(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
template <int T, bool MAX = false>
__device__ __forceinline__ float lanes_sum(float v) {
  static_assert(T == 16 || T == 64, "a row or a wavefront");
  auto both = [](float a, float b) __attribute__((always_inline)) { return MAX ? fmaxf(a, b) : a + b; };
  v = both(v, lane_move<0xB1>(v));         // neighbours
  v = both(v, lane_move<0x4E>(v));         // pairs
  v = both(v, lane_move<0x141>(v));        // halves of a row, mirrored
  v = both(v, lane_move<0x140>(v));        // the row, mirrored
  if (T == 64) {                           // the four rows' results, as scalars (the whole wavefront is here)
    const int x = __builtin_bit_cast(int, v);
    auto row = [&](int l) __attribute__((always_inline)) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(x, l)); };
    v = both(both(row(0), row(16)), both(row(32), row(48)));
  }
  return v;
}

// A column of h >= 4 floats as groups of four: group j starts at row 4 j, the last one at h - 4; the rows that it has in common with the
// one before (`lap`, only where h is no multiple of 4) are that one's.  Loads are never behind a branch (a lane without a group reads the last
// one): with them the compiler could not count what is on its way, and would wait for all of it.
// STREAM: non-temporal accesses, for what is touched once.
typedef float ColGroup __attribute__((ext_vector_type(4), aligned(4)));
template <bool STREAM>
__device__ __forceinline__ void col_load(float (&v)[4], const float* p) {
  const ColGroup* g = reinterpret_cast<const ColGroup*>(p);
  const ColGroup q = STREAM ? __builtin_nontemporal_load(g) : *g;
  v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
}
template <bool STREAM>
__device__ __forceinline__ void col_store(float* p, const float (&v)[4]) {
  ColGroup* g = reinterpret_cast<ColGroup*>(p);
  const ColGroup q = {v[0], v[1], v[2], v[3]};
  if (STREAM) __builtin_nontemporal_store(q, g);
  else *g = q;
}
template <int NV, bool TAIL>
struct ColGroups {
  int row[NV];                  // first row of a lane's group; of lanes that have none, the last group's
  bool in[NV];                  // whether it has one
  int lap;                      // rows of the last group that are its neighbour's, for the lane that has it (TAIL)
  int last;                     // which of its groups that is, or -1
  __device__ __forceinline__ void init(int lane, int T, int h) {
    lap = 0; last = -1;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int r = 4 * (lane + k * T);
      in[k] = r < h;
      row[k] = r + 4 <= h ? r : h - 4;
      if (TAIL && r < h && r + 4 > h) { lap = r - (h - 4); last = k; }
    }
  }
  __device__ __forceinline__ bool own(int k, int e) const { return in[k] && (!TAIL || k != last || e >= lap); }
};
// Stores a lane's group k.  OWN: without the rows that are its neighbour's, where two wavefronts may come to different roundings of them.
template <bool STREAM, bool OWN, int NV, bool TAIL>
__device__ __forceinline__ void col_store_group(const ColGroups<NV, TAIL>& at, int k, float* column, const float (&v)[4]) {
  if (!OWN || !TAIL || k != at.last) { col_store<STREAM>(column + at.row[k], v); return; }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e >= at.lap) column[at.row[k] + e] = v[e];
}
