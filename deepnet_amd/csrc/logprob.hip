// Log probabilities of given tokens, entropies and the best alternatives of columns of logits, and their gradient (no
// counterpart in cudamat.cu; softmax_ce_grad is the loss of a classifier, which stores its probabilities).
#include "columns.h"
#include "wide_math.h"
#include <float.h>

// Orders entries: the greater value first, of equal ones (0 and -0 are) the one further up; NaN ranks with -inf.
__device__ __forceinline__ unsigned long long lp_key(float x, int i) {
  x = x != x ? -INFINITY : x + 0.f;
  const unsigned u = __float_as_uint(x), v = u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
  return ((unsigned long long)v << 32) | (unsigned)~i;
}
__device__ __forceinline__ int lp_key_index(unsigned long long k) { return (int)~(unsigned)k; }
__device__ __forceinline__ float lp_key_value(unsigned long long key) {
  const unsigned v = (unsigned)(key >> 32);
  return __uint_as_float(v ^ ((v >> 31) ? 0x80000000u : 0xffffffffu));
}

// log(1 + r), r >= 0 (NaN stays NaN); 1 + r itself would round a small r away.
__device__ __forceinline__ double lp_log1p(double u) {
  return u >= 1e-5 ? dn_log_wide_pos(1.0 + u) : u * fma(u, fma(u, 1.0 / 3.0, -0.5), 1.0);
}

struct LogProbArgs {
  const float *mat, *labels;
  float *logp, *entropy, *log_z, *top, *top_labels;
  int h, w, k;
  int segments, length;            // of a column: LogProbPart's and k keys of each in `parts` and `keys`
  float* parts;
  unsigned long long* keys;
  unsigned* arrived;
};

// What one pass over some entries keeps: their maximum m (at least the lowest finite number), how many are equal to it, and over the
// others r, the sum of e^(x - m), and t, that of (x - m) e^(x - m).  So log(sum of exponentials) = m + log(1 + (count - 1 + r)), to full
// precision however small r is beside the maximum's own 1, and entropy = log(1 + ..) - t / (1 + ..).  Entries of -inf count nothing: a
// column of nothing else has count 0.  NaN and +inf make r NaN.
struct LogProbPart { float m; int count; float r, t; };
__device__ __forceinline__ LogProbPart lp_none() { return LogProbPart{-FLT_MAX, 0, 0.f, 0.f}; }
// e^d, d <= 0, by the hardware's exp2.  d is off by half a step already, which changes the result by u |d| of it (u = 2^-24); the product's
// rounding is as much again, and the constant is off by 0.22 u of it.
__device__ __forceinline__ float lp_exp_fast(float d) { return __builtin_amdgcn_exp2f(d * 1.44269502162933349609375f); }
// The part as seen from a maximum M >= m.
__device__ __forceinline__ void lp_raise(LogProbPart& p, float M) {
  if (M > p.m) {
    const float d = p.m - M, s = lp_exp_fast(d), all = p.r + (float)p.count;
    p.t = s * __fmaf_rn(fmaxf(d, -200.f), all, p.t);
    p.r = s * all;
    p.count = 0;
    p.m = M;
  }
}
__device__ __forceinline__ void lp_take(LogProbPart& p, float x) {
  const float d = x - p.m, e = lp_exp_fast(d);
  p.count += d == 0.f ? 1 : 0;
  p.r += d == 0.f ? 0.f : e;
  p.t = __fmaf_rn(fmaxf(d, -200.f), e, p.t);               // (-inf: e is 0; what is kept of d does not matter below -200)
}
// Over the 64 lanes of a wavefront; every lane gets it.
__device__ __forceinline__ LogProbPart lp_wave(LogProbPart p) {
  lp_raise(p, lanes_sum<64, true>(p.m));
  return LogProbPart{p.m, (int)lanes_sum<64>((float)p.count), lanes_sum<64>(p.r), lanes_sum<64>(p.t)};
}

struct LogProbResult { float m, log_z; double lz; bool none; };
__device__ __forceinline__ LogProbResult lp_result(const LogProbPart& p) {
  LogProbResult o;
  o.m = p.m;
  o.none = p.count == 0 && p.r == 0.f;
  o.lz = lp_log1p((double)(p.count - 1) + (double)p.r);
  o.log_z = o.none ? -INFINITY : p.r == p.r ? (float)((double)p.m + o.lz) : NAN;
  return o;
}
__device__ __forceinline__ float lp_of(const LogProbResult& o, float x) {
  return o.none ? -INFINITY : o.log_z != o.log_z ? NAN : (float)((double)x - (double)o.m - o.lz);
}
// The given token's entry, asked for before everything else: 0 for no token.
struct LogProbLabel { float x; bool token; };
__device__ __forceinline__ LogProbLabel lp_label(const LogProbArgs& a, int col) {
  LogProbLabel o = {0.f, false};
  if (a.logp) {
    const float l = a.labels[col];
    o.token = l >= 0.f && l < (float)a.h;
    if (o.token) o.x = a.mat[(size_t)col * a.h + (int)l];
  }
  return o;
}
// The results of a column but for the top list, by one lane.
__device__ __forceinline__ void lp_finish(const LogProbArgs& a, int col, const LogProbPart& p, const LogProbResult& o, const LogProbLabel& l) {
  if (a.log_z) a.log_z[col] = o.log_z;
  if (a.entropy) a.entropy[col] = o.none ? 0.f : o.log_z != o.log_z ? NAN : (float)(o.lz - (double)p.t / ((double)p.count + (double)p.r));
  if (a.logp) a.logp[col] = l.token ? lp_of(o, l.x) : 0.f;
}
__device__ __forceinline__ void lp_top_out(const LogProbArgs& a, int col, int rank, unsigned long long key, const LogProbResult& o) {
  if (a.top) a.top[(size_t)col * a.k + rank] = lp_of(o, lp_key_value(key));
  if (a.top_labels) a.top_labels[(size_t)col * a.k + rank] = (float)lp_key_index(key);
}
// How many of n keys in LDS (n even, 16-byte aligned) are greater.
__device__ __forceinline__ int lp_rank(unsigned long long key, const unsigned long long* keys, int n) {
  int r = 0;
#pragma unroll 4
  for (int i = 0; i < n; i += 2) {
    const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(keys + i);
    r += (q.x > key ? 1 : 0) + (q.y > key ? 1 : 0);
  }
  return r;
}

template <int CTRL>
__device__ __forceinline__ int lane_move_int(int v) { return __builtin_amdgcn_mov_dpp(v, CTRL, 0xf, 0xf, true); }
__device__ __forceinline__ int lp_quad_sum(int v) { v += lane_move_int<0xB1>(v); return v + lane_move_int<0x4E>(v); }
// How many of 64 values in LDS are greater than that of a quad of lanes, and how many are at least as great; each lane looks at 16.
__device__ __forceinline__ void lp_standing(unsigned value, const unsigned* values, int lane, int& greater, int& least) {
  int g = 0, l = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint4 q = *reinterpret_cast<const uint4*>(values + 16 * i + 4 * (lane & 3));
    g += (q.x > value ? 1 : 0) + (q.y > value ? 1 : 0) + (q.z > value ? 1 : 0) + (q.w > value ? 1 : 0);
    l += (q.x >= value ? 1 : 0) + (q.y >= value ? 1 : 0) + (q.z >= value ? 1 : 0) + (q.w >= value ? 1 : 0);
  }
  greater = lp_quad_sum(g);
  least = lp_quad_sum(l);
}
// Element i of 16.
__device__ __forceinline__ float lp_pick(const float (&x)[4][4], int i) {
  float a[8], b[4];
#pragma unroll
  for (int q = 0; q < 8; ++q) a[q] = i & 8 ? x[2 + q / 4][q % 4] : x[q / 4][q % 4];
#pragma unroll
  for (int q = 0; q < 4; ++q) b[q] = i & 4 ? a[4 + q] : a[q];
  const float c0 = i & 2 ? b[2] : b[0], c1 = i & 2 ? b[3] : b[1];
  return i & 1 ? c1 : c0;
}
// The greatest of the four of a quad.
__device__ __forceinline__ unsigned lp_quad_max(unsigned v) {
  const unsigned a = (unsigned)lane_move_int<0xB1>((int)v);
  v = a > v ? a : v;
  const unsigned b = (unsigned)lane_move_int<0x4E>((int)v);
  return b > v ? b : v;
}
// The k-th greatest of a wavefront's values (which has as many), bit by bit: the greatest number that k of them reach.
__device__ __forceinline__ unsigned lp_kth(unsigned value, int k) {
  unsigned r = 0;
#pragma unroll 4
  for (int b = 31; b >= 0; --b) {
    const unsigned t = r | 1u << b;
    if (__popcll(__ballot(value >= t)) >= k) r = t;
  }
  return r;
}
// Lanes before this one that are in the mask.
__device__ __forceinline__ int lp_before(unsigned long long mask) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0));
}
// The places of the `count` keys of a list (two zeros behind them): out(place, key) of the first k.  Four lanes share a key, `lanes` are here.
template <typename F>
__device__ __forceinline__ void lp_places(const unsigned long long* list, int count, int k, int lane, int lanes, F out) {
  for (int i0 = 0; i0 < count; i0 += lanes / 4) {
    const int i = i0 + lane / 4;
    const unsigned long long key = i < count ? list[i] : ~0ull;
    int r = 0;
#pragma unroll 4
    for (int j = 2 * (lane % 4); j < count; j += 8) {
      const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(list + j);
      r += (q.x > key ? 1 : 0) + (q.y > key ? 1 : 0);
    }
    r = lp_quad_sum(r);
    if (lane % 4 == 0 && i < count && r < k) out(r, key);
  }
}
// Upper halves of keys: the values' order; 0 is below all of them.
__device__ __forceinline__ unsigned lp_order(float x) { return (unsigned)(lp_key(x, 0) >> 32); }

// The top list of a team.  At least k entries reach the k-th of the maxima that 64 quads of lanes have of their own entries, and those that do
// lie in lanes whose own maximum does: these are the candidates, k and a few more (unless a few lanes have far more than their
// share), and a candidate's place is the number of greater ones.  Maxima are compared by value; where the k-th and the next one are alike
// (a mask, a constant column), by their places too, lane by lane.
#define LP_LIST 2048               // candidates that a workgroup holds

// ---- columns (or segments of them) by a workgroup of 256 lanes, eight 16-byte groups a lane on their way
// Bound by the bytes, 4 an entry: 32768 x 2048 41.8 to 42.2 us, 6.4 TB/s (copy rate: 41.6), 32003 x 2048 43.2; the exponentials take 0.8 of the
// vector unit's time.  Few columns are split, so that the chip reads them at once: 50000 x 4 in 52 workgroups 4.8 us.
// Columns of one to three rows come here too, a workgroup each: 3 x 1000000 1177 us.  Top lists are found in
// the same pass, after it: 32000 x 1024 with 20 best 38.2 us (20.3 by the bytes), 50000 x 4 10.0, a chain of some ten trips to LDS and three to
// memory, whose steps take 0.4 to 1.4 us each.
template <bool TOP, bool STREAM>
__global__ void __launch_bounds__(256) k_log_probs(LogProbArgs a) {
  __shared__ LogProbPart parts[4];
  __shared__ __attribute__((aligned(16))) unsigned long long lane_keys[TOP ? 256 : 2], list[TOP ? LP_LIST + 2 : 2];
  __shared__ int winners[TOP ? 256 : 1], wave_won[4], wave_like[4], won, listed, last;
  __shared__ unsigned least_order;
  __shared__ unsigned long long border_key;
  unsigned* const orders = reinterpret_cast<unsigned*>(lane_keys);
  const int tid = threadIdx.x, col = blockIdx.x / a.segments, seg = blockIdx.x - col * a.segments;
  const int row0 = seg * a.length, n = a.h - row0 < a.length ? a.h - row0 : a.length, n4 = n >> 2, trips = (n4 + 1023) >> 10;
  const float* c = a.mat + (size_t)col * a.h + row0;
  const LogProbLabel label = lp_label(a, col);
  LogProbPart p = lp_none();
  float best = -INFINITY;
  int best_at = 0;
  const int full = n4 >> 10;               // trips that every lane has four groups of: their loads are behind no branch, so that they can be counted
  auto load = [&](float (&v)[4][4], int it) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 4; ++u) col_load<STREAM>(v[u], c + 4 * (tid + 256 * u + 1024 * it));
  };
  auto take = [&](const float (&v)[4][4], int it) __attribute__((always_inline)) {
    float m = v[0][0];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) m = fmaxf(m, v[u][e]);
    if (TOP && m > best) { best = m; best_at = it; }
    lp_raise(p, m);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) lp_take(p, v[u][e]);
  };
  // two trips are on their way in turn
  float v[4][4], next[4][4];
  if (TOP && tid == 0) listed = won = 0;
  if (full > 0) load(v, 0);
  int it = 0;
  for (; it + 2 < full; it += 2) {
    load(next, it + 1);
    take(v, it);
    load(v, it + 2);
    take(next, it + 1);
  }
  if (it + 1 < full) {
    load(next, it + 1);
    take(v, it);
    take(next, it + 1);
  } else if (it < full) {
    take(v, it);
  }
  if (trips > full || TOP) {
    // the last one, which some lanes have fewer groups of (or, for the top list of a column of whole trips, the one that was taken last)
    const int at = trips > full ? full : full - 1;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int j = tid + 256 * u + 1024 * at;
      v[u][0] = v[u][1] = v[u][2] = v[u][3] = -INFINITY;
      if (at >= 0 && j < n4) col_load<false>(v[u], c + 4 * j);
    }
    if (trips > full) take(v, at);
  }
  const bool tail = tid < (n & 3);                         // the rows behind the last group: one a lane
  float tail_x = 0.f;
  if (tail) {
    tail_x = c[4 * n4 + tid];
    lp_raise(p, tail_x);
    lp_take(p, tail_x);
  }
  const unsigned long long tail_key = TOP && tail ? lp_key(tail_x, row0 + 4 * n4 + tid) : 0;
  p = lp_wave(p);
  if (tid % 64 == 0) parts[tid >> 6] = p;
  unsigned long long border = 1;           // candidates have keys from it on
  bool by_value = true;                    // ... which are those of values from its own on
  if (TOP) {
    const unsigned own = tid < n4 || tail ? lp_order(tail ? fmaxf(best, tail_x) : best) : 0, order = lp_quad_max(own);
    if (tid % 4 == 0) orders[tid >> 2] = order;
    __syncthreads();
    int greater, reach;
    lp_standing(order, orders, tid, greater, reach);
    if (order && greater < a.k && reach >= a.k) { least_order = order; won = reach; }      // (the k-th one, or several: they write the same)
    __syncthreads();
    border = won == a.k ? (unsigned long long)least_order << 32 : 1;
    bool in = own >= (unsigned)(border >> 32) && own;
    if (won > a.k) {
      // Several are alike at the border: now lane by lane, and of those alike the first places.
      unsigned* const lanes = orders + 64;
      auto standing = [&](unsigned value, int& greater, int& reach) __attribute__((always_inline)) {
        lanes[tid] = value;
        __syncthreads();
        greater = reach = 0;
#pragma unroll 4
        for (int i = 0; i < 256; i += 4) {
          const uint4 q = *reinterpret_cast<const uint4*>(lanes + i);
          greater += (q.x > value ? 1 : 0) + (q.y > value ? 1 : 0) + (q.z > value ? 1 : 0) + (q.w > value ? 1 : 0);
          reach += (q.x >= value ? 1 : 0) + (q.y >= value ? 1 : 0) + (q.z >= value ? 1 : 0) + (q.w >= value ? 1 : 0);
        }
        __syncthreads();
      };
      // (a masked stretch: of lanes that have nothing else than -inf, the first place is in the order of the lanes, so counting is enough)
      const bool nothing = least_order == lp_order(-INFINITY);
      const unsigned long long above = __ballot(own > least_order), alike = __ballot(own == least_order);
      if (tid % 64 == 0) { wave_won[tid >> 6] = __popcll(above); wave_like[tid >> 6] = __popcll(alike); }
      __syncthreads();
      const int over = wave_won[0] + wave_won[1] + wave_won[2] + wave_won[3];
      if (over >= a.k) {                                   // (else the quads' border is the lanes' too)
        standing(own, greater, reach);
        if (own && greater < a.k && reach >= a.k) { least_order = own; won = reach; }
        __syncthreads();
      }
      const unsigned value = least_order;
      by_value = won == a.k;
      // this lane's greatest entry: the first that is its trip's maximum (the last trip is still in registers), of nothing but -inf and
      // NaN the first of all; or its row of the tail
      int first = tid < n4 ? 4 * tid : n;
      if (best > -INFINITY) {
#pragma unroll
        for (int u = 3; u >= 0; --u) {
          const int j = tid + 256 * u + 1024 * best_at;
          float x[4] = {v[u][0], v[u][1], v[u][2], v[u][3]};
          if (best_at != trips - 1 && j < n4) col_load<false>(x, c + 4 * j);
#pragma unroll
          for (int e = 3; e >= 0; --e) first = x[e] == best ? 4 * j + e : first;
        }
      }
      if (tail && lp_order(tail_x) == own && (first >= n || lp_order(best) != own)) first = 4 * n4 + tid;
      const unsigned place = own == value ? (unsigned)~(row0 + first) : 0;
      if (tid == 0) border_key = (unsigned long long)value << 32;
      if (nothing && over < a.k) {
        __syncthreads();
        int before = over + lp_before(alike);
        for (int i = 0; i < tid >> 6; ++i) before += wave_like[i];
        if (place && before == a.k - 1) border_key |= place;
      } else {
        // (places without their top bit, which is set in all of them: lanes above the border are above row 0's place too)
        standing(own > value ? 0xffffffffu : place & 0x7fffffffu, greater, reach);
        if (!by_value && place && greater == a.k - 1) border_key |= place;
      }
      __syncthreads();
      border = border_key;
      in = ((unsigned long long)own << 32 | place) >= border && own;
    }
    if (trips > 1) {
      const unsigned long long all = __ballot(in);
      if (tid % 64 == 0) wave_won[tid >> 6] = __popcll(all);
      __syncthreads();
      int at = lp_before(all);
      for (int i = 0; i < tid >> 6; ++i) at += wave_won[i];
      if (in) winners[at] = tid;
    }
  }
  __syncthreads();
  {
    LogProbPart q = parts[tid & 3];
    lp_raise(q, fmaxf(fmaxf(parts[0].m, parts[1].m), fmaxf(parts[2].m, parts[3].m)));
    // (four neighbours have the four parts: sums over them)
    auto four = [](float x) __attribute__((always_inline)) { x += lane_move<0xB1>(x); return x + lane_move<0x4E>(x); };
    p = LogProbPart{q.m, (int)four((float)q.count), four(q.r), four(q.t)};
  }
  if (TOP) {
    const float least = border > 1 ? lp_key_value(border) : -INFINITY;
    auto offer = [&](unsigned long long q) __attribute__((always_inline)) {
      if (q >= border) {
        const int at = atomicAdd(&listed, 1);
        if (at < LP_LIST) list[at] = q;
      }
    };
    // a lane has one or two candidates among its sixteen entries at most times: one a turn (every lane of the wavefront is here)
    auto offer16 = [&](const int (&j)[4], const float (&x)[4][4]) __attribute__((always_inline)) {
      unsigned mask = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) mask |= !(x[i >> 2][i & 3] < least) ? 1u << i : 0;
      if (!by_value) {                                     // (of the ones alike, those from the border's place on are none)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (!(x[i >> 2][i & 3] > least) && row0 + 4 * j[i >> 2] + (i & 3) > lp_key_index(border)) mask &= ~(1u << i);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) mask &= j[u] < n4 ? ~0u : ~(15u << (4 * u));
      while (__ballot(mask != 0)) {
        const int i = mask ? __builtin_ctz(mask) : 0, u = i >> 2;
        const int g = u & 2 ? (u & 1 ? j[3] : j[2]) : (u & 1 ? j[1] : j[0]);
        const unsigned long long key = mask ? lp_key(lp_pick(x, i), row0 + 4 * g + (i & 3)) : 0, in = __ballot(key >= border);
        int at = 0;
        if ((tid & 63) == 0) at = atomicAdd(&listed, __popcll(in));
        at = __builtin_amdgcn_readfirstlane(at) + lp_before(in);
        if (key >= border && at < LP_LIST) list[at] = key;
        mask &= mask - 1;
      }
    };
    if (trips <= 1) {
      const int j[4] = {tid, tid + 256, tid + 512, tid + 768};
      offer16(j, v);
    } else {
      // (the entries of those lanes come from memory, four groups a lane on their way)
      const int items = (wave_won[0] + wave_won[1] + wave_won[2] + wave_won[3]) * 4 * trips;
      for (int i0 = 0; i0 < items; i0 += 1024) {
        float x[4][4];
        int at[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int i = i0 + tid + 256 * s, q = i / (4 * trips), g = i - q * (4 * trips);
          at[s] = i < items ? winners[q] + 256 * (g & 3) + 1024 * (g >> 2) : n4;
          if (at[s] < n4) col_load<false>(x[s], c + 4 * at[s]);
          else x[s][0] = x[s][1] = x[s][2] = x[s][3] = -INFINITY;
        }
        offer16(at, x);
      }
    }
    if (tail) offer(tail_key);
    __syncthreads();
  }
  // one segment: the column's results; several: this one's part, and the last to arrive joins them
  LogProbResult o = {};
  if (a.segments == 1) {
    o = lp_result(p);
    if (tid == 0) lp_finish(a, col, p, o, label);
  }
  unsigned long long* const keys = TOP ? a.keys + (size_t)blockIdx.x * a.k : nullptr;
  auto out = [&](int rank, unsigned long long key) __attribute__((always_inline)) {
    if (a.segments == 1) lp_top_out(a, col, rank, key, o);
    else __hip_atomic_store(keys + rank, key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  if (TOP) {
    const int count = listed;
    if (count <= LP_LIST) {
      if (tid < 2) list[count + tid] = 0;
      __syncthreads();
      lp_places(list, count, a.k, tid, 256, out);
      if (a.segments > 1)
        for (int i = count + tid; i < a.k; i += 256) out(i, 0);          // (a segment of fewer than k rows)
    } else {
      // more than fit: the greatest, the next one below it, and so on, a pass each
      unsigned long long above = ~0ull;
      for (int j = 0; j < a.k; ++j) {
        unsigned long long key = 0;
        for (int i = tid; i < n; i += 256) {
          const unsigned long long q = lp_key(c[i], row0 + i);
          key = q < above && q > key ? q : key;
        }
        __syncthreads();
        lane_keys[tid] = key;
        __syncthreads();
        if (key && lp_rank(key, lane_keys, 256) == 0) { border_key = key; out(j, key); }
        __syncthreads();
        above = border_key;
      }
    }
  }
  if (a.segments == 1) return;
  if (tid < 4) {
    const float f[4] = {p.m, __builtin_bit_cast(float, p.count), p.r, p.t};
    __hip_atomic_store(a.parts + 4 * (size_t)blockIdx.x + tid, f[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __builtin_amdgcn_s_waitcnt(0);         // the stores of this wavefront have been acknowledged
  __syncthreads();
  if (tid == 0) {
    const unsigned old = __hip_atomic_fetch_add(a.arrived + col, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last = old == (unsigned)a.segments - 1u;
    if (last) __hip_atomic_store(a.arrived + col, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (TOP && tid == 0) listed = won = 0;
  __syncthreads();
  if (!last) return;
  // at most 64 segments: a lane each, in a fixed order whoever came last
  const float* f = a.parts + 4 * ((size_t)col * a.segments + (tid & 63));
  auto get = [&](int i) __attribute__((always_inline)) { return __hip_atomic_load(f + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  const int count = a.segments * a.k;                      // (at most LP_JOIN: two keys a lane)
  unsigned long long q[2] = {0, 0};
  if (TOP) {
    const unsigned long long* from = a.keys + (size_t)col * count;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (tid + 256 * i < count) q[i] = __hip_atomic_load(from + tid + 256 * i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  p = lp_none();
  if ((tid & 63) < a.segments) p = LogProbPart{get(0), __builtin_bit_cast(int, get(1)), get(2), get(3)};
  p = lp_wave(p);
  o = lp_result(p);
  if (tid == 0) lp_finish(a, col, p, o, label);
  if (TOP) {
    // candidates: keys from the k-th of 64 maxima of four lanes each on (a key has one place: none are alike, and those of equal
    // value are taken together)
    const unsigned order = lp_quad_max((unsigned)((q[0] > q[1] ? q[0] : q[1]) >> 32));
    if (tid % 4 == 0) orders[tid >> 2] = order;
    __syncthreads();
    int greater, reach;
    lp_standing(order, orders, tid, greater, reach);
    if (order && greater < a.k && reach >= a.k) { least_order = order; won = reach; }
    __syncthreads();
    const unsigned from_order = won ? least_order : 1;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const unsigned long long in = __ballot((unsigned)(q[i] >> 32) >= from_order);
      int at = 0;
      if ((tid & 63) == 0 && in) at = atomicAdd(&listed, __popcll(in));
      at = __builtin_amdgcn_readfirstlane(at) + lp_before(in);
      if (in >> (tid & 63) & 1) list[at] = q[i];
    }
    __syncthreads();
    const int found = listed;
    if (tid < 2) list[found + tid] = 0;
    __syncthreads();
    lp_places(list, found, a.k, tid, 256, [&](int place, unsigned long long key) __attribute__((always_inline)) { lp_top_out(a, col, place, key, o); });
  }
}

// ---- columns of 4 to 1024 rows (many of them: to 4095, without a top list) by a wavefront, which holds them in registers
// Bound by the bytes: 1024 x 20000 15.5 us, 5.3 TB/s (with 20 best 38.4: by the vector instructions of the list), 2050 x 8192 14.6, 256 x 80000
// 15.2, 100 x 200000 22.3; 100 x 8192 with 20 best 11.9.  The results of a column take a hundred instructions in 64 bits, which four columns share.
// T: the lanes of a column, 64 or (up to 512 rows without a top list) 16, four columns a wavefront.
template <int T, int NV, bool TAIL, bool TOP, bool STREAM>
__global__ void __launch_bounds__(256) k_log_probs_wave(LogProbArgs a) {
  static_assert(T == 64 || !TOP, "a wavefront finds a list");
  __shared__ __attribute__((aligned(16))) unsigned long long lists[TOP ? 4 : 1][TOP ? 256 * NV + 2 : 2];
  const int lane = threadIdx.x % T, wv = threadIdx.x >> 6, col = blockIdx.x * (256 / T) + threadIdx.x / T;
  const bool live = col < a.w;
  const float* c = a.mat + (size_t)(live ? col : 0) * a.h;
  const LogProbLabel label = lp_label(a, live ? col : 0);
  ColGroups<NV, TAIL> at;
  at.init(lane, T, a.h);
  float v[NV][4], m = -FLT_MAX;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    col_load<STREAM>(v[k], c + at.row[k]);
  }
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (!at.own(k, e)) v[k][e] = -INFINITY;
      m = fmaxf(m, v[k][e]);
    }
  LogProbPart p = lp_none();
  p.m = lanes_sum<T, true>(m);
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) lp_take(p, v[k][e]);
  p = LogProbPart{p.m, (int)lanes_sum<T>((float)p.count), lanes_sum<T>(p.r), lanes_sum<T>(p.t)};
  const LogProbResult o = lp_result(p);
  if (live && lane == 0) lp_finish(a, col, p, o, label);
  if (!TOP) return;
  unsigned long long best = 0;
  auto key_of = [&](int k, int e) __attribute__((always_inline)) { return at.own(k, e) ? lp_key(v[k][e], at.row[k] + e) : 0ull; };
  // the lane's greatest entry: the first that is its maximum, of nothing but -inf and NaN the first of all
  int first = -1;
  float most = -INFINITY;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) most = fmaxf(most, v[k][e]);
#pragma unroll
  for (int k = NV - 1; k >= 0; --k)
#pragma unroll
    for (int e = 3; e >= 0; --e)
      if (at.own(k, e) && (v[k][e] == most || most == -INFINITY)) first = at.row[k] + e;
  if (first >= 0) best = lp_key(most, first);
  // (a wavefront's own part of LDS, whose accesses are in order: the compiler has to keep them so)
  auto ordered = []() __attribute__((always_inline)) { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); __builtin_amdgcn_wave_barrier(); };
  unsigned long long* list = lists[wv];
  const unsigned order = (unsigned)(best >> 32);
  unsigned long long border = 1;
  if (__popcll(__ballot(order != 0)) >= a.k) {             // the k-th of the lanes' maxima, or several that are alike
    const unsigned value = lp_kth(order, a.k);
    const int above = __popcll(__ballot(order > value));
    border = (unsigned long long)value << 32;
    // several are alike at the border: of those the first places
    if (__popcll(__ballot(order >= value)) != a.k) border |= lp_kth(order == value ? (unsigned)best : 0, a.k - above);
  }
  const float least = border > 1 ? lp_key_value(border) : -INFINITY;
  int count = 0;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool may = !(v[k][e] < least);
      if (__ballot(may)) {
        const unsigned long long q = may ? key_of(k, e) : 0, in = __ballot(q >= border);
        if (q >= border) list[count + lp_before(in)] = q;
        count += __popcll(in);
      }
    }
  ordered();
  if (lane < 2) list[count + lane] = 0;
  ordered();
  lp_places(list, count, a.k, lane, 64, [&](int place, unsigned long long key) __attribute__((always_inline)) { if (live) lp_top_out(a, col, place, key, o); });
}

// target = logp_weight (onehot(label) - p) - entropy_weight p (log p + entropy), log p = mat - log_z, p = e^(log p): one pass.  A unit of 64
// lanes (columns of up to 1024 rows) or 256 (pieces of 4096) takes up to 16 rows a lane of one column; the rows behind the last group of
// four go one a lane, so that target may be mat (no row is read by one lane when another may have written it).  8 bytes an entry: 32768 x
// 1000 45.5 us, 5.8 TB/s (copy rate: 40.6), 32003 x 1000 47.5, 1000 x 20000 31.6, 512 x 40000 29.3 (25.4).  A short column leaves lanes without work:
// 100 x 200000 52.2 (24.8), 64 x 100000 24.9 (7.9), 3 x 1000000 192 (3.7).
struct LogProbGradArgs {
  const float *mat, *labels, *log_z, *logp_weight, *entropy, *entropy_weight;
  float* target;
  int h, w, pieces, length;        // pieces of a column, and their rows (a multiple of 4)
};
template <int T, bool STREAM>
__global__ void __launch_bounds__(256) k_log_probs_grad(LogProbGradArgs a) {
  const int lane = threadIdx.x % T;
  const long long unit = (long long)blockIdx.x * (256 / T) + threadIdx.x / T;
  const long long col = T == 64 ? unit : unit / a.pieces;
  const int piece = T == 64 ? 0 : (int)(unit - col * a.pieces);
  if (col >= a.w) return;
  const int row0 = piece * a.length, n = a.h - row0 < a.length ? a.h - row0 : a.length, n4 = n >> 2;
  const float* c = a.mat + (size_t)col * a.h + row0;
  float* t = a.target + (size_t)col * a.h + row0;
  float v[4][4], last = 0.f;
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (lane + T * u < n4) col_load<STREAM>(v[u], c + 4 * (lane + T * u));
  const bool tail = lane < (n & 3);
  if (tail) last = c[4 * n4 + lane];
  const float z = a.log_z[col], l = a.labels ? a.labels[col] : -1.f;
  const bool token = l >= 0.f && l < (float)a.h;
  const int label = token ? (int)l - row0 : -1;
  const float lw = token ? (a.logp_weight ? a.logp_weight[col] : 1.f) : 0.f;
  const float ew = a.entropy_weight ? a.entropy_weight[col] : 0.f, ent = a.entropy ? a.entropy[col] : 0.f;
  auto one = [&](float x, int i) __attribute__((always_inline)) {
    const float lp = x - z;
    const float e = __builtin_amdgcn_exp2f(__fmaf_rn(lp, 1.925963033500011e-08f, lp * 1.44269502162933349609375f));
    const float p = x == -INFINITY ? 0.f : e;                        // (of a column of nothing else log p is no number)
    const float q = p == 0.f ? 0.f : p * (lp + ent);
    return lw * ((i == label ? 1.f : 0.f) - p) - ew * q;
  };
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int j = lane + T * u;
    if (j < n4) {
      const float y[4] = {one(v[u][0], 4 * j), one(v[u][1], 4 * j + 1), one(v[u][2], 4 * j + 2), one(v[u][3], 4 * j + 3)};
      col_store<STREAM>(t + 4 * j, y);
    }
  }
  if (tail) t[4 * n4 + lane] = one(last, 4 * n4 + lane);
}

static inline long long end_of(const cudamat* a) { return dn_len(a); }
static inline bool apart(const cudamat* a, const cudamat* b) {
  return !a || !b || a->data_device + end_of(a) <= b->data_device || b->data_device + end_of(b) <= a->data_device;
}
// NULL, or rows x cols on the device
static int check_shape(const cudamat* m, int rows, int cols) {
  if (!m) return 0;
  if (!m->on_device) return ERROR_NOT_ON_DEVICE;
  if (m->is_trans) return ERROR_TRANSPOSED;
  return m->size[0] == rows && m->size[1] == cols ? 0 : ERROR_INCOMPATIBLE_DIMENSIONS;
}
#define LP_SEGMENT 4096           // rows of one trip of a workgroup
#define LP_WAVE_COLUMNS (1 << 30)  // columns that wavefronts take: they are counted in 31 bits, four a workgroup
#define LP_JOIN 512               // keys that the last workgroup of a column ranks
#define DPTR(m) ((m) ? (m)->data_device : nullptr)

// The columns of one launch.
static int log_probs_launch(LogProbArgs a, bool stream) {
  const int h = a.h, w = a.w, k = a.k;
  // Columns of up to 1024 rows by a wavefront each, and where there are enough of them for the chip those that are shorter than one trip of a
  // workgroup (us, workgroup / wavefront: 2050 x 8192 26.3 / 16.9, 1500 x 20000 50.8 / 21.2; 4096 x 8192 23.0 / 23.9, 3001 x 1100 6.7 / 7.3).
  // Up to 512 rows four columns a wavefront (us, one / four: 100 x 200000 67.8 / 22.3, 256 x 80000 30.3 / 15.2, 500 x 40000 20.0 / 15.7, 1024 x
  // 20000 15.5 / 19.9).
  if (h >= 4 && (h <= 1024 || (h < LP_SEGMENT && !k && w >= 8 * dn_num_cus()))) {
#define LP_WAVE4(T, NV, TAIL, TOP, S) \
  hipLaunchKernelGGL((k_log_probs_wave<T, NV, TAIL, TOP, S>), dim3((unsigned)((w + 256 / T - 1) / (256 / T))), dim3(256), 0, dn_stream(), a)
#define LP_WAVE3(T, NV, TOP, S) do { if (h % 4) LP_WAVE4(T, NV, true, TOP, S); else LP_WAVE4(T, NV, false, TOP, S); } while (0)
#define LP_WAVES(T, NV) do { if (stream) LP_WAVE3(T, NV, false, true); else LP_WAVE3(T, NV, false, false); } while (0)
    if (k && h <= 256) LP_WAVE3(64, 1, true, false);
    else if (k && h <= 512) LP_WAVE3(64, 2, true, false);
    else if (k) LP_WAVE3(64, 4, true, false);
    else if (h <= 64) LP_WAVES(16, 1);
    else if (h <= 128) LP_WAVES(16, 2);
    else if (h <= 256) LP_WAVES(16, 4);
    else if (h <= 512) LP_WAVES(16, 8);
    else if (h <= 4 * 256) LP_WAVES(64, 4);
    else if (h <= 8 * 256) LP_WAVES(64, 8);
    else if (h <= 12 * 256) LP_WAVES(64, 12);
    else LP_WAVES(64, 16);
#undef LP_WAVES
#undef LP_WAVE3
#undef LP_WAVE4
    return dn_launch_status();
  }
  // few columns: segments of them, about two workgroups a CU, none shorter than LP_SEGMENT rows
  int segments = 2 * dn_num_cus() / (w < 2 * dn_num_cus() ? w : 2 * dn_num_cus());
  const int most[3] = {(h + LP_SEGMENT - 1) / LP_SEGMENT, 64, k ? LP_JOIN / k : 64};
  for (int m : most) segments = segments < m ? segments : m;
  if (segments < 1) segments = 1;                         // (no rows: columns of nothing)
  if (segments > 1) {
    a.length = ((h + segments - 1) / segments + 3) / 4 * 4;
    a.segments = segments = (h + a.length - 1) / a.length;
    const size_t parts = (size_t)w * segments;
    a.keys = (unsigned long long*)dn_scratch(parts * (8 * k + 16));
    a.arrived = dn_zero_words(w);
    if (!a.keys || !a.arrived) return CUDA_ERROR;
    a.parts = (float*)(a.keys + parts * k);
  }
#define LP_GO(TOP, S) hipLaunchKernelGGL((k_log_probs<TOP, S>), dim3((unsigned)(w * segments)), dim3(256), 0, dn_stream(), a)
  if (k) { if (stream) LP_GO(true, true); else LP_GO(true, false); }
  else if (stream) LP_GO(false, true);
  else LP_GO(false, false);
#undef LP_GO
  return dn_launch_status();
}

extern "C" {

int log_probs(cudamat* mat, cudamat* labels, cudamat* logp, cudamat* entropy, cudamat* log_z, cudamat* top, cudamat* top_labels) {
  const int h = mat->size[0], w = mat->size[1];
  if (!mat->on_device) return ERROR_NOT_ON_DEVICE;
  if (mat->is_trans) return ERROR_TRANSPOSED;
  cudamat* row[4] = {labels, logp, entropy, log_z};
  for (cudamat* m : row)
    if (int e = check_shape(m, 1, w)) return e;
  const int k = top ? top->size[0] : top_labels ? top_labels->size[0] : 0;
  if (int e = check_shape(top, k, w)) return e;
  if (int e = check_shape(top_labels, k, w)) return e;
  if (k > h || (logp && !labels)) return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (k > LOG_PROBS_MAX_TOP || h > (1 << 24)) return ERROR_UNSUPPORTED;     // (whole numbers as floats)
  cudamat* out[5] = {logp, entropy, log_z, top, top_labels};
  for (int i = 0; i < 5; ++i) {
    if (!apart(out[i], mat) || !apart(out[i], labels)) return ERROR_UNSUPPORTED;
    for (int j = 0; j < i; ++j)
      if (!apart(out[i], out[j])) return ERROR_UNSUPPORTED;
  }
  if (w <= 0) return 0;
  // (at any alignment: 32003 x 2048 50.6 -> 46.9 us; 32768 x 2048 51.5 -> 45.4)
  const bool stream = (long long)h * w >= DN_STREAM_MIN_ELEMS;
  // Columns of up to 1024 rows go four or sixteen to a workgroup, others one.  Even ranges, so that all take the same kernel.
  const long long most = h >= 4 && h <= 1024 ? 4 * DN_MAX_GROUPS : DN_MAX_GROUPS, launches = (w + most - 1) / most, each = (w + launches - 1) / launches;
  for (long long c0 = 0; c0 < w; c0 += each) {
    const int n = (int)(w - c0 < each ? w - c0 : each);
    auto from = [c0](float* p, int rows) { return p ? p + c0 * rows : nullptr; };
    const LogProbArgs a = {mat->data_device + c0 * h, from(DPTR(labels), 1), from(DPTR(logp), 1), from(DPTR(entropy), 1), from(DPTR(log_z), 1),
                           from(DPTR(top), k), from(DPTR(top_labels), k), h, n, k, 1, h, nullptr, nullptr, nullptr};
    if (int e = log_probs_launch(a, stream)) return e;
  }
  return 0;
}

int log_probs_grad(cudamat* mat, cudamat* labels, cudamat* log_z, cudamat* logp_weight, cudamat* entropy, cudamat* entropy_weight,
                   cudamat* target) {
  const int h = mat->size[0], w = mat->size[1];
  if (!mat->on_device || !target->on_device || !log_z->on_device) return ERROR_NOT_ON_DEVICE;
  if (mat->is_trans || target->is_trans) return ERROR_TRANSPOSED;
  if (target->size[0] != h || target->size[1] != w) return ERROR_INCOMPATIBLE_DIMENSIONS;
  cudamat* row[5] = {labels, log_z, logp_weight, entropy, entropy_weight};
  for (cudamat* m : row)
    if (int e = check_shape(m, 1, w)) return e;
  if ((logp_weight && !labels) || (!entropy) != (!entropy_weight)) return ERROR_INCOMPATIBLE_DIMENSIONS;
  for (cudamat* m : row)
    if (!apart(m, target)) return ERROR_UNSUPPORTED;
  if ((!apart(mat, target) && mat->data_device != target->data_device) || h > (1 << 24)) return ERROR_UNSUPPORTED;
  if (h <= 0 || w <= 0) return 0;
  const bool wave = h <= 1024;
  const int pieces = wave ? 1 : (h + 4095) / 4096;
  // (at any alignment: 32003 x 1000 51.7 -> 47.7 us)
  const bool stream = (long long)h * w >= DN_STREAM_MIN_ELEMS;
  const long long most = wave ? 4 * DN_MAX_GROUPS : DN_MAX_GROUPS / pieces;            // columns of one launch
  for (long long c0 = 0; c0 < w; c0 += most) {
    const int n = (int)(w - c0 < most ? w - c0 : most);
    auto from = [c0](const cudamat* m) { return m ? m->data_device + c0 : nullptr; };
    const LogProbGradArgs a = {mat->data_device + c0 * h, from(labels), from(log_z), from(logp_weight), from(entropy), from(entropy_weight),
                               target->data_device + c0 * h, h, n, pieces, wave ? h : ((h + pieces - 1) / pieces + 3) / 4 * 4};
    const unsigned blocks = wave ? (unsigned)((n + 3ll) / 4) : (unsigned)n * (unsigned)pieces;
#define LP_GRAD(T, S) hipLaunchKernelGGL((k_log_probs_grad<T, S>), dim3(blocks), dim3(256), 0, dn_stream(), a)
    if (wave) { if (stream) LP_GRAD(64, true); else LP_GRAD(64, false); }
    else if (stream) LP_GRAD(256, true);
    else LP_GRAD(256, false);
#undef LP_GRAD
    if (int e = dn_launch_status()) return e;
  }
  return 0;
}

}  // extern "C"
