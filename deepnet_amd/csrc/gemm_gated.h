// Gated products on the tiles of k_gemm_split and k_gemm_ring.  Included by gemm.hip behind gemm_split.h.
#pragma once
#include "gated_act.h"

// A tile's first operand has BM / 2 rows of the gate's half and the same rows of the other half below them, so that a tile ends
// with both factors of its BM / 2 x BN outputs in LDS: the product runs as it does elsewhere, only its rows are fetched from two places,
// and neither half goes through memory (but for `pre`, where the backward pass wants them).
template <class Tile>
struct GatedOperand : RingOperand<Tile> {
  using Base = RingOperand<Tile>;
  __device__ __forceinline__ void init(const float* P, unsigned bytes, int ld, int row0, int f, int K, int tid) {
    constexpr int HALF = Tile::ROWS / 2;
    Base::init(P, bytes, ld, row0, K, tid);
#pragma unroll
    for (int u = 0; u < Base::NG; ++u) {
      const int r = Tile::group_row(tid, u);                         // (a group of four rows is within a half)
      if (r >= HALF) Base::voff[u] += 4u * (unsigned)(f - HALF) * (Tile::KC ? (unsigned)ld : 1u);
    }
  }
};

template <int ROWS_, int BK_, bool KC_>
struct GatedRingTile : RingTile<ROWS_, BK_, KC_> { static constexpr int ROWS = ROWS_; };

struct GatedArgs { RingArgs g; GatedOut out; };         // g.M: 2 f, g.gx: tiles along f

// tile t of a grid of gx x gy, and whether there is one: contiguous runs of tiles per XCD, along the shorter side first
__device__ __forceinline__ bool gated_tile(const RingArgs& g, int& bx, int& by) {
  const int tiles = g.gx * g.gy, run = (tiles + 7) >> 3, t = (int)(blockIdx.x & 7) * run + (int)(blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= run || t >= tiles) return false;
  bx = g.gx >= g.gy ? t / g.gy : t % g.gx;
  by = g.gx >= g.gy ? t % g.gy : t / g.gx;
  return true;
}

// On the bf16 matrix cores (split_tile.h), where the plain product would run there.  Bound as that is, by the rate of those cores at the clock that
// the power limit leaves: 4096 -> 8192 units of 4096 columns 2.76 to 2.81 ms, 196 to 199 TFLOP/s of fp32 results (the product of 8192 x 8192 x
// 8192 reaches 197); the product alone and a pass over the halves took 3.82.
template <bool A_KC, bool B_KC>
__global__ void __launch_bounds__(SPLIT_THREADS, 2) k_gated_split(GatedArgs a) {
  constexpr int BM = SPLIT_BM, BN = SPLIT_BM, BK = SPLIT_BK, NT = SPLIT_THREADS, HALF = BM / 2;
  const RingArgs& g = a.g;
  using OA = GatedOperand<SplitTile<BM, BK, A_KC, NT>>;
  using OB = RingOperand<SplitTile<BN, BK, B_KC, NT>>;
  using Shape = SplitShape<BM, BN, BK, 2, 4, 1, 2, OA, OB>;
  __shared__ __attribute__((aligned(16))) char lds[Shape::LDS];
  const int tid = threadIdx.x, f = a.out.f, N = g.N, K = g.K;
  int bx, by;
  if (!gated_tile(g, bx, by)) return;
  // a tile over the edge moves back inside; the outputs it shares with its neighbour are that one's to store
  const int m_lo = bx * HALF, n_lo = by * BN, m0 = m_lo + HALF <= f ? m_lo : f - HALF, n0 = n_lo + BN <= N ? n_lo : N - BN;
  const int nst = (K + BK - 1) / BK;
  OA oa; OB ob;
  oa.init(g.A, g.a_bytes, g.lda, m0, f, K, tid);
  ob.init(g.B, g.b_bytes, g.ldb, n0, K, tid);
  Shape::template run<true>(lds, oa, ob, nst, nst * BK - K, [] {});
  const float* part = reinterpret_cast<const float*>(lds);
  const int i = tid % HALF;
  for (int c = tid / HALF; c < BN; c += NT / HALF)
    if (m0 + i >= m_lo && n0 + c >= n_lo) gated_out(a.out, m0 + i, n0 + c, part[c * BM + i], part[c * BM + HALF + i]);
}

// On the tiles of the mid-sized products.  Bound by the fp32 matrix cores: 1001 -> 1500 units of 300 columns, gelu, bias and halves kept,
// 21.0 us (86 TFLOP/s; one 64 x 64 tile a CU takes 13.4 at the peak rate of a CU, the rest is its start and end), 20.0 without; the
// other tiles 22.9 to 31.7.  2048 -> 1024 of 500 34.3 us, 122 TFLOP/s.
template <int TB, int BM, int BN, int BK, bool A_KC, bool B_KC>
__global__ void __launch_bounds__(RING_THREADS, 4) k_gated_ring(GatedArgs a) {
  using OA = GatedOperand<GatedRingTile<BM, BK, A_KC>>;
  using OB = RingOperand<RingTile<BN, BK, B_KC>>;
  using Shape = RingShape<TB, BM, BN, BK, OA, OB>;
  constexpr int HALF = BM / 2;
  __shared__ __attribute__((aligned(16))) float lds[Shape::LDS];
  const RingArgs& g = a.g;
  const int tid = threadIdx.x, f = a.out.f, N = g.N, K = g.K;
  int bx, by;
  if (!gated_tile(g, bx, by)) return;
  // (a single tile of fewer columns reads zeros behind the last one, the buffer's range check gives them; dn_gemm_gated)
  const int m_lo = bx * HALF, n_lo = by * BN, m0 = m_lo + HALF <= f ? m_lo : f - HALF, n0 = n_lo + BN <= N || N < BN ? n_lo : N - BN;
  const int nst = (K + BK - 1) / BK;
  OA oa; OB ob;
  oa.init(g.A, g.a_bytes, g.lda, m0, f, K, tid);
  ob.init(g.B, g.b_bytes, g.ldb, n0, K, tid);
  float sum[Shape::EPL];
  Shape::template run<true, false>(lds, oa, ob, nst, nst * BK - K, sum, [] {});
  // (the partial tiles are still in LDS, [n][m])
  const int i = tid % HALF;
  for (int c = tid / HALF; c < BN; c += RING_THREADS / HALF) {
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < Shape::KS; ++w) {
      x += lds[w * (BM * BN) + c * BM + i];
      y += lds[w * (BM * BN) + c * BM + HALF + i];
    }
    if (m0 + i >= m_lo && n0 + c >= n_lo && n0 + c < N) gated_out(a.out, m0 + i, n0 + c, x, y);
  }
}

// target = act(P[0:f]) * P[f:2f] of P = op(A) * op(B) + bias in one launch, where the product of that size runs on tiles that can.
bool dn_gemm_gated(bool a_trans, bool b_trans, int N, int K, const float* A, int lda, const float* B, int ldb, const GatedOut& out, int* err) {
  const int f = out.f, M = 2 * f;
  const bool a_kc = a_trans, b_kc = !b_trans;
  if (f <= 0 || N <= 0 || K <= 0) return false;
  GemmPlan plan = gemm_plan(a_kc, b_kc, M, N, K, A, lda, B, ldb, 0.f);
  // Where the product would run on a kernel without tiles like these, the ring's are taken all the same: no launch and no trip of the halves
  // through memory behind it (us, product and pass / ring: 128 -> 2048 units of 2048 columns 39.8 / 32.1, 128 -> 512 of 128 7.9 / 4.0, 500 ->
  // 1000 of 20 7.8 / 5.7, 2048 -> 5632 of 17 42.3 / 27.2, 4096 -> 512 of 64 19.6 / 13.9).
  if (plan.kind != GEMM_SPLIT && plan.kind != GEMM_RING) {
    const size_t a_bytes = (size_t)lda * (a_kc ? M : K) * sizeof(float), b_bytes = (size_t)ldb * (b_kc ? N : K) * sizeof(float);
    const RingPlan ring = ring_plan(M, N, K, a_bytes, b_bytes, dn_num_cus());
    if (ring.cfg >= 0) plan = GemmPlan{GEMM_RING, ring, false};
    // Strips of 9 to 15 columns, whose other kernels read the weights several times (2048 -> 5632 of 9 44.3 -> 22 us): the tile of 16 columns,
    // where a column beyond the last one lies behind the operand's bytes.
    else if (N > 8 && N < 16 && f >= 16 && K >= 128 && b_kc && a_bytes < (1ull << 31) && (size_t)16 * ldb * sizeof(float) < (1ull << 31))
      plan = GemmPlan{GEMM_RING, RingPlan{4, 0.}, false};
  }
  GatedArgs a = {RingArgs{A, B, nullptr, (unsigned)((size_t)lda * (a_kc ? M : K) * sizeof(float)), (unsigned)((size_t)ldb * (b_kc ? N : K) * sizeof(float)),
                          lda, ldb, 0, M, N, K, 0, 0, 1.f, 0.f}, out};
  auto grid = [&](int half, int bn) {
    a.g.gx = (f + half - 1) / half;
    a.g.gy = (N + bn - 1) / bn;
    return dim3((unsigned)(8 * ((a.g.gx * a.g.gy + 7) / 8)));
  };
#define GATED_KINDS(GO)          \
  if (a_kc && b_kc) GO(true, true);   \
  else if (a_kc) GO(true, false);     \
  else if (b_kc) GO(false, true);     \
  else GO(false, false)
  if (plan.kind == GEMM_SPLIT) {
    const dim3 blocks = grid(SPLIT_BM / 2, SPLIT_BM);
#define GATED_GO(AK, BK_) hipLaunchKernelGGL((k_gated_split<AK, BK_>), blocks, dim3(SPLIT_THREADS), 0, dn_stream(), a)
    GATED_KINDS(GATED_GO);
#undef GATED_GO
  } else if (plan.kind == GEMM_RING) {
    const auto& c = g_ring_cfgs[plan.ring.cfg];
    const dim3 blocks = grid(c.bm / 2, c.bn);
#define GATED_RING(TB, BM, BN, BK)                                                                                                       \
  do {                                                                                                                                   \
    if (a_kc && b_kc) hipLaunchKernelGGL((k_gated_ring<TB, BM, BN, BK, true, true>), blocks, dim3(RING_THREADS), 0, dn_stream(), a);        \
    else if (a_kc) hipLaunchKernelGGL((k_gated_ring<TB, BM, BN, BK, true, false>), blocks, dim3(RING_THREADS), 0, dn_stream(), a);          \
    else if (b_kc) hipLaunchKernelGGL((k_gated_ring<TB, BM, BN, BK, false, true>), blocks, dim3(RING_THREADS), 0, dn_stream(), a);          \
    else hipLaunchKernelGGL((k_gated_ring<TB, BM, BN, BK, false, false>), blocks, dim3(RING_THREADS), 0, dn_stream(), a);                   \
  } while (0)
    switch (plan.ring.cfg) {
      case 0: GATED_RING(32, 64, 64, 32); break;
      case 1: GATED_RING(32, 64, 32, 64); break;
      case 2: GATED_RING(32, 32, 64, 64); break;
      case 3: GATED_RING(16, 32, 32, 64); break;
      case 4: GATED_RING(16, 32, 16, 128); break;
      default: GATED_RING(16, 16, 32, 128); break;
    }
#undef GATED_RING
  } else {
    return false;
  }
#undef GATED_KINDS
  *err = dn_launch_status();
  return true;
}
