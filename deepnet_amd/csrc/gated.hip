// Gated products act(G) * U of the two halves of one product, and their backward pass (no counterpart in cudamat.cu).
#include "columns.h"
#include "gated_act.h"
#include <type_traits>

int dn_row_sums(const float* M, int h, int w, float* y, float alpha, float beta);
bool dn_gemm_gated(bool a_trans, bool b_trans, int N, int K, const float* A, int lda, const float* B, int ldb, const GatedOut& out, int* err);

// ------------------------------------------------------------------ up to eight columns
// One to eight columns (single tokens of a few sequences) against weights whose rows are contiguous: bound by the weights' bytes.  A
// wavefront (or the four of a workgroup, a quarter of the terms each, where there are few units) has R units, that is 2 R rows, for all
// columns; its lanes take 16 bytes of every row at any 4-byte boundary, U pieces of 256 terms on their way at once.  us, 2048 -> 5632 units (14.3 by
// the bytes) of 1, 2, 4, 8 columns: 14.8 to 15.2, 16.6, 18.1, 22.6; 4096 -> 8192 of one 38.2, 7.0 TB/s (some of it from the caches); 2048 -> 512 of one
// 3.6.  Two units a wavefront read the inputs half as often: 17.2 for one column, four and eight columns take 19.0 and 28.0 with one.  Weights read
// with cached loads 16.6 for 14.9, loads of whole trips behind no branch 15.8 for 15.3.
struct GatedColumnsArgs {
  const float *A, *B;
  int lda, ldb, K, n;
  GatedOut out;
  int first;                       // unit that the launch begins at
};
template <int N, int R, int U, bool SHARED>
__global__ void __launch_bounds__(256) k_gated_columns(GatedColumnsArgs a) {
  __shared__ float part[SHARED ? 4 : 1][2 * R * N];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), f = a.out.f;
  const int unit0 = a.first + (SHARED ? (int)blockIdx.x : (int)blockIdx.x * 4 + wv) * R, n4 = a.K >> 2;
  if (!SHARED && unit0 >= f) return;
  // (columns of the group: the last one moves back and leaves the same results for those that it shares)
  const int col0 = (int)(blockIdx.y + 1) * N <= a.n ? (int)blockIdx.y * N : a.n - N;
  const float* B = a.B + (size_t)col0 * a.ldb;
  // (units beyond the last one repeat it and store nothing)
  const float* row[2 * R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = unit0 + r < f ? unit0 + r : f - 1;
    row[2 * r] = a.A + (size_t)i * a.lda;
    row[2 * r + 1] = a.A + ((size_t)f + i) * a.lda;
  }
  float acc[2 * R][N];
#pragma unroll
  for (int r = 0; r < 2 * R; ++r)
#pragma unroll
    for (int c = 0; c < N; ++c) acc[r][c] = 0.f;
  const int step = 64 * U * (SHARED ? 4 : 1);
  for (int j0 = SHARED ? 64 * U * wv : 0; j0 < n4; j0 += step) {
    float w[U][2 * R][4], x[U][N][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + 64 * u + lane;
#pragma unroll
      for (int r = 0; r < 2 * R; ++r) {
        w[u][r][0] = w[u][r][1] = w[u][r][2] = w[u][r][3] = 0.f;
        if (j < n4) col_load<true>(w[u][r], row[r] + 4 * j);
      }
#pragma unroll
      for (int c = 0; c < N; ++c) {
        x[u][c][0] = x[u][c][1] = x[u][c][2] = x[u][c][3] = 0.f;
        if (j < n4) col_load<false>(x[u][c], B + (size_t)c * a.ldb + 4 * j);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int r = 0; r < 2 * R; ++r)
#pragma unroll
        for (int c = 0; c < N; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r][c] = __fmaf_rn(w[u][r][e], x[u][c][e], acc[r][c]);
  }
  if (lane < (a.K & 3) && (!SHARED || wv == 0)) {
    const int k = 4 * n4 + lane;
#pragma unroll
    for (int r = 0; r < 2 * R; ++r)
#pragma unroll
      for (int c = 0; c < N; ++c) acc[r][c] = __fmaf_rn(row[r][k], B[(size_t)c * a.ldb + k], acc[r][c]);
  }
#pragma unroll
  for (int r = 0; r < 2 * R; ++r)
#pragma unroll
    for (int c = 0; c < N; ++c) acc[r][c] = lanes_sum<64>(acc[r][c]);
  if (SHARED) {
    if (lane == 0) {
#pragma unroll
      for (int r = 0; r < 2 * R; ++r)
#pragma unroll
        for (int c = 0; c < N; ++c) part[wv][r * N + c] = acc[r][c];
    }
    __syncthreads();
    if (wv) return;
#pragma unroll
    for (int r = 0; r < 2 * R; ++r)
#pragma unroll
      for (int c = 0; c < N; ++c) acc[r][c] = (part[0][r * N + c] + part[SHARED ? 1 : 0][r * N + c]) + (part[SHARED ? 2 : 0][r * N + c] + part[SHARED ? 3 : 0][r * N + c]);
  }
  // lane r N + c finishes unit r, column c
  float g = 0.f, u = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < N; ++c) {
      g = lane == r * N + c ? acc[2 * r][c] : g;
      u = lane == r * N + c ? acc[2 * r + 1][c] : u;
    }
  if (lane < R * N && unit0 + lane / N < f) gated_out(a.out, unit0 + lane / N, col0 + lane % N, g, u);
}

#define GATED_COLUMNS 8
// More than eight: in groups of as many, all in one grid.
static int gated_columns(GatedColumnsArgs a) {
  const int f = a.out.f, groups = (a.n + GATED_COLUMNS - 1) / GATED_COLUMNS, n = (a.n + groups - 1) / groups;
  // A workgroup's wavefronts share a unit's terms, if there are more than one holds (200 -> 1500 units of eight columns 6.6 us shared, 4.8 not), where there
  // are fewer than eight wavefronts a CU by themselves (us, by themselves / shared: 2048 -> 512 4.3 / 3.6, 500 -> 1000 of four 4.65 / 4.2), and
  // where up to four columns have more than a thousand terms (4096 -> 8192 42.3 / 38.2, 2048 -> 5632 15.8 / 15.2, of three 18.6 / 16.8; 1001 ->
  // 3000 5.9 / 6.9, 500 -> 3000 of four 5.9 / 6.7, 2048 -> 5632 of eight 22.6 / 26.9).
  const bool shared = a.K > 256 && (f < 8 * dn_num_cus() || (n <= 4 && a.K > 1024));
#define GATED_COLS(N, R, U)                                                                                                       \
  case N:                                                                                                                         \
    if (shared) hipLaunchKernelGGL((k_gated_columns<N, R, U, true>), dim3((unsigned)((f + R - 1) / R), (unsigned)groups), dim3(256), 0, dn_stream(), a); \
    else                                                                                                                          \
      for (long long i0 = 0; i0 < f; i0 += 4 * R * DN_MAX_GROUPS) {                                                               \
        const long long units = f - i0 < 4 * R * DN_MAX_GROUPS ? f - i0 : 4 * R * DN_MAX_GROUPS;                                  \
        a.first = (int)i0;                                                                                                        \
        hipLaunchKernelGGL((k_gated_columns<N, R, U, false>), dim3((unsigned)((units + 4 * R - 1) / (4 * R)), (unsigned)groups), dim3(256), 0, dn_stream(), a); \
      }                                                                                                                           \
    break
  switch (n) {
    GATED_COLS(1, 1, 4);
    GATED_COLS(2, 1, 4);
    GATED_COLS(3, 2, 2);
    GATED_COLS(4, 2, 2);
    GATED_COLS(5, 2, 2);
    GATED_COLS(6, 2, 2);
    GATED_COLS(7, 2, 2);
    GATED_COLS(8, 2, 2);
  }
#undef GATED_COLS
  return dn_launch_status();
}

// ------------------------------------------------------------------ a pass over the halves
// A wavefront takes 256 rows of one column or fewer, four a lane; the rows behind the last group go one a lane.  Bound by the bytes, 20 a unit and
// column backward and 12 forward: 4096 units of 2048 columns backward 30 to 32 us, 5.2 to
// 5.6 TB/s.  (Four groups a lane on their way at once: 4096 units of 1000 columns
// with 256 inputs, all of the backward pass, 92.4 us for 90.3, of 100 columns 48.3 for 45.7, of one with 2048 inputs 37.2 for 34.7.)
struct GatePass {
  const float *deriv, *pre;
  float* target;
  int f, w, act, pieces, length;
};
// GRAD: target (2 f rows, may be pre) = the derivatives by the halves; else target = act(gate) * up.
template <bool GRAD, bool STREAM>
__global__ void __launch_bounds__(256) k_gate_pass(GatePass a) {
  const int lane = threadIdx.x & 63;
  const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
  const long long col = unit / a.pieces;
  if (col >= a.w) return;
  const int row0 = (int)(unit - col * a.pieces) * a.length, n = a.f - row0 < a.length ? a.f - row0 : a.length, n4 = n >> 2;
  const float* g = a.pre + 2 * (size_t)col * a.f + row0;
  const float* d = GRAD ? a.deriv + (size_t)col * a.f + row0 : nullptr;
  float* t = a.target + (GRAD ? 2 : 1) * (size_t)col * a.f + row0;
  auto one = [&](float gate, float up, float deriv, float& to_gate, float& to_up) __attribute__((always_inline)) {
    if (GRAD) {
      float slope;
      const float v = gate_act_slope(gate, a.act, &slope);
      to_gate = deriv * up * slope;
      to_up = deriv * v;
    } else {
      to_gate = gate_act(gate, a.act) * up;
    }
  };
  if (lane < n4) {
    float x[4], y[4], z[4], p[4], q[4];
    col_load<STREAM>(x, g + 4 * lane);
    col_load<STREAM>(y, g + a.f + 4 * lane);
    if (GRAD) col_load<STREAM>(z, d + 4 * lane);
#pragma unroll
    for (int e = 0; e < 4; ++e) one(x[e], y[e], GRAD ? z[e] : 0.f, p[e], q[e]);
    col_store<STREAM>(t + 4 * lane, p);
    if (GRAD) col_store<STREAM>(t + a.f + 4 * lane, q);
  }
  if (lane < (n & 3)) {
    const int i = 4 * n4 + lane;
    float p, q;
    one(g[i], g[a.f + i], GRAD ? d[i] : 0.f, p, q);
    t[i] = p;
    if (GRAD) t[a.f + i] = q;
  }
}
template <bool GRAD>
static int gate_pass(const float* deriv, const float* pre, float* target, int f, int w, int act) {
  const int pieces = (f + 255) / 256;
  const bool stream = (long long)f * w >= DN_STREAM_MIN_ELEMS;
  const long long most = 4 * DN_MAX_GROUPS / pieces;         // columns of one launch
  for (long long c0 = 0; c0 < w; c0 += most) {
    const int n = (int)(w - c0 < most ? w - c0 : most);
    const GatePass a = {GRAD ? deriv + c0 * f : nullptr, pre + 2 * c0 * f, target + (GRAD ? 2 : 1) * c0 * f, f, n, act, pieces, ((f + pieces - 1) / pieces + 3) / 4 * 4};
    const unsigned blocks = (unsigned)(((long long)n * pieces + 3) / 4);
    if (stream) hipLaunchKernelGGL((k_gate_pass<GRAD, true>), dim3(blocks), dim3(256), 0, dn_stream(), a);
    else hipLaunchKernelGGL((k_gate_pass<GRAD, false>), dim3(blocks), dim3(256), 0, dn_stream(), a);
  }
  return dn_launch_status();
}

// ------------------------------------------------------------------ the backward products of up to sixteen columns
// Both are bound by the weights' bytes: their gradient mult x d^T (k rows, 2 f columns) is written, the inputs' gradient W d reads them.  One kernel
// does both, so that reads and writes share the memory's time.  A wavefront has 256 rows, four a lane at any 4-byte boundary, and every fourth
// unit of a slice of the 2 f; the derivatives d of the slice wait in LDS.  The four meet in LDS for W d, the slices' parts are added up by
// k_few_finish.  2048 -> 4096 units, one column: 31.7 us in all (20.8 by the bytes), of which k_few_finish
// is 3 and the pass over the halves 2; eight 34.6, 500 -> 500 of one 9.4.  In a kernel each: 34.7, 41.2, 13.6.  Eight units are on their way at once
// (four: 39.1, 44.7, sixteen: 31.5, 36.3), four from nine columns on: sixteen 39.1 (eight 48.1; the two products by k_gemm's kernels 51.9), twelve 36.5
// (37.3; 51.5), 4096 -> 8192 of sixteen 140.6 (168.8; 154.9).
#define FEW_ROWS 256
#define FEW_SLICE 128
#define FEW_COLUMNS 16
struct FewArgs {
  const float *W, *x, *d;
  float *dw, *dx, *partial, *bias_grad;
  int n, k, units, slice, slices;       // n: columns (N may be one more: it counts as zeros)
  float beta, mult;
};
// DX: dx = W d.  DW: dw = mult x d^T, with ADD + beta dw.  The sums of d to bias_grad, where that is given, by the first block of rows.
template <int N, bool DX, bool DW, bool ADD>
__global__ void __launch_bounds__(256) k_few(FewArgs a) {
  __shared__ float ds[FEW_SLICE][N], part[DX ? 4 : 1][N][DX ? FEW_ROWS : 1];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int j0 = blockIdx.y * a.slice, len = a.units - j0 < a.slice ? a.units - j0 : a.slice;
  for (int i = threadIdx.x; i < len * N; i += 256) {
    const int c = i / len, j = i - c * len;
    ds[j][c] = c < a.n ? a.d[(size_t)c * a.units + j0 + j] : 0.f;
  }
  __syncthreads();
  if (a.bias_grad && blockIdx.x == 0)
    for (int j = threadIdx.x; j < len; j += 256) {
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < N; ++c) s += ds[j][c];
      float* b = a.bias_grad + j0 + j;
      *b = a.beta != 0.f ? __fmaf_rn(a.mult, s, a.beta * *b) : a.mult * s;
    }
  // a group over the last row moves back; of the rows that it shares with its neighbour it stores none
  const int first = (int)blockIdx.x * FEW_ROWS + 4 * lane, row = first + 4 <= a.k ? first : a.k - 4, lap = first - row;
  float x[N][4], acc[N][4];
#pragma unroll
  for (int c = 0; c < N; ++c) {
    if (DW) {
      col_load<false>(x[c], a.x + (size_t)(c < a.n ? c : a.n - 1) * a.k + row);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[c][e] = c < a.n ? x[c][e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[c][e] = 0.f;
  }
  constexpr int AHEAD = N > 8 ? 4 : 8;
  const size_t at = (size_t)j0 * a.k + row;
  auto trip = [&](int j, auto units) __attribute__((always_inline)) {
    constexpr int U = decltype(units)::value;
    float v[U][4], old[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const size_t o = at + (size_t)(j + 4 * u) * a.k;
      if (DX) col_load<true>(v[u], a.W + o);
      if (ADD) col_load<true>(old[u], a.dw + o);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < N; ++c) {
        const float d = ds[j + 4 * u][c];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (DX) acc[c][e] = __fmaf_rn(v[u][e], d, acc[c][e]);
          if (DW) y[e] = __fmaf_rn(x[c][e], d, y[e]);
        }
      }
      if (!DW) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = ADD ? __fmaf_rn(a.mult, y[e], a.beta * old[u][e]) : a.mult * y[e];
      float* out = a.dw + at + (size_t)(j + 4 * u) * a.k;
      if (lap == 0) {
        col_store<true>(out, y);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e >= lap) out[e] = y[e];
      }
    }
  };
  int j = wv;
  for (; j + 4 * (AHEAD - 1) < len; j += 4 * AHEAD) trip(j, std::integral_constant<int, AHEAD>());
  for (; j < len; j += 4) trip(j, std::integral_constant<int, 1>());
  if (!DX) return;
#pragma unroll
  for (int c = 0; c < N; ++c)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e >= lap) part[wv][c][row + e - (int)blockIdx.x * FEW_ROWS] = acc[c][e];
  __syncthreads();
  const int r = blockIdx.x * FEW_ROWS + threadIdx.x;
  if (r < a.k)
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if (c >= a.n) break;
      const float s = (part[0][c][threadIdx.x] + part[DX ? 1 : 0][c][threadIdx.x]) + (part[DX ? 2 : 0][c][threadIdx.x] + part[DX ? 3 : 0][c][threadIdx.x]);
      (a.slices > 1 ? a.partial + (size_t)blockIdx.y * a.n * a.k : a.dx)[(size_t)c * a.k + r] = s;
    }
}
// dx: n outputs of `slices` partial results, from `first` on, 64 a workgroup, whose wavefronts take every fourth slice.
__global__ void __launch_bounds__(256) k_few_finish(const float* partial, float* dx, long long first, long long n, int slices) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  const long long i = first + (long long)blockIdx.x * 64 + lane;
  float s = 0.f;
  if (i < n)
#pragma unroll 8
    for (int q = wv; q < slices; q += 4) s += partial[q * n + i];
  red[wv][lane] = s;
  __syncthreads();
  if (wv == 0 && i < n) dx[i] = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
}

// At least four rows and 2^30 at most (they are counted in 31 bits); units of 65535 slices of 32 at most.
template <int N>
static int few_columns(FewArgs a) {
  const int cus = dn_num_cus(), blocks = (a.k + FEW_ROWS - 1) / FEW_ROWS;
  // Slices as short as give two workgroups a CU (2048 -> 4096 units of one and of eight columns, us: one workgroup 41.6, 45.8, two 31.7, 34.6, four
  // 37.5, 40.4, eight 31.0, 38.9).
  a.slice = FEW_SLICE;
  while (a.slice > 32 && (long long)blocks * ((a.units + a.slice - 1) / a.slice) < 2 * cus) a.slice >>= 1;
  a.slices = (a.units + a.slice - 1) / a.slice;
  if (a.dx && a.slices > 1) {
    a.partial = (float*)dn_scratch((size_t)a.slices * a.n * a.k * sizeof(float));
    if (!a.partial) return CUDA_ERROR;
  }
  const dim3 grid((unsigned)blocks, (unsigned)a.slices);
#define FEW_GO(DX, DW, ADD) hipLaunchKernelGGL((k_few<N, DX, DW, ADD>), grid, dim3(256), 0, dn_stream(), a)
  const bool add = a.beta != 0.f;
  if (a.dw && a.dx) { if (add) FEW_GO(true, true, true); else FEW_GO(true, true, false); }
  else if (a.dw) { if (add) FEW_GO(false, true, true); else FEW_GO(false, true, false); }
  else if (a.dx) FEW_GO(true, false, false);
  else if (a.bias_grad) FEW_GO(false, false, false);
#undef FEW_GO
  if (a.dx && a.slices > 1) {
    const long long n = (long long)a.n * a.k;
    for (long long i0 = 0; i0 < n; i0 += 64 * DN_MAX_GROUPS) {
      const long long count = n - i0 < 64 * DN_MAX_GROUPS ? n - i0 : 64 * DN_MAX_GROUPS;
      hipLaunchKernelGGL(k_few_finish, dim3((unsigned)((count + 63) / 64)), dim3(256), 0, dn_stream(), (const float*)a.partial, a.dx, i0, n, a.slices);
    }
  }
  return dn_launch_status();
}

static inline bool apart(const cudamat* a, const cudamat* b) {
  return !a || !b || a->data_device + dn_len(a) <= b->data_device || b->data_device + dn_len(b) <= a->data_device;
}
static int check_column(const cudamat* v, int rows) {
  if (!v) return 0;
  if (!v->on_device) return ERROR_NOT_ON_DEVICE;
  if (v->is_trans) return ERROR_TRANSPOSED;
  return v->size[0] == rows && v->size[1] == 1 ? 0 : ERROR_INCOMPATIBLE_DIMENSIONS;
}

extern "C" {

int dot_gated(cudamat* mat1, cudamat* mat2, cudamat* bias, cudamat* target, cudamat* pre, int act) {
  if (!mat1->on_device || !mat2->on_device || !target->on_device || (pre && !pre->on_device)) return ERROR_NOT_ON_DEVICE;
  if (target->is_trans || (pre && pre->is_trans)) return ERROR_TRANSPOSED;
  const int f = target->size[0], n = target->size[1], k = get_leading_dimension(mat2);
  if (f > 0x3fffffff || get_leading_dimension(mat1) != 2 * f || get_nonleading_dimension(mat2) != n || get_nonleading_dimension(mat1) != k ||
      (pre && (pre->size[0] != 2 * f || pre->size[1] != n)))
    return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (int e = check_column(bias, 2 * f)) return e;
  cudamat* in[3] = {mat1, mat2, bias};
  for (cudamat* m : in)
    if (!apart(m, target) || !apart(m, pre)) return ERROR_UNSUPPORTED;       // (the same handle in two places too)
  if (!apart(pre, target)) return ERROR_UNSUPPORTED;
  if (act < GATE_LINEAR || act > GATE_GELU) return ERROR_UNSUPPORTED;
  const long long count = (long long)f * n;
  if (count <= 0) return 0;
  const bool ta = mat1->is_trans != 0, tb = mat2->is_trans != 0;
  const GatedOut out = {bias ? bias->data_device : nullptr, target->data_device, pre ? pre->data_device : nullptr, f, act};
  const GatedColumnsArgs columns = {mat1->data_device, mat2->data_device, mat1->size[0], mat2->size[0], k, n, out, 0};
  if (n <= GATED_COLUMNS && ta && !tb && k > 0) return gated_columns(columns);
  int done = 0;
  if (n > 1 && dn_gemm_gated(ta, tb, n, k, mat1->data_device, mat1->size[0], mat2->data_device, mat2->size[0], out, &done)) return done;
  // Up to two groups of such columns with few terms, which no tile fits, as long as the sums over the lanes take less than a second launch (us, two
  // launches / so: 71 -> 160 units of 10 columns 7.9 / 3.9, 100 -> 1000 of 16 7.6 / 4.5, 64 -> 4096 of 9 8.4 / 5.4; 120 -> 4000 of 16 8.0 / 8.7, 64 -> 8000
  // of 16 7.7 / 13.6).
  if (n <= 2 * GATED_COLUMNS && ta && !tb && k > 0 && k < 128 && count <= 40000) return gated_columns(columns);
  // other products: the halves, then a pass over them
  cudamat both = *target;
  both.size[0] = 2 * f;
  both.data_device = pre ? pre->data_device : (float*)dn_scratch((size_t)2 * count * sizeof(float), 1);
  if (!both.data_device) return CUDA_ERROR;
  const int held = set_deferred_epilogues(0);
  int e = dot(mat1, mat2, &both, 0.f, 1.f);
  if (!e && bias) e = add_col_vec(&both, bias, &both);
  set_deferred_epilogues(held);
  if (e) return e;
  return gate_pass<false>(nullptr, both.data_device, target->data_device, f, n, act);
}

int dot_gated_grad(cudamat* deriv, cudamat* mat1, cudamat* mat2, cudamat* pre, cudamat* target, cudamat* mat1_grad, cudamat* mat2_grad,
                   cudamat* bias_grad, int act, float beta, float mult) {
  cudamat* all[8] = {deriv, mat1, mat2, pre, target, mat1_grad, mat2_grad, bias_grad};
  for (cudamat* m : all)
    if (m && !m->on_device) return ERROR_NOT_ON_DEVICE;
  if (deriv->is_trans || pre->is_trans || target->is_trans || (mat1_grad && mat1_grad->is_trans) || (mat2_grad && mat2_grad->is_trans)) return ERROR_TRANSPOSED;
  const int f = deriv->size[0], n = deriv->size[1], k = get_leading_dimension(mat2);
  if (f > 0x3fffffff || get_leading_dimension(mat1) != 2 * f || get_nonleading_dimension(mat2) != n || get_nonleading_dimension(mat1) != k ||
      pre->size[0] != 2 * f || pre->size[1] != n || target->size[0] != 2 * f || target->size[1] != n ||
      (mat1_grad && (mat1_grad->size[0] != mat1->size[0] || mat1_grad->size[1] != mat1->size[1])) ||
      (mat2_grad && (mat2_grad->size[0] != mat2->size[0] || mat2_grad->size[1] != mat2->size[1])))
    return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (int e = check_column(bias_grad, 2 * f)) return e;
  if (act < GATE_LINEAR || act > GATE_GELU) return ERROR_UNSUPPORTED;
  // target may be pre; everything else that is written is apart from all the rest
  for (int o = 4; o < 8; ++o)
    for (int i = 0; i < o; ++i)
      if (!apart(all[o], all[i]) && !(o == 4 && i == 3 && target->data_device == pre->data_device)) return ERROR_UNSUPPORTED;
  const long long count = (long long)f * n;
  int e = count > 0 ? gate_pass<true>(deriv->data_device, pre->data_device, target->data_device, f, n, act) : 0;
  if (e) return e;
  const float *w = mat1->data_device, *x = mat2->data_device, *d = target->data_device;
  const bool wt = mat1->is_trans != 0, xt = mat2->is_trans != 0;
  if (n >= 1 && n <= FEW_COLUMNS && wt && !xt && f > 0 && k >= 4 && k <= 1 << 30 && 2 * f <= 65535 * 32) {
    const FewArgs a = {w, x, d, mat1_grad ? mat1_grad->data_device : nullptr, mat2_grad ? mat2_grad->data_device : nullptr, nullptr,
                       bias_grad ? bias_grad->data_device : nullptr, n, k, 2 * f, 0, 1, beta, mult};
#define FEW(N) case N: return few_columns<N>(a)
    switch (n <= 8 ? n : (n + 1) / 2 * 2) { FEW(1); FEW(2); FEW(3); FEW(4); FEW(5); FEW(6); FEW(7); FEW(8); FEW(10); FEW(12); FEW(14); FEW(16); }
#undef FEW
  }
  // The sums go with the weights' gradient where a kernel takes both, and the two products, which have nothing to do with each
  // other, share a launch where their tiles do.
  DnRowSumJob job = {d, bias_grad ? bias_grad->data_device : nullptr, 2 * f, n, mult, beta, 0};
  const int kind = bias_grad && mat1_grad && n > 0 && k > 0 ? dn_row_sum_job_kind(d, 2 * f, n) : 0;
  job.scalar = kind == 2;
  dn_group_allow(true);
  // From 64 columns on, on the ring's tiles where they fit: the two products share a launch then (us, by the plain products' rules / so: 1001 -> 1500
  // units of 300 columns 68.9 / 52.8, 256 -> 256 of 64 12.0 / 8.8, 100 -> 500 of 100 12.3 / 10.8, 2048 -> 4096 of 100 101.9 / 104.5; 2048 -> 4096 of
  // 20 56.7 / 71.9, 500 -> 2000 of 50 23.7 / 26.1).
  const bool ring_first = n >= 64;
  // by op(mat1): d op(mat2)^T; where mat1 is stored transposed, so is that
  if (mat1_grad && f > 0 && k > 0) {
    e = wt ? dn_gemm_sums(xt, true, k, 2 * f, n, mult, x, mat2->size[0], d, 2 * f, beta, mat1_grad->data_device, k, &job, kind ? 1 : 0, ring_first)
           : dn_gemm_sums(false, !xt, 2 * f, k, n, mult, d, 2 * f, x, mat2->size[0], beta, mat1_grad->data_device, 2 * f, &job, kind ? 1 : 0, ring_first);
  }
  // by op(mat2): op(mat1)^T d
  if (!e && mat2_grad && k > 0 && n > 0)
    e = xt ? dn_gemm_sums(true, wt, n, k, 2 * f, 1.f, d, 2 * f, w, mat1->size[0], 0.f, mat2_grad->data_device, n, nullptr, 0, ring_first)
           : dn_gemm_sums(!wt, false, k, n, 2 * f, 1.f, w, mat1->size[0], d, 2 * f, 0.f, mat2_grad->data_device, k, nullptr, 0, ring_first);
  dn_group_allow(false);
  dn_close_group();
  if (!e && bias_grad && !kind) e = dn_row_sums(d, 2 * f, n, bias_grad->data_device, mult, beta);
  return e ? e : dn_launch_status();
}

}  // extern "C"
