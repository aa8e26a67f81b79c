// Layer norm of columns and its gradients (no counterpart in cudamat.cu): a column is the h features of one case.
#include "columns.h"
#include <math.h>

// Sums over the 256 lanes of a workgroup; every lane gets them.  `red` is free again after the next barrier.
__device__ __forceinline__ double wave_sum(double v) { return wave_sum_d(v); }
template <int N, typename V>
__device__ __forceinline__ void block_sums(V (&v)[N], V (*red)[4]) {
  const int wv = threadIdx.x >> 6;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) red[i][wv] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = (red[i][0] + red[i][1]) + (red[i][2] + red[i][3]);
}

// ------------------------------------------------------------------ columns that no team holds
// A workgroup a column, three passes over it (the later ones from the caches): more than 16384 rows, where a lane would have to hold more than
// 16.  20000 x 1000 107 us (1.5 TB/s), its gradients 260: waits for each pass's loads and its meeting.
// The mean as a pair m + d (m rounded to fp32, d what the deviations from m still sum to) and 1 / sqrt(variance + eps):
// deviations are taken from m, so that a mean far from zero costs no digits of the variance.  That takes an m that is off by its own rounding only:
// a lane adds up h / 256 entries, and in 32 bits m was off by so much (1000003 equal entries of 98765.4: by 2.8) that d^2 outweighed
// the variance and what was left of it could be below zero.
struct NormStats { float m, d, r; };
__device__ __forceinline__ NormStats norm_stats(const float* c, int h, float eps, float (*red)[4]) {
  __shared__ double sums[1][4];
  NormStats s;
  double one[1] = {0.0};
  for (int i = threadIdx.x; i < h; i += 256) one[0] += (double)c[i];
  block_sums(one, sums);
  s.m = (float)(one[0] / (double)h);
  float two[2] = {0.f, 0.f};
  for (int i = threadIdx.x; i < h; i += 256) {
    const float x = c[i] - s.m;
    two[0] += x;
    two[1] += x * x;
  }
  block_sums(two, red);
  s.d = two[0] / (float)h;
  const float var = two[1] / (float)h - s.d * s.d;
  s.r = 1.f / sqrtf((var < 0.f ? 0.f : var) + eps);        // (NaN stays)
  return s;
}

__global__ void __launch_bounds__(256) k_layer_norm(const float* mat, const float* gain, const float* bias, float* target, int h, float eps) {
  __shared__ float red[2][4];
  const float* c = mat + (size_t)blockIdx.x * h;
  float* t = target + (size_t)blockIdx.x * h;
  const NormStats s = norm_stats(c, h, eps, red);
  for (int i = threadIdx.x; i < h; i += 256) {
    const float x = ((c[i] - s.m) - s.d) * s.r;
    t[i] = __fmaf_rn(gain ? gain[i] : 1.f, x, bias ? bias[i] : 0.f);
  }
}

// Per column: m, d, r, and the means of g = gain * deriv and of g * x^ (x^: the normalised input).
__global__ void __launch_bounds__(256) k_layer_norm_grad_stats(const float* deriv, const float* mat, const float* gain, float* stats, int h, float eps) {
  __shared__ float red[2][4];
  const float *c = mat + (size_t)blockIdx.x * h, *dy = deriv + (size_t)blockIdx.x * h;
  const NormStats s = norm_stats(c, h, eps, red);
  float two[2] = {0.f, 0.f};
  for (int i = threadIdx.x; i < h; i += 256) {
    const float g = gain ? gain[i] * dy[i] : dy[i];
    two[0] += g;
    two[1] += g * (((c[i] - s.m) - s.d) * s.r);
  }
  block_sums(two, red);
  if (threadIdx.x == 0) {
    float* o = stats + (size_t)blockIdx.x * 5;
    o[0] = s.m; o[1] = s.d; o[2] = s.r; o[3] = two[0] / (float)h; o[4] = two[1] / (float)h;
  }
}
// Gradients of gain and bias: 64 rows a workgroup, its wavefronts take every fourth column.
__global__ void __launch_bounds__(256) k_layer_norm_grad_rows(const float* deriv, const float* mat, const float* stats, float* gain_grad, float* bias_grad,
                                                              int h, int w, float beta, float mult) {
  __shared__ float red[2][4][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, i = blockIdx.x * 64 + lane;
  float sg = 0.f, sb = 0.f;
  if (i < h)
    for (size_t c = wv; c < (size_t)w; c += 4) {
      const float* s = stats + c * 5;
      const float dy = deriv[c * h + i];
      sg += dy * (((mat[c * h + i] - s[0]) - s[1]) * s[2]);
      sb += dy;
    }
  red[0][wv][lane] = sg; red[1][wv][lane] = sb;
  __syncthreads();
  if (wv == 0 && i < h) {
    float* out[2] = {gain_grad, bias_grad};
    for (int k = 0; k < 2; ++k)
      if (out[k]) {
        const float sum = (red[k][0][lane] + red[k][1][lane]) + (red[k][2][lane] + red[k][3][lane]);
        out[k][i] = beta != 0.f ? __fmaf_rn(mult, sum, beta * out[k][i]) : mult * sum;
      }
  }
}
__global__ void __launch_bounds__(256) k_layer_norm_grad_inputs(const float* deriv, const float* mat, const float* gain, const float* stats, float* target, int h) {
  const float* s = stats + (size_t)blockIdx.x * 5;
  const size_t at = (size_t)blockIdx.x * h;
  for (int i = threadIdx.x; i < h; i += 256) {
    const float x = ((mat[at + i] - s[0]) - s[1]) * s[2], g = gain ? gain[i] * deriv[at + i] : deriv[at + i];
    target[at + i] = s[2] * ((g - s[3]) - x * s[4]);
  }
}

// ------------------------------------------------------------------ columns that stay in registers
// A team (16 or 64 lanes, or T = 0: the workgroup) holds a column, NV groups of four rows a lane, from its one read to its one write; gain and bias stay in
// registers for all columns that the team takes, and the next column is on its way while this one is reduced.  Arithmetic of
// k_layer_norm: sum, then deviations from the rounded mean.  Bound by the bytes, 8 an entry: 4096 x 8192 45.7 us, 5.87 TB/s (a copy
// reaches 6.45, 41.6 us), 1024 x 16384 24.2, 16384 x 1024 24.6, 64 x 100000 11.1; at heights that are no multiple of four the columns start
// anywhere in a memory line, 4098 x 4099 27.6 (4.9 TB/s).  1024 x 4: 3.7 to 4.1, of which a launch is 3.
__device__ __forceinline__ float norm_rstd(float sq, float d, float inv_h, float eps) {
  const float var = sq * inv_h - d * d;
  return 1.f / sqrtf((var < 0.f ? 0.f : var) + eps);       // (NaN stays)
}

// A team's sums of deviations.  A wavefront (or a row of 16 lanes) takes deviations from the rounded mean of its own n rows, so that
// nothing is exchanged for the mean first; the wavefronts of a team meet once, in LDS, where each shifts every other's sums to the team's mean
// m: sum (x - m) = S1 + n (m_i - m), sum (x - m)^2 = S2 + 2 (m_i - m) S1 + n (m_i - m)^2, sum g (x - m) = GX + (m_i - m) G.
// `v` holds x on entry and x - m on return (0 outside).
struct NormSums { float d, sq, g, gx; };      // sums of x - m, of its square, of g and of g (x - m)
template <int T, int NV, bool TAIL, bool GRAD>
__device__ __forceinline__ NormSums norm_sums(const ColGroups<NV, TAIL>& at, float (&v)[NV][4], const float (&g)[NV][4], const float (&dy)[NV][4],
                                              float* part, float n, float inv_n, float inv_h, int lane, int W) {
#pragma clang fp contract(off)      // (the deviations are from the rounded means that the wavefronts exchange)
  constexpr int R = T == 16 ? 16 : 64;
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) s += at.own(k, e) ? v[k][e] : 0.f;
  const float mi = lanes_sum<R>(s) * inv_n;
  NormSums o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[k][e] = v[k][e] - mi;
      const float x = at.own(k, e) ? v[k][e] : 0.f;
      o.d += x;
      o.sq = __fmaf_rn(x, x, o.sq);
      if (GRAD) {
        const float y = at.own(k, e) ? g[k][e] * dy[k][e] : 0.f;
        o.g += y;
        o.gx = __fmaf_rn(y, x, o.gx);
      }
    }
  o.d = lanes_sum<R>(o.d); o.sq = lanes_sum<R>(o.sq);
  if (GRAD) { o.g = lanes_sum<R>(o.g); o.gx = lanes_sum<R>(o.gx); }
  if (T) return o;
  // (six arrays of 16)
  if (lane % 64 == 0) {
    float* p = part + lane / 64;
    p[0] = mi; p[16] = n; p[32] = o.d; p[48] = o.sq;
    if (GRAD) { p[64] = o.g; p[80] = o.gx; }
  }
  __syncthreads();
  const int q = lane % 16;
  const bool in = q < W;
  const float mq = in ? part[q] : 0.f, nq = in ? part[16 + q] : 0.f, dq = in ? part[32 + q] : 0.f, sq = in ? part[48 + q] : 0.f;
  const float gq = GRAD && in ? part[64 + q] : 0.f, gxq = GRAD && in ? part[80 + q] : 0.f;
  const float m = lanes_sum<16>(nq * mq) * inv_h, by = mq - m;
  o.d = lanes_sum<16>(__fmaf_rn(nq, by, dq));
  o.sq = lanes_sum<16>(__fmaf_rn(by, __fmaf_rn(nq, by, 2.f * dq), sq));
  if (GRAD) { o.g = lanes_sum<16>(gq); o.gx = lanes_sum<16>(__fmaf_rn(by, gq, gxq)); }
  const float mine = mi - m;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[k][e] += mine;
  return o;
}
// The rows of a wavefront of a team (T = 0), or of a team.
template <int T, int NV>
__device__ __forceinline__ float norm_rows(int lane, int lanes, int h) {
  if (T) return (float)h;
  int n = 0;
  const int first = 4 * (lane & ~63);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int left = h - first - 4 * k * lanes;
    n += left < 0 ? 0 : left < 256 ? left : 256;
  }
  return (float)n;
}

template <int T, int NV, bool TAIL, bool STREAM>
__global__ void __launch_bounds__(T ? 256 : 1024)
k_layer_norm_cols(const float* mat, const float* gain, const float* bias, float* target, int h, int w, float eps) {
  constexpr int TEAMS = T ? 256 / T : 1;
  __shared__ float part[2][T ? 1 : 64];      // (two in turn: one may be read still when the other is written)
  const int lane = T ? threadIdx.x % (T ? T : 1) : threadIdx.x, W = blockDim.x / 64;
  ColGroups<NV, TAIL> at;
  at.init(lane, T ? T : blockDim.x, h);
  const float inv_h = 1.f / (float)h, rows = norm_rows<T, NV>(lane, T ? T : blockDim.x, h), inv_rows = 1.f / rows;
  int turn = 0;
  float gv[NV][4], bv[NV][4], x[NV][4], next[NV][4];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { gv[k][e] = 1.f; bv[k][e] = 0.f; x[k][e] = next[k][e] = 0.f; }
    if (gain) col_load<false>(gv[k], gain + at.row[k]);
    if (bias) col_load<false>(bv[k], bias + at.row[k]);
  }
  const int stride = gridDim.x * TEAMS;
  int c = blockIdx.x * TEAMS + (T ? threadIdx.x / (T ? T : 1) : 0);
  if (c >= w) return;                                      // (whole workgroups where teams meet at barriers)
  auto fetch = [&](float (&v)[NV][4], int col) __attribute__((always_inline)) {
    const float* p = mat + (size_t)col * h;
#pragma unroll
    for (int k = 0; k < NV; ++k) col_load<STREAM>(v[k], p + at.row[k]);
  };
  fetch(x, c);
  for (;;) {
    const int n = c + stride;
    if (n < w) fetch(next, n);
    const NormSums o = norm_sums<T, NV, TAIL, false>(at, x, gv, x, part[turn], rows, inv_rows, inv_h, lane, W);
    turn ^= T ? 0 : 1;
    const float d = o.d * inv_h, r = norm_rstd(o.sq, d, inv_h, eps);
    float* t = target + (size_t)c * h;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (at.in[k]) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = __fmaf_rn(gv[k][e], (x[k][e] - d) * r, bv[k][e]);
        col_store_group<STREAM, T == 0>(at, k, t, y);
      }
    if (n >= w) break;
    c = n;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[k][e] = next[k][e];
  }
}

// Backward in one pass over mat and deriv: with m known, sums of the deviations, their squares, g = gain * deriv and g times
// the deviations come from one round.  The gradients of gain and bias stay in the lanes that have their rows, for all columns of
// the workgroup; its teams meet in LDS at the end, and a second kernel adds up the workgroups (a single one finishes by itself).  12 bytes an
// entry: 4096 x 8192 72.8 us, 5.5 TB/s (copy rate: 62.4), of which the second kernel is 4.2; 1024 x 16384 38.9, 4098 x 4099 45.2 (31.2), 4096 x 4099,
// whose columns start at a memory line, 42.1, 1026 and 1024 x 8192 26.7 and 23.9 (15.6), 4096 x 1000 19.7 (7.6), 4096 x 300 13.8 (2.3), 16384 x 1024
// 52.9 (31.2), 1024 x 4 5.1.  What is over the bytes is the partial sums of up to 256 workgroups with their second launch, whatever the columns'
// number, and the barrier a column, at which a workgroup's teams go in step; vector instructions issue in half of the cycles.
struct NormGradArgs {
  const float *deriv, *mat, *gain;
  float *target, *partial, *gain_grad, *bias_grad;
  int h, w, waves;                // waves: of a team of whole wavefronts
  float eps, beta, mult;
};
__device__ __forceinline__ void norm_param_out(float* out, int i, float sum, float beta, float mult) {
  out[i] = beta != 0.f ? __fmaf_rn(mult, sum, beta * out[i]) : mult * sum;
}

template <int T, int NV, bool TAIL, bool STREAM>
__global__ void __launch_bounds__(1024) k_layer_norm_grad_cols(NormGradArgs a) {
  constexpr int AHEAD = NV <= 3 ? 1 : 0;                   // columns on their way (none fit the registers of 1024 lanes beyond)
  __shared__ float part[2][T ? 1 : 16][T ? 1 : 96];
  __shared__ float meet[NV <= 3 ? 512 * NV * 8 : 1];
  const int h = a.h, w = a.w, W = a.waves, lanes = T ? T : 64 * W, teams = blockDim.x / lanes;
  const int team = T ? threadIdx.x / (T ? T : 1) : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / W, lane = threadIdx.x - team * lanes;
  ColGroups<NV, TAIL> at;
  at.init(lane, lanes, h);
  const float inv_h = 1.f / (float)h, rows = norm_rows<T, NV>(lane, lanes, h), inv_rows = 1.f / rows;
  int turn = 0;
  float gv[NV][4], x[NV][4], dy[NV][4], nx[AHEAD ? AHEAD : 1][NV][4], ny[AHEAD ? AHEAD : 1][NV][4], sg[NV][4], sb[NV][4];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      gv[k][e] = 1.f; x[k][e] = dy[k][e] = sg[k][e] = sb[k][e] = 0.f;
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) nx[q][k][e] = ny[q][k][e] = 0.f;
    }
    if (a.gain) col_load<false>(gv[k], a.gain + at.row[k]);
  }
  const int stride = gridDim.x * teams;
  auto fetch = [&](float (&u)[NV][4], float (&v)[NV][4], int col) __attribute__((always_inline)) {
    const size_t o = (size_t)col * h;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      col_load<STREAM>(u[k], a.mat + o + at.row[k]);
      col_load<STREAM>(v[k], a.deriv + o + at.row[k]);
    }
  };
  // every team of a workgroup makes the same number of trips; those beyond the last column count and store nothing
  int c = blockIdx.x * teams + team;
  auto column = [&](int n) __attribute__((always_inline)) { return n < w ? n : w - 1; };      // (behind the last one: that one again, from the caches)
  if (AHEAD) fetch(x, dy, column(c));
#pragma unroll
  for (int q = 0; q + 1 < AHEAD; ++q) fetch(nx[q], ny[q], column(c + (q + 1) * stride));
  for (int base = blockIdx.x * teams; base < w; base += stride) {
    const bool live = c < w;
    const int n = column(c + AHEAD * stride);
    if (AHEAD) fetch(nx[AHEAD ? AHEAD - 1 : 0], ny[AHEAD ? AHEAD - 1 : 0], n);
    else fetch(x, dy, n);
    const NormSums o = norm_sums<T, NV, TAIL, true>(at, x, gv, dy, part[T ? 0 : turn][T ? 0 : team], rows, inv_rows, inv_h, lane, W);
    turn ^= 1;
    const float d = o.d * inv_h, r = norm_rstd(o.sq, d, inv_h, a.eps);
    const float mg = o.g * inv_h, mgx = r * (o.gx - d * o.g) * inv_h;
    if (live) {
      float* t = a.target + (size_t)c * h;
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (at.in[k]) {
          float out[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float xh = (x[k][e] - d) * r;
            sg[k][e] = __fmaf_rn(dy[k][e], xh, sg[k][e]);
            sb[k][e] += dy[k][e];
            out[e] = r * (__fmaf_rn(gv[k][e], dy[k][e], -mg) - xh * mgx);
          }
          col_store_group<STREAM, T == 0>(at, k, t, out);
        }
    }
    c += stride;
    if (AHEAD) {
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[k][e] = nx[0][k][e]; dy[k][e] = ny[0][k][e];
#pragma unroll
          for (int q = 0; q + 1 < AHEAD; ++q) { nx[q][k][e] = nx[q + 1][k][e]; ny[q][k][e] = ny[q + 1][k][e]; }
        }
    }
  }
  if (!a.gain_grad && !a.bias_grad) return;
  if (T == 16) {                  // teams of one wavefront
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) {
          sg[k][e] += __shfl_xor(sg[k][e], o, WAVE);
          sb[k][e] += __shfl_xor(sb[k][e], o, WAVE);
        }
  }
  // the later half of the teams (wavefronts, of teams that share one) hands its sums to the earlier one
  const int U = T == 16 ? 64 : lanes, unit = T == 16 ? threadIdx.x >> 6 : team;
  for (int units = blockDim.x / U; units > 1; units = (units + 1) >> 1) {
    const int half = (units + 1) >> 1;
    __syncthreads();
    if (unit >= half && unit < units) {
      const int to = (int)threadIdx.x - half * U;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) { meet[(8 * k + e) * 512 + to] = sg[k][e]; meet[(8 * k + 4 + e) * 512 + to] = sb[k][e]; }
    }
    __syncthreads();
    if (unit + half < units) {
      const int from = threadIdx.x;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) { sg[k][e] += meet[(8 * k + e) * 512 + from]; sb[k][e] += meet[(8 * k + 4 + e) * 512 + from]; }
    }
  }
  if ((int)threadIdx.x < lanes) {
    float* p = a.partial + (size_t)blockIdx.x * 2 * h;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (at.own(k, e)) {
          const int i = at.row[k] + e;
          if (gridDim.x > 1) { p[i] = sg[k][e]; p[h + i] = sb[k][e]; }
          else {
            if (a.gain_grad) norm_param_out(a.gain_grad, i, sg[k][e], a.beta, a.mult);
            if (a.bias_grad) norm_param_out(a.bias_grad, i, sb[k][e], a.beta, a.mult);
          }
        }
  }
}
// The sums of `parts` workgroups: 64 of the 2 h rows a workgroup, its 16 wavefronts take every sixteenth part, eight on their way at once.
__global__ void __launch_bounds__(1024) k_layer_norm_grad_finish(NormGradArgs a, int parts) {
  __shared__ float red[16][64];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, rows = 2 * a.h, i = blockIdx.x * 64 + lane;
  const float* from = a.partial + (i < rows ? i : rows - 1);
  float s = 0.f;
  for (int p = wv; p < parts; p += 16 * 8) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = from[(size_t)(p + 16 * u < parts ? p + 16 * u : p) * rows];
#pragma unroll
    for (int u = 0; u < 8; ++u) s += p + 16 * u < parts ? v[u] : 0.f;
  }
  red[wv][lane] = s;
  __syncthreads();
  if (wv == 0 && i < rows) {
#pragma unroll
    for (int k = 1; k < 16; ++k) s += red[k][lane];
    float* out = i < a.h ? a.gain_grad : a.bias_grad;
    if (out) norm_param_out(out, i < a.h ? i : i - a.h, s, a.beta, a.mult);
  }
}

// ------------------------------------------------------------------ columns of one to three rows
// A lane a column: nothing is exchanged but the sums of gain and bias, at the end.  us, a workgroup a column before: 3 x 1000000 916 -> 8.0, its
// gradients 57123 -> 15.2 (those of gain and bias went through one workgroup).
template <int H>
__device__ __forceinline__ NormSums norm_short(float (&x)[H], const float (&g)[H], const float (&dy)[H]) {
#pragma clang fp contract(off)
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < H; ++i) s += x[i];
  const float m = s / (float)H;
  NormSums o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < H; ++i) {
    x[i] -= m;
    o.d += x[i];
    o.sq = __fmaf_rn(x[i], x[i], o.sq);
    o.g += g[i] * dy[i];
    o.gx = __fmaf_rn(g[i] * dy[i], x[i], o.gx);
  }
  return o;
}
template <int H>
__global__ void __launch_bounds__(256) k_layer_norm_short(const float* mat, const float* gain, const float* bias, float* target, int w, float eps) {
  for (size_t c = (size_t)blockIdx.x * 256 + threadIdx.x; c < (size_t)w; c += (size_t)gridDim.x * 256) {
    float x[H];
#pragma unroll
    for (int i = 0; i < H; ++i) x[i] = mat[c * H + i];
    const NormSums o = norm_short<H>(x, x, x);
    const float d = o.d / (float)H, r = norm_rstd(o.sq, d, 1.f / (float)H, eps);
#pragma unroll
    for (int i = 0; i < H; ++i) target[c * H + i] = __fmaf_rn(gain ? gain[i] : 1.f, (x[i] - d) * r, bias ? bias[i] : 0.f);
  }
}
template <int H>
__global__ void __launch_bounds__(256) k_layer_norm_grad_short(NormGradArgs a) {
  __shared__ float red[4][2 * H];
  float g[H], sum[2 * H];
#pragma unroll
  for (int i = 0; i < H; ++i) { g[i] = a.gain ? a.gain[i] : 1.f; sum[i] = sum[H + i] = 0.f; }
  for (size_t c = (size_t)blockIdx.x * 256 + threadIdx.x; c < (size_t)a.w; c += (size_t)gridDim.x * 256) {
    float x[H], dy[H];
#pragma unroll
    for (int i = 0; i < H; ++i) { x[i] = a.mat[c * H + i]; dy[i] = a.deriv[c * H + i]; }
    const NormSums o = norm_short<H>(x, g, dy);
    const float d = o.d / (float)H, r = norm_rstd(o.sq, d, 1.f / (float)H, a.eps), mg = o.g / (float)H, mgx = r * (o.gx - d * o.g) / (float)H;
#pragma unroll
    for (int i = 0; i < H; ++i) {
      const float xh = (x[i] - d) * r;
      sum[i] = __fmaf_rn(dy[i], xh, sum[i]);
      sum[H + i] += dy[i];
      a.target[c * H + i] = r * (__fmaf_rn(g[i], dy[i], -mg) - xh * mgx);
    }
  }
  if (!a.gain_grad && !a.bias_grad) return;
#pragma unroll
  for (int i = 0; i < 2 * H; ++i) sum[i] = lanes_sum<64>(sum[i]);
  if (threadIdx.x % 64 == 0) {
#pragma unroll
    for (int i = 0; i < 2 * H; ++i) red[threadIdx.x / 64][i] = sum[i];
  }
  __syncthreads();
  const int i = threadIdx.x;
  if (i >= 2 * H) return;
  const float s = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
  float* out = i < H ? a.gain_grad : a.bias_grad;
  if (gridDim.x > 1) a.partial[(size_t)blockIdx.x * 2 * H + i] = s;
  else if (out) norm_param_out(out, i % H, s, a.beta, a.mult);
}

#define NORM_COLS_MAX 16384       // tallest columns that a team holds
#define NORM_COLS_W (1 << 29)     // most of them in a launch (they are counted in 31 bits)
#define NORM_ROWS_MAX ((1 << 30) - 1)
// Columns of one launch; those of up to three rows are counted in 64 bits.
static inline long long norm_launch_columns(int h) { return h < 4 ? 0x7fffffffll : h <= NORM_COLS_MAX ? NORM_COLS_W : DN_MAX_GROUPS; }

// waves: of the workgroup, where that is a team
template <int T, int NV>
static void norm_launch(const float* mat, const float* gain, const float* bias, float* target, int h, int w, float eps, int waves = 4) {
  const int teams = T ? 256 / (T ? T : 1) : 1, nt = 64 * waves;
  // (at any alignment: 4098 x 4099 32.7 -> 28.8 us, 1001 x 8000 14.7 -> 13.3)
  const bool tail = h % 4 != 0, stream = (long long)h * w >= DN_STREAM_MIN_ELEMS;
  // as many workgroups as fit the CUs, or one for as many columns as makes them even
  const int groups = (w + teams - 1) / teams, most = dn_num_cus() * (2048 / nt), each = (groups + most - 1) / most;
  const dim3 grid((unsigned)((groups + each - 1) / each));
  if (tail && stream) hipLaunchKernelGGL((k_layer_norm_cols<T, NV, true, true>), grid, dim3(nt), 0, dn_stream(), mat, gain, bias, target, h, w, eps);
  else if (tail) hipLaunchKernelGGL((k_layer_norm_cols<T, NV, true, false>), grid, dim3(nt), 0, dn_stream(), mat, gain, bias, target, h, w, eps);
  else if (stream) hipLaunchKernelGGL((k_layer_norm_cols<T, NV, false, true>), grid, dim3(nt), 0, dn_stream(), mat, gain, bias, target, h, w, eps);
  else hipLaunchKernelGGL((k_layer_norm_cols<T, NV, false, false>), grid, dim3(nt), 0, dn_stream(), mat, gain, bias, target, h, w, eps);
}

template <int T, int NV>
static int norm_grad_launch(NormGradArgs a) {
  const int lanes = T ? T : 64 * a.waves, cus = dn_num_cus(), least = T == 16 ? 4 : 1;
  // teams of a workgroup: all that fit, or fewer where that leaves CUs without one; a workgroup a CU (two of half the teams: 4098 x 4099 45.2 ->
  // 51.4 us, 4096 x 8192 72.6 -> 76.2)
  int teams = 1024 / lanes;
  // What one workgroup does in a trip (two, of teams within a wavefront) it does alone, without a launch for the sums (us, two launches / one: 1024 x 4
  // 7.1 / 5.1, 1024 x 8 7.4 / 6.7, 256 x 16 7.1 / 4.3, 256 x 32 7.4 / 5.4, 64 x 64 7.3 / 4.2; two trips of larger teams 1024 x 16 7.5 / 8.7).
  const bool sums = a.gain_grad || a.bias_grad, alone = sums && a.w <= (T ? 2 : 1) * teams;
  if (alone && a.w < teams) teams = (a.w + least - 1) / least * least;       // (whole wavefronts)
  while (!alone && teams > least && (a.w + teams - 1) / teams < cus) teams = (teams + 1) / 2 > least ? (teams + 1) / 2 : least;
  int blocks = (a.w + teams - 1) / teams;
  if (alone) blocks = 1;
  if (blocks > cus) blocks = cus;
  if (sums && blocks > 1) {
    a.partial = (float*)dn_scratch((size_t)blocks * 2 * a.h * sizeof(float));
    if (!a.partial) return CUDA_ERROR;
  }
  // (at any alignment: 4098 x 4099 46.4 -> 45.3 us, 1026 x 8192 29.3 -> 26.9)
  const bool tail = a.h % 4 != 0, stream = (long long)a.h * a.w >= DN_STREAM_MIN_ELEMS;
  const dim3 grid((unsigned)blocks), block((unsigned)(teams * lanes));
  if (tail && stream) hipLaunchKernelGGL((k_layer_norm_grad_cols<T, NV, true, true>), grid, block, 0, dn_stream(), a);
  else if (tail) hipLaunchKernelGGL((k_layer_norm_grad_cols<T, NV, true, false>), grid, block, 0, dn_stream(), a);
  else if (stream) hipLaunchKernelGGL((k_layer_norm_grad_cols<T, NV, false, true>), grid, block, 0, dn_stream(), a);
  else hipLaunchKernelGGL((k_layer_norm_grad_cols<T, NV, false, false>), grid, block, 0, dn_stream(), a);
  if (sums && blocks > 1)
    hipLaunchKernelGGL(k_layer_norm_grad_finish, dim3((unsigned)((2 * a.h + 63) / 64)), dim3(1024), 0, dn_stream(), a, blocks);
  return dn_launch_status();
}

template <int H>
static int norm_grad_short(NormGradArgs a) {
  // (columns of a lane: one, or as many as leave two workgroups a CU)
  const long long groups = (a.w + 255ll) / 256, most = 2 * dn_num_cus();
  const int blocks = (int)(groups < most ? groups : most);
  const bool sums = a.gain_grad || a.bias_grad;
  if (sums && blocks > 1) {
    a.partial = (float*)dn_scratch((size_t)blocks * 2 * H * sizeof(float));
    if (!a.partial) return CUDA_ERROR;
  }
  hipLaunchKernelGGL(k_layer_norm_grad_short<H>, dim3((unsigned)blocks), dim3(256), 0, dn_stream(), a);
  if (sums && blocks > 1) hipLaunchKernelGGL(k_layer_norm_grad_finish, dim3(1), dim3(1024), 0, dn_stream(), a, blocks);
  return dn_launch_status();
}

static inline bool apart(const cudamat* a, const cudamat* b) {
  return !a || !b || a->data_device + dn_len(a) <= b->data_device || b->data_device + dn_len(b) <= a->data_device;
}
static inline bool same_or_apart(const cudamat* a, const cudamat* b) {
  return apart(a, b) || (a->data_device == b->data_device && a->size[0] == b->size[0] && a->size[1] == b->size[1]);
}
static int check_vector(const cudamat* v, int h) {
  if (!v) return 0;
  if (!v->on_device) return ERROR_NOT_ON_DEVICE;
  if (v->is_trans) return ERROR_TRANSPOSED;
  return v->size[0] == h && v->size[1] == 1 ? 0 : ERROR_INCOMPATIBLE_DIMENSIONS;
}

// What one launch takes of the columns.
static int norm_columns(const float* x, const float* g, const float* b, float* t, int h, int w, float eps) {
  if (h >= 4 && h <= NORM_COLS_MAX) {
    // Teams of 16 lanes up to 64 rows, a wavefront up to 1024 (us, against the next larger team: 64 x 100000 11.0 / 23.9, 60 x 300 3.3 / 4.2, 700 x
    // 20000 22.3 / 24.0, 1024 x 16384 24.1 / 24.4; gradients 64 x 100000 19.1 / 38.3).
    if (h <= 64) norm_launch<16, 1>(x, g, b, t, h, w, eps);
    else if (h <= 256) norm_launch<64, 1>(x, g, b, t, h, w, eps);
    else if (h <= 512) norm_launch<64, 2>(x, g, b, t, h, w, eps);
    else if (h <= 1024) norm_launch<64, 4>(x, g, b, t, h, w, eps);
    // Two groups a lane (us, two / four: 4096 x 8192 45.7 / 47.0, 6001 x 5000 44.0 / 46.2, 1026 x 8192 15.0 / 16.5; 3000 x 8192 39.6 / 38.6; a
    // wavefront with eight takes 18.4 for 1026 x 8192), four where that is more than 16 wavefronts.
    else if (h <= 8192) norm_launch<0, 2>(x, g, b, t, h, w, eps, (h + 511) / 512);
    else norm_launch<0, 4>(x, g, b, t, h, w, eps, (h + 1023) / 1024);
    return dn_launch_status();
  }
  if (h < 4) {
    const long long groups = (w + 255ll) / 256, most = 8 * dn_num_cus();
    const dim3 grid((unsigned)(groups < most ? groups : most));
    if (h == 1) hipLaunchKernelGGL(k_layer_norm_short<1>, grid, dim3(256), 0, dn_stream(), x, g, b, t, w, eps);
    else if (h == 2) hipLaunchKernelGGL(k_layer_norm_short<2>, grid, dim3(256), 0, dn_stream(), x, g, b, t, w, eps);
    else hipLaunchKernelGGL(k_layer_norm_short<3>, grid, dim3(256), 0, dn_stream(), x, g, b, t, w, eps);
    return dn_launch_status();
  }
  hipLaunchKernelGGL(k_layer_norm, dim3((unsigned)w), dim3(256), 0, dn_stream(), x, g, b, t, h, eps);
  return dn_launch_status();
}

static int norm_grad_columns(NormGradArgs a) {
  const int h = a.h, w = a.w;
  if (w > 0 && h <= NORM_COLS_MAX) {
    if (h == 1) return norm_grad_short<1>(a);
    if (h == 2) return norm_grad_short<2>(a);
    if (h == 3) return norm_grad_short<3>(a);
    if (h <= 64) return norm_grad_launch<16, 1>(a);
    if (h <= 256) return norm_grad_launch<64, 1>(a);
    if (h <= 512) return norm_grad_launch<64, 2>(a);
    if (h <= 8192) {
      // Two groups a lane, or three where that gives a workgroup half as many teams again: more columns are on their way (us, two / three:
      // 4098 x 4099 47.4 / 45.2, 1500 x 8192 33.9 / 33.4, 6144 x 4096 66.8 / 62.3, 700 x 20000 40.9 / 38.1; 6001 x 5000 74.6 / 75.1; 2048 x 8192, four
      // teams against five, 42.8 / 45.1).
      const int two = (h + 511) / 512, three = (h + 767) / 768;
      a.waves = two;
      if (2 * (16 / three) < 3 * (16 / two)) return norm_grad_launch<0, 2>(a);
      a.waves = three;
      return norm_grad_launch<0, 3>(a);
    }
    a.waves = (h + 1023) / 1024;
    return norm_grad_launch<0, 4>(a);
  }
  float* stats = (float*)dn_scratch((size_t)(w > 0 ? w : 1) * 5 * sizeof(float));
  if (!stats) return CUDA_ERROR;
  if (w > 0) hipLaunchKernelGGL(k_layer_norm_grad_stats, dim3((unsigned)w), dim3(256), 0, dn_stream(), a.deriv, a.mat, a.gain, stats, h, a.eps);
  if (a.gain_grad || a.bias_grad)
    hipLaunchKernelGGL(k_layer_norm_grad_rows, dim3((unsigned)((h + 63) / 64)), dim3(256), 0, dn_stream(), a.deriv, a.mat, (const float*)stats, a.gain_grad,
                       a.bias_grad, h, w, a.beta, a.mult);
  if (w > 0) hipLaunchKernelGGL(k_layer_norm_grad_inputs, dim3((unsigned)w), dim3(256), 0, dn_stream(), a.deriv, a.mat, a.gain, (const float*)stats, a.target, h);
  return dn_launch_status();
}

extern "C" {

int layer_norm(cudamat* mat, cudamat* gain, cudamat* bias, cudamat* target, float eps) {
  const int h = mat->size[0], w = mat->size[1];
  if (!mat->on_device || !target->on_device) return ERROR_NOT_ON_DEVICE;
  if (mat->is_trans || target->is_trans) return ERROR_TRANSPOSED;
  if (target->size[0] != h || target->size[1] != w) return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (int e = check_vector(gain, h)) return e;
  if (int e = check_vector(bias, h)) return e;
  if (!(eps >= 0.f) || !same_or_apart(mat, target) || !apart(gain, target) || !apart(bias, target)) return ERROR_UNSUPPORTED;
  if (h > NORM_ROWS_MAX) return ERROR_UNSUPPORTED;         // (rows are counted in 31 bits, 256 at a time)
  if (h <= 0 || w <= 0) return 0;
  const float *x = mat->data_device, *g = gain ? gain->data_device : nullptr, *b = bias ? bias->data_device : nullptr;
  const long long most = norm_launch_columns(h);
  for (long long c0 = 0; c0 < w; c0 += most)
    if (int e = norm_columns(x + c0 * h, g, b, target->data_device + c0 * h, h, (int)(w - c0 < most ? w - c0 : most), eps)) return e;
  return 0;
}

int layer_norm_grad(cudamat* deriv, cudamat* mat, cudamat* gain, cudamat* target, cudamat* gain_grad, cudamat* bias_grad, float eps,
                    float beta, float mult) {
  const int h = mat->size[0], w = mat->size[1];
  if (!deriv->on_device || !mat->on_device || !target->on_device) return ERROR_NOT_ON_DEVICE;
  if (deriv->is_trans || mat->is_trans || target->is_trans) return ERROR_TRANSPOSED;
  if (deriv->size[0] != h || deriv->size[1] != w || target->size[0] != h || target->size[1] != w) return ERROR_INCOMPATIBLE_DIMENSIONS;
  cudamat* vec[3] = {gain, gain_grad, bias_grad};
  for (cudamat* v : vec)
    if (int e = check_vector(v, h)) return e;
  if (!(eps >= 0.f) || !same_or_apart(deriv, target) || !same_or_apart(mat, target) || !apart(gain, target)) return ERROR_UNSUPPORTED;
  cudamat* in[4] = {deriv, mat, gain, target};
  for (cudamat* m : in)
    if (!apart(m, gain_grad) || !apart(m, bias_grad)) return ERROR_UNSUPPORTED;
  if (!apart(gain_grad, bias_grad)) return ERROR_UNSUPPORTED;
  if (h > NORM_ROWS_MAX) return ERROR_UNSUPPORTED;
  if (h <= 0) return 0;
  NormGradArgs a = {deriv->data_device, mat->data_device, gain ? gain->data_device : nullptr, target->data_device, nullptr,
                    gain_grad ? gain_grad->data_device : nullptr, bias_grad ? bias_grad->data_device : nullptr, h, w, 0, eps, beta, mult};
  const long long most = norm_launch_columns(h);
  for (long long c0 = 0;;) {
    a.w = (int)(w - c0 < most ? w - c0 : most);
    if (int e = norm_grad_columns(a)) return e;
    c0 += most;
    if (c0 >= w) return 0;
    a.deriv += most * h; a.mat += most * h; a.target += most * h;
    a.beta = 1.f;                                          // (the gradients of gain and bias go on from what these columns left)
  }
}

}  // extern "C"
