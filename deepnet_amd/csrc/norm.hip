// Layer norm of columns and its gradients (no counterpart in cudamat.cu): a column is the h features of one case.
#include "common.h"
#include <math.h>

// Sums over the 256 lanes of a workgroup; every lane gets them.  `red` is free again after the next barrier.
template <int N>
__device__ __forceinline__ void block_sums(float (&v)[N], float (*red)[4]) {
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

// The mean as a pair m + d (m the rounded sum's, d what the deviations from m still sum to) and 1 / sqrt(variance + eps):
// deviations are taken from m, so that a mean far from zero costs no digits of the variance.
struct NormStats { float m, d, r; };
__device__ __forceinline__ NormStats norm_stats(const float* c, int h, float eps, float (*red)[4]) {
  NormStats s;
  float one[1] = {0.f};
  for (int i = threadIdx.x; i < h; i += 256) one[0] += c[i];
  block_sums(one, red);
  s.m = one[0] / (float)h;
  float two[2] = {0.f, 0.f};
  for (int i = threadIdx.x; i < h; i += 256) {
    const float x = c[i] - s.m;
    two[0] += x;
    two[1] += x * x;
  }
  block_sums(two, red);
  s.d = two[0] / (float)h;
  s.r = 1.f / sqrtf(two[1] / (float)h - s.d * s.d + eps);
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
    for (int c = wv; c < w; c += 4) {
      const float* s = stats + (size_t)c * 5;
      const float dy = deriv[(size_t)c * h + i];
      sg += dy * (((mat[(size_t)c * h + i] - s[0]) - s[1]) * s[2]);
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

extern "C" {

int layer_norm(cudamat* mat, cudamat* gain, cudamat* bias, cudamat* target, float eps) {
  const int h = mat->size[0], w = mat->size[1];
  if (!mat->on_device || !target->on_device) return ERROR_NOT_ON_DEVICE;
  if (mat->is_trans || target->is_trans) return ERROR_TRANSPOSED;
  if (target->size[0] != h || target->size[1] != w) return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (int e = check_vector(gain, h)) return e;
  if (int e = check_vector(bias, h)) return e;
  if (!(eps >= 0.f) || !same_or_apart(mat, target) || !apart(gain, target) || !apart(bias, target)) return ERROR_UNSUPPORTED;
  if (h <= 0 || w <= 0) return 0;
  hipLaunchKernelGGL(k_layer_norm, dim3((unsigned)w), dim3(256), 0, dn_stream(), (const float*)mat->data_device,
                     (const float*)(gain ? gain->data_device : nullptr), (const float*)(bias ? bias->data_device : nullptr), target->data_device, h, eps);
  return dn_launch_status();
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
  if (h <= 0) return 0;
  float* stats = (float*)dn_scratch((size_t)(w > 0 ? w : 1) * 5 * sizeof(float));
  if (!stats) return CUDA_ERROR;
  const float* gp = gain ? gain->data_device : nullptr;
  if (w > 0)
    hipLaunchKernelGGL(k_layer_norm_grad_stats, dim3((unsigned)w), dim3(256), 0, dn_stream(), (const float*)deriv->data_device,
                       (const float*)mat->data_device, gp, stats, h, eps);
  if (gain_grad || bias_grad)
    hipLaunchKernelGGL(k_layer_norm_grad_rows, dim3((unsigned)((h + 63) / 64)), dim3(256), 0, dn_stream(), (const float*)deriv->data_device,
                       (const float*)mat->data_device, (const float*)stats, gain_grad ? gain_grad->data_device : nullptr,
                       bias_grad ? bias_grad->data_device : nullptr, h, w, beta, mult);
  if (w > 0)
    hipLaunchKernelGGL(k_layer_norm_grad_inputs, dim3((unsigned)w), dim3(256), 0, dn_stream(), (const float*)deriv->data_device,
                       (const float*)mat->data_device, gp, (const float*)stats, target->data_device, h);
  return dn_launch_status();
}

}  // extern "C"
