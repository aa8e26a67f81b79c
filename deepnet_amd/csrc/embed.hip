// Columns of a table by token, and the gradient of the table (no counterpart in cudamat.cu; selectRows has no scale and gives NaN for what is
// no token, accumulate_columns is for up to 512 columns).
#include "columns.h"
#include "tokens.h"

// target(:, c) = mult * mat(:, labels[c]), 0 where that is no token.
__global__ void __launch_bounds__(256) k_embed(const float* mat, const float* labels, float* target, int h, int n, float mult) {
  const int c = blockIdx.x, t = tok_label(labels[c], n);
  for (int i = threadIdx.x; i < h; i += 256) target[(size_t)c * h + i] = t >= 0 ? mult * mat[(size_t)t * h + i] : 0.f;
}

// target(:, t) = beta * target(:, t) + mult * sum of the columns of token t, in the order of the columns: a workgroup a token.
__global__ void __launch_bounds__(256) k_embed_grad(const float* deriv, const float* labels, float* target, int h, int w, int n, float beta, float mult) {
  __shared__ int list[256], counts[4];
  const int t = blockIdx.x, lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
  for (int i0 = 0; i0 < h; i0 += 256) {
    const int i = i0 + threadIdx.x;
    float s = 0.f;
    for (int c0 = 0; c0 < w; c0 += 256) {
      const int c = c0 + threadIdx.x;
      const bool in = c < w && tok_label(labels[c], n) == t;
      const unsigned long long all = __ballot(in);
      if (lane == 0) counts[wv] = __popcll(all);
      __syncthreads();
      int at = __popcll(all & ((1ull << lane) - 1)), count = 0;
      for (int k = 0; k < 4; ++k) { if (k < wv) at += counts[k]; count += counts[k]; }
      if (in) list[at] = c;
      __syncthreads();
      if (i < h)
        for (int k = 0; k < count; ++k) s += deriv[(size_t)list[k] * h + i];
      __syncthreads();
    }
    if (i < h) {
      float* out = target + (size_t)t * h + i;
      *out = beta != 0.f ? __fmaf_rn(mult, s, beta * *out) : mult * s;
    }
  }
}

extern "C" {

int embed(cudamat* mat, cudamat* labels, cudamat* target, float mult) {
  cudamat* const all[3] = {mat, labels, target};
  if (int e = tok_check_device(all)) return e;
  const int h = mat->size[0], n = mat->size[1], w = target->size[1];
  if (target->size[0] != h || !tok_shape(labels, 1, w)) return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (n > (1 << 24) || !tok_apart(mat, target) || !tok_apart(labels, target)) return ERROR_UNSUPPORTED;
  if (h <= 0 || w <= 0) return 0;
  hipLaunchKernelGGL(k_embed, dim3(w), dim3(256), 0, dn_stream(), mat->data_device, labels->data_device, target->data_device, h, n, mult);
  return dn_launch_status();
}

int embed_grad(cudamat* deriv, cudamat* labels, cudamat* target, float beta, float mult) {
  cudamat* const all[3] = {deriv, labels, target};
  if (int e = tok_check_device(all)) return e;
  const int h = deriv->size[0], n = target->size[1], w = deriv->size[1];
  if (target->size[0] != h || !tok_shape(labels, 1, w)) return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (n > (1 << 24) || !tok_apart(deriv, target) || !tok_apart(labels, target)) return ERROR_UNSUPPORTED;
  if (h <= 0 || n <= 0) return 0;
  hipLaunchKernelGGL(k_embed_grad, dim3(n), dim3(256), 0, dn_stream(), deriv->data_device, labels->data_device, target->data_device, h, w, n, beta, mult);
  return dn_launch_status();
}

}  // extern "C"
