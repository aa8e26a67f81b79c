// A gated linear recurrence along the columns of sequences, and its gradients (no counterpart in cudamat.cu).  With the halves g, u of
// pre and a = sigmoid(g):  h_t = a_t h_{t-1} + (1 - a_t) u_t.
#include "columns.h"
#include "gated_act.h"
#include "tokens.h"

struct ScanArgs {
  const float *pre, *offsets, *state, *deriv, *out, *last_deriv;
  float *target, *last, *state_grad;
  int f, w, n, each;               // units, columns, sequences; columns of each where there are no offsets
};

// The first column of sequence q, q <= n; numbers that are out of place stay within the matrix.
__device__ __forceinline__ int scan_border(const ScanArgs& a, int q) {
  if (!a.offsets) return q * a.each;
  const float o = a.offsets[q];
  return o > 0.f ? (o < (float)a.w ? (int)o : a.w) : 0;
}

// A lane a unit, a workgroup a sequence.
__global__ void __launch_bounds__(256) k_gated_scan(ScanArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x, q = blockIdx.y;
  if (i >= a.f) return;
  const size_t f = a.f;
  float h = a.state ? a.state[q * f + i] : 0.f;
  for (int c = scan_border(a, q), end = scan_border(a, q + 1); c < end; ++c) {
    float s;
    const float g = gate_sigmoid(a.pre[2 * f * c + i], &s), u = a.pre[2 * f * c + f + i];
    h = __fmaf_rn(g, h, s * u);
    a.target[f * c + i] = h;
  }
  if (a.last) a.last[q * f + i] = h;
}
__global__ void __launch_bounds__(256) k_gated_scan_grad(ScanArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x, q = blockIdx.y;
  if (i >= a.f) return;
  const size_t f = a.f;
  float back = a.last_deriv ? a.last_deriv[q * f + i] : 0.f;
  const int first = scan_border(a, q);
  for (int c = scan_border(a, q + 1) - 1; c >= first; --c) {
    float s;
    const float g = gate_sigmoid(a.pre[2 * f * c + i], &s), u = a.pre[2 * f * c + f + i];
    const float before = c > first ? a.out[f * (c - 1) + i] : a.state ? a.state[q * f + i] : 0.f;
    const float all = a.deriv[f * c + i] + back;
    a.target[2 * f * c + i] = g * s * (before - u) * all;
    a.target[2 * f * c + f + i] = s * all;
    back = g * all;
  }
  if (a.state_grad) a.state_grad[q * f + i] = back;
}

// Sequences: as many as are asked for, or (0) as the offsets or the states tell, or one.
static int scan_sequences(int asked, const cudamat* offsets, const cudamat* s0, const cudamat* s1, const cudamat* s2) {
  if (asked) return asked;
  if (offsets) return offsets->size[1] - 1;
  for (const cudamat* s : {s0, s1, s2})
    if (s) return s->size[1];
  return 1;
}

extern "C" {

int gated_scan(cudamat* pre, cudamat* offsets, cudamat* state, cudamat* target, cudamat* last, int sequences) {
  cudamat* const all[5] = {pre, offsets, state, target, last};
  if (int e = tok_check_device(all)) return e;
  const int f = target->size[0], w = target->size[1], n = scan_sequences(sequences, offsets, state, last, nullptr);
  if (pre->size[0] != 2 * (long long)f || pre->size[1] != w || n < 1 || !tok_shape(offsets, 1, n + 1) || (!offsets && w % n) ||
      !tok_shape(state, f, n) || !tok_shape(last, f, n))
    return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (!tok_apart(pre, target) || !tok_apart(offsets, target) || !tok_apart(state, target) || !tok_apart(pre, last) || !tok_apart(offsets, last) ||
      !tok_apart(target, last) || (state && last && !tok_same_or_apart(state, last)) || (offsets && w > (1 << 24)))
    return ERROR_UNSUPPORTED;
  if (f <= 0 || (w <= 0 && !last)) return 0;
  const ScanArgs a = {pre->data_device, tok_data(offsets), tok_data(state), nullptr, nullptr, nullptr, target->data_device, tok_data(last), nullptr, f, w, n, w / n};
  hipLaunchKernelGGL(k_gated_scan, dim3((f + 255) / 256, n), dim3(256), 0, dn_stream(), a);
  return dn_launch_status();
}

int gated_scan_grad(cudamat* deriv, cudamat* pre, cudamat* out, cudamat* offsets, cudamat* state, cudamat* last_deriv, cudamat* target,
                    cudamat* state_grad, int sequences) {
  cudamat* const all[8] = {deriv, pre, out, offsets, state, last_deriv, target, state_grad};
  if (int e = tok_check_device(all)) return e;
  const int f = deriv->size[0], w = deriv->size[1], n = scan_sequences(sequences, offsets, state, last_deriv, state_grad);
  if (pre->size[0] != 2 * (long long)f || pre->size[1] != w || !tok_shape(out, f, w) || target->size[0] != pre->size[0] || target->size[1] != w || n < 1 ||
      !tok_shape(offsets, 1, n + 1) || (!offsets && w % n) || !tok_shape(state, f, n) || !tok_shape(last_deriv, f, n) || !tok_shape(state_grad, f, n))
    return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (!tok_same_or_apart(pre, target) || (last_deriv && state_grad && !tok_same_or_apart(last_deriv, state_grad)) || !tok_apart(pre, state_grad) ||
      !tok_apart(target, state_grad) || !tok_apart(last_deriv, target) || (offsets && w > (1 << 24)))
    return ERROR_UNSUPPORTED;
  for (const cudamat* m : {deriv, out, offsets, state})
    if (!tok_apart(m, target) || !tok_apart(m, state_grad)) return ERROR_UNSUPPORTED;
  if (f <= 0 || (w <= 0 && !state_grad)) return 0;
  const ScanArgs a = {pre->data_device, tok_data(offsets), tok_data(state), deriv->data_device, out->data_device, tok_data(last_deriv),
                      target->data_device, nullptr, tok_data(state_grad), f, w, n, w / n};
  hipLaunchKernelGGL(k_gated_scan_grad, dim3((f + 255) / 256, n), dim3(256), 0, dn_stream(), a);
  return dn_launch_status();
}

}  // extern "C"
