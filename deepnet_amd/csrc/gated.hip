// Gated products act(G) * U of the two halves of one product, and their backward pass (no counterpart in cudamat.cu).
#include "common.h"
#include "wide_math.h"
#include <math.h>

enum { GATE_LINEAR = 0, GATE_SIGMOID = 1, GATE_RELU = 2, GATE_TANH = 3, GATE_SILU = 4, GATE_GELU = 5 };

// The share of a normal variable below g; erfc keeps the digits of the small ones.
__device__ __forceinline__ float gate_phi(float g) { return 0.5f * erfcf(g * -0.70710678118654752440f); }

__device__ __forceinline__ float gate_act(float g, int act) {
  switch (act) {
    case GATE_SIGMOID: return dn_sigmoid(g);
    case GATE_RELU: return g < 0.f ? 0.f : g;
    case GATE_TANH: return dn_tanh(g);
    case GATE_SILU: return g * dn_sigmoid(g);
    case GATE_GELU: return g * gate_phi(g);
    default: return g;
  }
}
// The activation and its slope.
__device__ __forceinline__ float gate_act_slope(float g, int act, float* slope) {
  switch (act) {
    case GATE_SIGMOID: { const float s = dn_sigmoid(g); *slope = s * dn_sigmoid(-g); return s; }
    case GATE_RELU: *slope = g > 0.f ? 1.f : 0.f; return g < 0.f ? 0.f : g;
    case GATE_TANH: { const float s = dn_tanh(g); *slope = (1.f - s) * (1.f + s); return s; }
    case GATE_SILU: { const float s = dn_sigmoid(g), v = g * s; *slope = __fmaf_rn(v, dn_sigmoid(-g), s); return v; }
    case GATE_GELU: { const float p = gate_phi(g); *slope = __fmaf_rn(g * 0.39894228040143267794f, dn_exp(-0.5f * g * g), p); return g * p; }
    default: *slope = 1.f; return g;
  }
}

// pre: the halves, f rows each, one above the other.
__global__ void __launch_bounds__(256) k_gate(const float* pre, float* target, long long n, int f, int act) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= n) return;
  const long long c = at / f, i = at - c * f;
  target[at] = gate_act(pre[2 * c * f + i], act) * pre[2 * c * f + f + i];
}
// target (may be pre): the derivatives by the halves.
__global__ void __launch_bounds__(256) k_gate_grad(const float* deriv, const float* pre, float* target, long long n, int f, int act) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= n) return;
  const long long c = at / f, g = 2 * c * f + (at - c * f);
  float slope;
  const float d = deriv[at], u = pre[g + f], v = gate_act_slope(pre[g], act, &slope);
  target[g] = d * u * slope;
  target[g + f] = d * v;
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
  cudamat* in[4] = {mat1, mat2, bias, pre};
  for (cudamat* m : in)
    if (!apart(m, target) || (m != pre && !apart(m, pre))) return ERROR_UNSUPPORTED;
  if (act < GATE_LINEAR || act > GATE_GELU) return ERROR_UNSUPPORTED;
  const long long count = (long long)f * n;
  if (count <= 0) return 0;
  if ((count + 255) / 256 > 0x7fffffffll) return ERROR_UNSUPPORTED;
  cudamat both = *target;
  both.size[0] = 2 * f;
  both.data_device = pre ? pre->data_device : (float*)dn_scratch((size_t)2 * count * sizeof(float), 1);
  if (!both.data_device) return CUDA_ERROR;
  const int held = set_deferred_epilogues(0);
  int e = dot(mat1, mat2, &both, 0.f, 1.f);
  if (!e && bias) e = add_col_vec(&both, bias, &both);
  set_deferred_epilogues(held);
  if (e) return e;
  hipLaunchKernelGGL(k_gate, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, dn_stream(), (const float*)both.data_device, target->data_device, count, f, act);
  return dn_launch_status();
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
  if ((count + 255) / 256 > 0x7fffffffll) return ERROR_UNSUPPORTED;
  if (count > 0)
    hipLaunchKernelGGL(k_gate_grad, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, dn_stream(), (const float*)deriv->data_device,
                       (const float*)pre->data_device, target->data_device, count, f, act);
  int e = dn_launch_status();
  const int held = set_deferred_epilogues(0);
  cudamat d = *target, x = *mat2, w = *mat1;
  if (!e && mat1_grad) {
    // by op(mat1): d op(mat2)^T; where mat1 is stored transposed, so is that
    if (mat1->is_trans) { d.is_trans = 1; e = dot(&x, &d, mat1_grad, beta, mult); d.is_trans = 0; }
    else { x.is_trans = !x.is_trans; e = dot(&d, &x, mat1_grad, beta, mult); x.is_trans = mat2->is_trans; }
  }
  if (!e && mat2_grad) {
    // by op(mat2): op(mat1)^T d
    if (mat2->is_trans) { d.is_trans = 1; e = dot(&d, &w, mat2_grad, 0.f, 1.f); d.is_trans = 0; }
    else { w.is_trans = !w.is_trans; e = dot(&w, &d, mat2_grad, 0.f, 1.f); }
  }
  if (!e && bias_grad) e = beta == 0.f && mult == 1.f ? sum_by_axis(&d, bias_grad, 1) : 0;
  if (!e && bias_grad && !(beta == 0.f && mult == 1.f)) {
    if (beta == 0.f) e = assign_scalar(bias_grad, 0.f);
    else if (beta != 1.f) e = mult_by_scalar(bias_grad, beta, bias_grad);
    if (!e) e = add_sum_by_axis(&d, bias_grad, 1, mult);
  }
  set_deferred_epilogues(held);
  return e;
}

}  // extern "C"
