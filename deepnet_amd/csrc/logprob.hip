// Log probabilities of given tokens, entropies and the best alternatives of columns of logits, and their gradient (no
// counterpart in cudamat.cu; softmax_ce_grad is the loss of a classifier, which stores its probabilities).
#include "common.h"
#include "wide_math.h"
#include <float.h>

// e^t for t <= 0: t log2(e) in two terms, the hardware's exp2, a correction.  -inf gives 0, NaN stays NaN.
__device__ __forceinline__ float lp_exp(float t) {
  t = t < -128.f ? -128.f : t;      // (e^-128 is 0 in fp32; keeps -inf out of the correction)
  const float L2E = 1.44269502162933349609375f, L2E_LO = 1.925963033500011e-08f;
  const float p = t * L2E;
  const float lo = __fmaf_rn(t, L2E_LO, __fmaf_rn(t, L2E, -p));
  const float e = __builtin_amdgcn_exp2f(p);
  return __fmaf_rn(e, lo * 0.693147182464599609375f, e);
}

// Orders entries: the greater value first, of equal ones (0 and -0 are) the one further up; NaN ranks with -inf.
__device__ __forceinline__ unsigned long long lp_key(float x, int i) {
  x = x != x ? -INFINITY : x + 0.f;
  const unsigned u = __float_as_uint(x), v = u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
  return ((unsigned long long)v << 32) | (unsigned)~i;
}
__device__ __forceinline__ int lp_key_index(unsigned long long k) { return (int)~(unsigned)k; }

__device__ __forceinline__ unsigned long long block_max_key(unsigned long long k, unsigned long long* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor(k, o, WAVE);
    k = other > k ? other : k;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = k;
  __syncthreads();
  for (int i = 0; i < 4; ++i) k = red[i] > k ? red[i] : k;
  return k;
}
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// log(1 + r), r >= 0 (NaN stays NaN); 1 + r itself would round a small r away.
__device__ __forceinline__ double lp_log1p(float r) {
  const double u = (double)r;
  return u >= 1e-5 ? dn_log_wide_pos(1.0 + u) : u * fma(u, fma(u, 1.0 / 3.0, -0.5), 1.0);
}

struct LogProbArgs {
  const float *mat, *labels;
  float *logp, *entropy, *log_z, *top, *top_labels;
  int h, k;
};

// With m the maximum and r the sum of e^(x - m) over the others: log_z = m + log(1 + r), to full precision however small r
// is; entropy = log(1 + r) - sum (x - m) e^(x - m) / (1 + r).
__global__ void __launch_bounds__(256) k_log_probs(LogProbArgs a) {
  __shared__ unsigned long long kred[4];
  __shared__ float red[4];
  const int h = a.h, col = blockIdx.x;
  const float* c = a.mat + (size_t)col * h;
  unsigned long long best = 0;
  for (int i = threadIdx.x; i < h; i += 256) {
    const unsigned long long k = lp_key(c[i], i);
    best = k > best ? k : best;
  }
  best = block_max_key(best, kred);
  const int first = lp_key_index(best);
  const float m = c[first];
  float r = 0.f, t = 0.f;
  bool nan = false;
  for (int i = threadIdx.x; i < h; i += 256) {
    const float d = c[i] - m, e = i == first ? 0.f : lp_exp(d);
    nan |= c[i] != c[i];
    r += e;
    t += e > 0.f ? d * e : 0.f;
  }
  r = block_sum(nan ? NAN : r, red);
  t = block_sum(t, red);
  const bool none = m == -INFINITY && r != r && block_max_key(nan, kred) == 0;      // every entry is -inf
  const double lz = lp_log1p(r);
  float log_z = none ? -INFINITY : m < INFINITY && r == r ? (float)((double)m + lz) : NAN;
  if (threadIdx.x == 0) {
    if (a.log_z) a.log_z[col] = log_z;
    if (a.entropy) a.entropy[col] = none ? 0.f : log_z != log_z ? NAN : (float)(lz - (double)t / (1.0 + (double)r));
    if (a.logp) {
      const float l = a.labels[col];
      const bool token = l >= 0.f && l < (float)h;
      a.logp[col] = !token ? 0.f : none ? -INFINITY : log_z != log_z ? NAN : (float)((double)c[(int)l] - (double)m - lz);
    }
  }
  for (int j = 0; j < a.k; ++j) {
    if (threadIdx.x == 0) {
      const int i = lp_key_index(best);
      if (a.top) a.top[(size_t)col * a.k + j] = none ? -INFINITY : log_z != log_z ? NAN : (float)((double)c[i] - (double)m - lz);
      if (a.top_labels) a.top_labels[(size_t)col * a.k + j] = (float)i;
    }
    unsigned long long next = 0;
    for (int i = threadIdx.x; i < h; i += 256) {
      const unsigned long long k = lp_key(c[i], i);
      next = k < best && k > next ? k : next;
    }
    best = block_max_key(next, kred);
  }
}

// target = logp_weight (onehot(label) - p) - entropy_weight p (log p + entropy), log p = mat - log_z: one pass.
__global__ void __launch_bounds__(256)
k_log_probs_grad(const float* mat, const float* labels, const float* log_z, const float* logp_weight, const float* entropy,
                 const float* entropy_weight, float* target, int h) {
  const int col = blockIdx.x;
  const float z = log_z[col], l = labels ? labels[col] : -1.f;
  const bool token = l >= 0.f && l < (float)h;
  const int label = token ? (int)l : -1;
  const float lw = token ? (logp_weight ? logp_weight[col] : 1.f) : 0.f;
  const float ew = entropy_weight ? entropy_weight[col] : 0.f, ent = entropy ? entropy[col] : 0.f;
  const float* c = mat + (size_t)col * h;
  float* t = target + (size_t)col * h;
  for (int i = threadIdx.x; i < h; i += 256) {
    const float x = c[i], lp = x - z;
    const float p = x == -INFINITY ? 0.f : lp_exp(lp);
    const float q = p > 0.f || p != p ? p * (lp + ent) : 0.f;
    t[i] = lw * ((i == label ? 1.f : 0.f) - p) - ew * q;
  }
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
#define DPTR(m) ((m) ? (m)->data_device : nullptr)

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
  if (h <= 0 || w <= 0) return 0;
  hipLaunchKernelGGL(k_log_probs, dim3((unsigned)w), dim3(256), 0, dn_stream(),
                     LogProbArgs{mat->data_device, DPTR(labels), DPTR(logp), DPTR(entropy), DPTR(log_z), DPTR(top), DPTR(top_labels), h, k});
  return dn_launch_status();
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
  hipLaunchKernelGGL(k_log_probs_grad, dim3((unsigned)w), dim3(256), 0, dn_stream(), (const float*)mat->data_device, (const float*)DPTR(labels),
                     (const float*)log_z->data_device, (const float*)DPTR(logp_weight), (const float*)DPTR(entropy), (const float*)DPTR(entropy_weight),
                     target->data_device, h);
  return dn_launch_status();
}

}  // extern "C"
