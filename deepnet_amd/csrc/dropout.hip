// Dropout by a counter-based generator (no counterpart in cudamat.cu, whose dropout draws from 12288 streams that go on):
// whether an entry is dropped is a function of its place, a step, a stream and a seed, so the backward pass is the same
// call on the derivative and no mask is stored.
#include "common.h"
#include <math.h>

// Philox4x32-10 (J. K. Salmon, M. A. Moraes, R. O. Dror, D. E. Shaw: Parallel random numbers: as easy as 1, 2, 3, SC 2011):
// four words from a counter of four words and a key of two.
struct PhiloxKey { uint32_t k0, k1; };
__device__ __forceinline__ void philox10(uint32_t (&c)[4], PhiloxKey k) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c[0], b = (uint64_t)0xCD9E8D57u * c[2];
    const uint32_t x = (uint32_t)(b >> 32) ^ c[1] ^ k.k0, y = (uint32_t)(a >> 32) ^ c[3] ^ k.k1;
    c[0] = x; c[1] = (uint32_t)b; c[2] = y; c[3] = (uint32_t)a;
    k.k0 += 0x9E3779B9u; k.k1 += 0xBB67AE85u;
  }
}

// Entry i of the matrix (column-major) is dropped when word i % 4 of counter (i / 4, i / 4 >> 32, bits of the step,
// stream) is below border.  target may be mat or residual.
__global__ void __launch_bounds__(256)
k_counter_dropout(const float* mat, const float* residual, float* target, const float* step, long long n, uint64_t border, float mult,
                  uint32_t stream, PhiloxKey key) {
  const long long g = (long long)blockIdx.x * 256 + threadIdx.x;
  if (4 * g >= n) return;
  uint32_t c[4] = {(uint32_t)g, (uint32_t)(g >> 32), step ? __float_as_uint(*step) : 0u, stream};
  philox10(c, key);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const long long i = 4 * g + j;
    if (i < n) {
      const float x = c[j] >= border ? mat[i] : 0.f;
      target[i] = residual ? __fmaf_rn(mult, x, residual[i]) : mult * x;
    }
  }
}

static inline bool same_or_apart(const cudamat* a, const cudamat* b) {
  return a->data_device == b->data_device || a->data_device + dn_len(a) <= b->data_device || b->data_device + dn_len(b) <= a->data_device;
}

extern "C" int counter_dropout(cudamat* mat, cudamat* residual, cudamat* target, cudamat* step, float dropprob, float mult,
                               unsigned seed_lo, unsigned seed_hi, unsigned stream) {
  if (!mat->on_device || !target->on_device || (residual && !residual->on_device) || (step && !step->on_device)) return ERROR_NOT_ON_DEVICE;
  if (mat->is_trans || target->is_trans || (residual && residual->is_trans)) return ERROR_TRANSPOSED;
  if (target->size[0] != mat->size[0] || target->size[1] != mat->size[1] ||
      (residual && (residual->size[0] != mat->size[0] || residual->size[1] != mat->size[1])) ||
      (step && (step->size[0] != 1 || step->size[1] != 1)))
    return ERROR_INCOMPATIBLE_DIMENSIONS;
  if (!(dropprob >= 0.f && dropprob <= 1.f) || !same_or_apart(mat, target) || (residual && !same_or_apart(residual, target)) ||
      (step && step->data_device >= target->data_device && step->data_device < target->data_device + dn_len(target)))
    return ERROR_UNSUPPORTED;
  const long long n = dn_len(mat);
  if (n <= 0) return 0;
  const long long blocks = ((n + 3) / 4 + 255) / 256;
  if (blocks > 0x7fffffffll) return ERROR_UNSUPPORTED;
  hipLaunchKernelGGL(k_counter_dropout, dim3((unsigned)blocks), dim3(256), 0, dn_stream(), (const float*)mat->data_device,
                     (const float*)(residual ? residual->data_device : nullptr), target->data_device,
                     (const float*)(step ? step->data_device : nullptr), n, (uint64_t)((double)dropprob * 4294967296.0), mult, stream,
                     PhiloxKey{seed_lo, seed_hi});
  return dn_launch_status();
}
