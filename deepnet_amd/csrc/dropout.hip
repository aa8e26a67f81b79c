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
// stream) is below border; a launch begins at counter `first`.  target may be mat or residual.  A lane has one counter and its four entries, 16 bytes at any 4-byte
// boundary that are on their way while the generator runs.  Bound by the bytes: 4096 x 8192 onto a residual 62.4 us, 6.46 TB/s, what a
// copy reaches; 42.3 us without, 4097 x 4097 32.1.  Two, four, eight counters a lane: 64.0, 66.9, 68.7 us.  The generator is hidden: with
// seven of its rounds instead of ten, four counters a lane take 66.4.
struct __attribute__((packed, aligned(4))) DropGroup { float x, y, z, w; };
template <bool RES, bool STREAM>
__global__ void __launch_bounds__(256)
k_counter_dropout(const float* mat, const float* residual, float* target, const float* step, long long first, long long n, uint64_t border,
                  float mult, uint32_t stream, PhiloxKey key) {
  const long long g = first + (long long)blockIdx.x * 256 + threadIdx.x, whole = n >> 2;
  if (4 * g >= n) return;
  auto load = [](float (&v)[4], const float* p) __attribute__((always_inline)) {
    if (STREAM) { const float4 q = dn_ld4<true>(p); v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w; }
    else { const DropGroup q = *reinterpret_cast<const DropGroup*>(p); v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w; }
  };
  auto one = [&](float x, float r, uint32_t word) __attribute__((always_inline)) {
    return word >= border ? (RES ? __fmaf_rn(mult, x, r) : mult * x) : (RES ? r : 0.f);
  };
  float x[4], r[4] = {0.f, 0.f, 0.f, 0.f};
  if (g < whole) {
    load(x, mat + 4 * g);
    if (RES) load(r, residual + 4 * g);
  }
  uint32_t c[4] = {(uint32_t)g, (uint32_t)(g >> 32), step ? __float_as_uint(*step) : 0u, stream};
  philox10(c, key);
  if (g < whole) {
    const float y[4] = {one(x[0], r[0], c[0]), one(x[1], r[1], c[1]), one(x[2], r[2], c[2]), one(x[3], r[3], c[3])};
    if (STREAM) dn_st4<true>(target + 4 * g, make_float4(y[0], y[1], y[2], y[3]));
    else *reinterpret_cast<DropGroup*>(target + 4 * g) = DropGroup{y[0], y[1], y[2], y[3]};
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (4 * g + j < n) target[4 * g + j] = one(mat[4 * g + j], RES ? residual[4 * g + j] : 0.f, c[j]);
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
  const float *x = mat->data_device, *r = residual ? residual->data_device : nullptr, *s = step ? step->data_device : nullptr;
  float* t = target->data_device;
  const bool wide = n >= DN_STREAM_MIN_ELEMS && dn_aligned16(x) && dn_aligned16(t) && dn_aligned16(r);
  const uint64_t border = (uint64_t)((double)dropprob * 4294967296.0);
  const long long counters = (n + 3) / 4;
  for (long long first = 0; first < counters; first += 256 * DN_MAX_GROUPS) {
    const long long blocks = (counters - first + 255) / 256;
    const dim3 grid((unsigned)(blocks < DN_MAX_GROUPS ? blocks : DN_MAX_GROUPS));
#define DROP_GO(R, S) hipLaunchKernelGGL((k_counter_dropout<R, S>), grid, dim3(256), 0, dn_stream(), x, r, t, s, first, n, border, mult, stream, PhiloxKey{seed_lo, seed_hi})
    if (r) { if (wide) DROP_GO(true, true); else DROP_GO(true, false); }
    else if (wide) DROP_GO(false, true);
    else DROP_GO(false, false);
  }
#undef DROP_GO
  return dn_launch_status();
}
