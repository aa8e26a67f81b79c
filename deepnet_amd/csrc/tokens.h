// What the operators on tokens check of their arguments, and the order of logits.
#pragma once
#include "common.h"
#include <math.h>

// Whether no entry is in both; one that is not there (NULL) is apart from everything.
static inline bool tok_apart(const cudamat* a, const cudamat* b) {
  return !a || !b || a->data_device + dn_len(a) <= b->data_device || b->data_device + dn_len(b) <= a->data_device;
}
static inline bool tok_same_or_apart(const cudamat* a, const cudamat* b) {
  return tok_apart(a, b) || (a->data_device == b->data_device && a->size[0] == b->size[0] && a->size[1] == b->size[1]);
}
// Of optional matrices (NULL where they are not given): on the device and not transposed; and their shape.
template <int N>
static inline int tok_check_device(cudamat* const (&m)[N]) {
  for (const cudamat* x : m)
    if (x && !x->on_device) return ERROR_NOT_ON_DEVICE;
  for (const cudamat* x : m)
    if (x && x->is_trans) return ERROR_TRANSPOSED;
  return 0;
}
static inline bool tok_shape(const cudamat* m, int rows, int cols) { return !m || (m->size[0] == rows && m->size[1] == cols); }
static inline float* tok_data(const cudamat* m) { return m ? m->data_device : nullptr; }

// The token of a label, -1 for no token (outside [0, n), NaN).
__device__ __forceinline__ int tok_label(float l, int n) { return l >= 0.f && l < (float)n ? (int)l : -1; }

// Orders entries: the greater value first, of equal ones (0 and -0 are) the one further up; NaN ranks with -inf.
__device__ __forceinline__ unsigned long long lp_key(float x, int i) {
  x = x != x ? -INFINITY : x + 0.f;
  const unsigned u = __float_as_uint(x), v = u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
  return ((unsigned long long)v << 32) | (unsigned)~i;
}
__device__ __forceinline__ int lp_key_index(unsigned long long k) { return (int)~(unsigned)k; }
__device__ __forceinline__ float lp_key_value(unsigned long long key) {
  const unsigned v = (unsigned)(key >> 32);
  return __uint_as_float(v ^ ((v >> 31) ? 0x80000000u : 0xffffffffu));
}
