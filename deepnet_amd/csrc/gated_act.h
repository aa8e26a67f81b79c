// The activations of gated products: act(gate) * up, and their slopes.
#pragma once
#include "wide_math.h"

enum { GATE_LINEAR = 0, GATE_SIGMOID = 1, GATE_RELU = 2, GATE_TANH = 3, GATE_SILU = 4, GATE_GELU = 5 };

// The share of a normal variable below g; erfc keeps the digits of the small ones.
__device__ __forceinline__ float gate_phi(float g) { return 0.5f * erfcf(g * -0.70710678118654752440f); }

// 1 / (1 + e^-g), and with the other sign: e^-|g| by the hardware's exp2 of a fraction (with the rounding of the product and of the
// constant added) and an exact scaling, 1 / (1 + e) by its estimate and a Newton step, e / (1 + e).  Each about 2 ulp, results below the
// normal range too.
__device__ __forceinline__ float gate_sigmoid(float g, float* other) {
#pragma clang fp contract(off)      // (`low` is what the rounding of p left)
  const float L2E = 1.44269502162933349609375f, t = -fminf(fabsf(g), 120.f), p = t * L2E, n = rintf(p);
  const float low = __fmaf_rn(t, 1.925963033500011e-08f, __fmaf_rn(t, L2E, -p));
  const float e = ldexpf(__builtin_amdgcn_exp2f((p - n) + low), (int)n), d = 1.f + e;
  float r = __builtin_amdgcn_rcpf(d);
  r = __fmaf_rn(r, __fmaf_rn(-d, r, 1.f), r);
  const float q = e * r;
  if (g != g) { *other = g; return g; }
  *other = g > 0.f ? q : r;
  return g > 0.f ? r : q;
}

__device__ __forceinline__ float gate_act(float g, int act) {
  float other;
  switch (act) {
    case GATE_SIGMOID: return gate_sigmoid(g, &other);
    case GATE_RELU: return g < 0.f ? 0.f : g;
    case GATE_TANH: return dn_tanh(g);
    case GATE_SILU: return g * gate_sigmoid(g, &other);
    case GATE_GELU: return g * gate_phi(g);
    default: return g;
  }
}
// The activation and its slope.
__device__ __forceinline__ float gate_act_slope(float g, int act, float* slope) {
  float other;
  switch (act) {
    case GATE_SIGMOID: { const float s = gate_sigmoid(g, &other); *slope = s * other; return s; }
    case GATE_RELU: *slope = g > 0.f ? 1.f : 0.f; return g < 0.f ? 0.f : g;
    case GATE_TANH: { const float s = dn_tanh(g); *slope = (1.f - s) * (1.f + s); return s; }
    case GATE_SILU: { const float s = gate_sigmoid(g, &other), v = g * s; *slope = __fmaf_rn(v, other, s); return v; }
    case GATE_GELU: { const float p = gate_phi(g); *slope = __fmaf_rn(g * 0.39894228040143267794f, dn_exp(-0.5f * g * g), p); return g * p; }
    default: *slope = 1.f; return g;
  }
}

// What a gated product leaves: row i of the halves at column c is pre[2 f c + i] and pre[2 f c + f + i] (pre may be null), the result
// target[f c + i].  bias: 2 f, or null.
struct GatedOut {
  const float* bias;
  float *target, *pre;
  int f, act;
};
__device__ __forceinline__ void gated_out(const GatedOut& o, int i, int c, float g, float u) {
  if (o.bias) { g += o.bias[i]; u += o.bias[o.f + i]; }
  if (o.pre) {
    float* p = o.pre + 2 * (size_t)c * o.f + i;
    p[0] = g;
    p[o.f] = u;
  }
  o.target[(size_t)c * o.f + i] = gate_act(g, o.act) * u;
}
