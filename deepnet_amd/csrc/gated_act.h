// The activations of gated products: act(gate) * up, and their slopes.
#pragma once
#include "wide_math.h"

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
