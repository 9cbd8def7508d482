// Activations of the gated feed-forward block and their slopes, in 32 bits (gfx950).
//
//   act(g) = g s,  s = 1 / (1 + e^-z);  silu: z = g;  gelu in its tanh form: z = g (c + d g^2), c = 2 sqrt(2 / pi), d = 0.044715 c
//   act'(g) = s + g s (1 - s) z'(g)
#pragma once

#include "mfma_util.h"

namespace cm {

constexpr float kGeluC = 1.5957691216057308f, kGeluD = 0.07135481627159893f;

__device__ __forceinline__ float gate_share(float g, int activation) {
  const float z = activation == CPPMEGA_MI355_GATE_SILU ? g : g * fmaf(kGeluD, g * g, kGeluC);
  return __builtin_amdgcn_rcpf(1.0f + fast_exp2(-kLog2e * z));  // (e^-z of a far z is infinite, and its share 0)
}
__device__ __forceinline__ float gated(float g, float u, int activation) { return g * gate_share(g, activation) * u; }
// dg and du from dy; where s or 1 - s is nothing the slope is s (z' may be infinite there)
__device__ __forceinline__ void gate_grads(float g, float u, float dy, int activation, float& dg, float& du) {
  const float s = gate_share(g, activation), t = s * (1.0f - s);
  const float z = activation == CPPMEGA_MI355_GATE_SILU ? 1.0f : fmaf(3.0f * kGeluD, g * g, kGeluC);
  dg = dy * u * (t == 0.0f ? s : fmaf(g * t, z, s));
  du = dy * (g * s);
}

}  // namespace cm
