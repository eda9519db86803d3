// The activations of a gated block in binary32, act(g) and its derivative.
//
// Both are g sigmoid(2 z): silu with 2 z = g, and gelu's tanh form with z = sqrt(2 / pi) (g + 0.044715 g^3), since
// (1 + tanh z) / 2 = sigmoid(2 z).  exp2 and the reciprocal are the hardware's, 1 ulp each; the exponent's own rounding
// is 2^-24 of it, so a result is off by some 2^-20 at most where it counts (2^-17 far down the tails), against the one
// rounding to bf16, 2^-9, that follows.
#pragma once

#include "mx_common.h"

namespace mxl {

enum GateAct : int { kActSilu = 0, kActGeluTanh = 1 };

// act(g); slope: its derivative, s + g s (1 - s) d(2 z)/dg.
template <int ACT>
__device__ __forceinline__ float gate_act(float g, float& slope) {
  constexpr float kLog2E = 1.44269504088896341f;
  constexpr float kC = 1.5957691216057308f;  // 2 sqrt(2 / pi)
  const float g2 = g * g;
  const float z2 = ACT == kActSilu ? g : kC * g * __builtin_fmaf(0.044715f, g2, 1.0f);
  const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2E * z2));
  const float t = s * (1.0f - s);
  const float d = ACT == kActSilu ? 1.0f : kC * __builtin_fmaf(3.0f * 0.044715f, g2, 1.0f);
  slope = t == 0.0f ? s : __builtin_fmaf(g * t, d, s);  // (far out g^2 may be infinite where t is 0)
  return g * s;
}

}  // namespace mxl
