// The activations of a gated block in binary32, act(g) and its derivative.
//
// Both are g sigmoid(2 z): silu with 2 z = g, and gelu's tanh form with z = sqrt(2 / pi) (g + 0.044715 g^3), since
// (1 + tanh z) / 2 = sigmoid(2 z).  exp2 and the reciprocal are the hardware's, 1 ulp each, and the exponent's own rounding
// is 2^-24 of it.  Against 64 bits over 4.5 million gates, both operations off by an ulp to either side: values are off by
// 2^-21 of themselves (silu) and 2^-19 (gelu, whose 2 z is a sum of products) at |g| < 4, by 2^-19.8 and 2^-18.5 as long as
// they are above 2^-20; slopes by 2^-21.6 absolute, of some 1 at most (with 1 - s subtracted it was 2^-18, as g d reaches
// 35 where s is next to 1).  The one rounding to bf16 that follows takes up to 2^-8 of a value.
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
  const float e = __builtin_amdgcn_exp2f(-kLog2E * z2), s = __builtin_amdgcn_rcpf(1.0f + e);
  const float t = s * (e * s);  // s (1 - s) without the difference
  const float d = ACT == kActSilu ? 1.0f : kC * __builtin_fmaf(3.0f * 0.044715f, g2, 1.0f);
  slope = t > 0.0f ? __builtin_fmaf(g * t, d, s) : s;  // (far out e or g^2 may be infinite, where t is 0 or NaN)
  return g * s;
}

}  // namespace mxl
