// MXFP4 (E2M1 codes, one E8M0 scale per 32) on gfx950: the quantization that the quantizer, the
// SwiGLU producer and the GEMM's own wavefronts share.
//
// E2M1 holds 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives (bit 3 the sign), two codes per byte, the
// even column in the low half.  A block's scale is the power of two that brings its largest magnitude
// between 4 and 8 (exponent - 2); of what then lies past 7, rule floor_carry175 (kFloorCarry175) doubles
// the scale -- from 1.75 2^e on, the first bf16 amax that rounds past 6 -- and rule floor (kFloorOcp,
// OCP MX v1.0 section 6.3) saturates it at 6.  E2M1 has no infinity or NaN: a block that holds one
// takes the NaN scale (255) and zero codes, so that whatever is computed from it is NaN.
#pragma once

#include "mx_common.h"

namespace mxl {

// The E8M0 code of a block from the bf16 magnitude bits of its amax (a NaN's above infinity's).  carry: 32
// (floor_carry175) or 0 (floor): bf16 keeps seven mantissa bits, so +32, a quarter, carries into the exponent from
// 1.75 on.
__device__ __forceinline__ uint32_t scale_e2m1(uint32_t amax, uint32_t carry) {
  const uint32_t e = (amax + carry) >> 7;
  return amax >= 0x7F80u ? 255u : e > 2u ? e - 2u : 0u;
}
inline bool fp4_rule(int rule) { return rule == kFloorCarry175 || rule == kFloorOcp; }
inline uint32_t fp4_carry(int rule) { return rule == kFloorCarry175 ? 32u : 0u; }

// Eight raw bf16 values (four pairs) -> eight E2M1 codes divided by 2^(s - 127), one dword:
// v_cvt_scalef32_pk_fp4_bf16 divides by the power of two that its scale operand's exponent field
// names and rounds once, to the nearest even, saturating at 6 (equal to the plain arithmetic for every
// bf16 value under every scale of its own block).  s = 255: zero codes.
__device__ __forceinline__ uint32_t codes_e2m1(const uint32_t* d, uint32_t s) {
  const float scale = u2f(s << 23);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, d[0]), scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, d[1]), scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, d[2]), scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, d[3]), scale, 3);
  return s == 255u ? 0u : c;
}

// A block of 32 held by four consecutive lanes, eight values each: its E8M0 code (in every lane) and
// the lane's codes.
__device__ __forceinline__ uint32_t quant_e2m1_x4(const uint32_t* d, uint32_t carry, uint32_t& codes) {
  uint32_t amax = amax_bf16_bits<4, false>(d);
  amax = __builtin_elementwise_max(amax, (uint32_t)__shfl_xor((int)amax, 1, 4));
  amax = __builtin_elementwise_max(amax, (uint32_t)__shfl_xor((int)amax, 2, 4));
  const uint32_t s = scale_e2m1(amax, carry);
  codes = codes_e2m1(d, s);
  return s;
}

}  // namespace mxl
