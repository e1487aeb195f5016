// The MX4 codec: blocks of 32 values as E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
// their negatives; element e at nibble e of 16 bytes) and one power of two.
#pragma once

#include "mx4_args.h"
#include "rolaq_common.h"

namespace rolaq {

// Scale byte of a block whose largest magnitude has the bits `big`: 2^(s - 127) is
// the least power of two under which it is below 7, so that no value is off by
// more than half a step (6 is the largest code, and [6, 7) is within half of the
// step that would follow it). At least 2^-64; a block that is not finite, or
// would need more than 2^32, is NaN.
__device__ __forceinline__ uint32_t mx4_scale(uint32_t big) {
  const int s = (int)((big + 0x00200000u) >> 23) - 2;  // 1.75 2^k and more count as 2^(k + 1)
  return s > kMx4High ? kMx4NaN : (uint32_t)max(s, kMx4Low);
}

// 2^(s - 127) as a float, the scale operand of the conversions (which read its exponent).
__device__ __forceinline__ float mx4_pow2(uint32_t s) { return __uint_as_float(s << 23); }

// Eight fp32 values -> eight codes at the scale f (round to nearest even, up to 6).
__device__ __forceinline__ uint32_t mx4_codes8(f32x4 u, f32x4 v, float f) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, u[0], u[1], f, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, u[2], u[3], f, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], f, 3);
}

// Eight codes -> eight bf16 values at the scale byte s (exact).
__device__ __forceinline__ u32x4 mx4_values8(uint32_t w, uint32_t s) {
  if (s == (uint32_t)kMx4NaN) return u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
  const float f = mx4_pow2(s);
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 3))};
}

}  // namespace rolaq
