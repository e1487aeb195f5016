// What the MX4 kernels share: products of E2M1 with E4M3 operands on the matrix cores,
// the split of a bf16 row into two of the latter, asynchronous copies into LDS.
#pragma once

#include "rolaq_common.h"

#include <utility>

namespace rolaq {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short s16x2 __attribute__((ext_vector_type(2)));

// D = A(16x128, E2M1) * B(128x16, E4M3) + C. Lane l holds A[l%16][32(l/16)+i] (nibble
// i of four dwords) with the scale of those 32 in byte SA of sa, and
// B[16(l/16)+i][l%16], B[64+16(l/16)+i][l%16] (bytes i and 16+i) with the scale of
// B[32(l/16)..+31] in byte SB of sb.
template <int SA, int SB>
__device__ __forceinline__ f32x4 mfma_fp4_fp8(u32x4 a, i32x8 b, f32x4 c, uint32_t sa, uint32_t sb) {
  const i32x8 aa = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(aa, b, c, 4, 0, SA, (int)sa, SB, (int)sb);
}

// The same with the operands' places exchanged: A(16x128, E4M3), B(128x16, E2M1).
template <int SA, int SB>
__device__ __forceinline__ f32x4 mfma_fp8_fp4(i32x8 a, u32x4 b, f32x4 c, uint32_t sa, uint32_t sb) {
  const i32x8 bb = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, bb, c, 0, 4, SA, (int)sa, SB, (int)sb);
}

// A bf16 row of 128 KS values as two e4m3 operands, hi + lo / 16, with one power of two:
// eight significant bits are two times four, so the split is exact for values down to
// 2^-13 of the row's largest and off by less than 2^-21 of it below. Lanes la + 16 gq hold
// the row's parts v (16 values for each [s][h]) and get their bytes of hi and lo; returned are
// the scale bytes of both (hi, lo << 8; NaN for a row that is not finite).
template <int KS>
__device__ __forceinline__ uint32_t mx4_split(const u32x4 (&v)[KS][2][2], i32x8 (&hi8)[KS], i32x8 (&lo8)[KS]) {
  uint32_t big = 0;  // largest magnitude, as bits (NaN above infinity)
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = v[s][h][e][i] & 0x7fff7fffu;
          big = max(big, max(w & 0xffffu, w >> 16));
        }
  big = max(big, (uint32_t)__shfl_xor((int)big, 16));
  big = max(big, (uint32_t)__shfl_xor((int)big, 32));
  const int e = max((int)(big >> 7), 16);  // biased exponent
  // scaled so that the largest lies in [2^7, 2^8); lo is 2^4 finer
  const float fh = __uint_as_float((uint32_t)(e - 7) << 23), fl = __uint_as_float((uint32_t)(e - 11) << 23);
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int d = 0; d < 4; ++d) {  // dword d: values 4 d .. 4 d + 3 of 16
        const uint32_t w0 = v[s][h][d >> 1][2 * (d & 1)], w1 = v[s][h][d >> 1][2 * (d & 1) + 1];
        s16x2 p = {0, 0}, q = {0, 0};
        p = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(p, __builtin_bit_cast(bf16x2_t, w0), fh, false);
        p = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(p, __builtin_bit_cast(bf16x2_t, w1), fh, true);
        const int hi = __builtin_bit_cast(int, p);
        const f32x2 b0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, fh, false);
        const f32x2 b1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, fh, true);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(q, bf16_lo(w0) - b0.x, bf16_hi(w0) - b0.y, fl, false);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(q, bf16_lo(w1) - b1.x, bf16_hi(w1) - b1.y, fl, true);
        hi8[s][4 * h + d] = hi;
        lo8[s][4 * h + d] = __builtin_bit_cast(int, q);
      }
  return e >= 255 ? 0xffffu : (uint32_t)(e - 7) | (uint32_t)(e - 11) << 8;
}

// Asynchronous copies into LDS, 16 or 4 bytes for each lane, lane l's to
// lds + 16 l (4 l). In assembly because the compiler, which tracks such copies,
// would wait for all of them before any LDS read; the kernel waits by count.
__device__ __forceinline__ void copy16(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void copy4(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(src) : "memory", "m0");
}

// The same from a scalar base and a 32-bit offset for each lane.
__device__ __forceinline__ void copy16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}
__device__ __forceinline__ void copy4(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base)
               : "memory", "m0");
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

template <typename F, int... I>
__device__ __forceinline__ void for_each_of(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  for_each_of(f, std::make_integer_sequence<int, N>{});
}

}  // namespace rolaq
