// MX4 latent cache rows without a rotation (gfx950): the writer of un-rotated
// layers and the read-back of rows as they are stored. Both move bytes: a row
// is 2 (D + R) bytes of bf16 against D / 2 + D / 32 + 2 R in the cache, and what bounds
// them is HBM (131072 rows at D = 512: written in 41.6 us, 4.9 TB/s, read in 39.6, 5.1). Rows of
// rotated layers are written by writer_kernel and read by mx4_unrotate_kernel.
#include "mx4_codec.h"

#include <algorithm>

namespace rolaq {

constexpr int kMx4RowThreads = 256;

// A launch's blocks lie in two dimensions: one holds less than 2^32 threads, which
// 2^31 rows of up to 72 pass.
__device__ __forceinline__ int64_t mx4_row_thread() {
  return ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kMx4RowThreads + threadIdx.x;
}
dim3 mx4_row_grid(int64_t threads) {
  const int64_t blocks = (threads + kMx4RowThreads - 1) / kMx4RowThreads, x = std::min<int64_t>(blocks, 1 << 23);
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}

// A thread takes eight latent values (16 bytes in, a dword of codes out): four
// lanes make a block of 32, whose largest magnitude is a quad maximum on integer
// bits (which keeps NaN above infinity). Threads past the latent's take 16 bytes
// of rope each.
template <int D, int R>
__global__ __launch_bounds__(kMx4RowThreads) void mx4_write_kernel(Mx4RowsArgs a, int pe_vec) {
  constexpr int LAT = D / 8, PER = LAT + R / 8;  // threads of a row
  const int64_t i = mx4_row_thread();
  const int64_t nlat = a.n * LAT;
  // all latent pieces first, so that the lanes of a block lie together
  const bool lat = i < nlat;
  const int64_t row = lat ? i / LAT : (i - nlat) / (PER - LAT);
  const int c = lat ? (int)(i % LAT) : (int)((i - nlat) % (PER - LAT));
  if (row >= a.n) return;
  const int64_t slot = a.slots[row];
  const bool live = slot >= 0 && slot < a.num_slots;
  if (lat) {
    // (the lanes of a block share their row: all of them take part in the maximum)
    const u32x4 v = *reinterpret_cast<const u32x4*>(a.x + row * a.xs + 8 * c);
    uint32_t big = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t w = v[k] & 0x7fff7fffu;
      big = max(big, max(w & 0xffffu, w >> 16));
    }
    big = max(big, (uint32_t)__builtin_amdgcn_mov_dpp((int)big, 0xB1, 0xF, 0xF, true));  // quad [1, 0, 3, 2]
    big = max(big, (uint32_t)__builtin_amdgcn_mov_dpp((int)big, 0x4E, 0xF, 0xF, true));  // quad [2, 3, 0, 1]
    const uint32_t s = mx4_scale(big << 16);
    const float f = mx4_pow2(s);
    const uint32_t x0 = v[0], x1 = v[1], x2 = v[2], x3 = v[3];  // (bit casts of vector elements all take the first)
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x0), f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x1), f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x2), f, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x3), f, 3);
    if (live) {
      *reinterpret_cast<uint32_t*>(a.codes + slot * (D / 2) + 4 * c) = w;
      if (c % 4 == 0) a.scales[slot * (D / 32) + c / 4] = (uint8_t)s;
    }
  } else if (live) {
    u32x4 v;
    if (pe_vec) {
      v = *reinterpret_cast<const u32x4*>(a.k_pe + row * a.pe_s0 + 8 * c);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint16_t* const p = a.k_pe + row * a.pe_s0 + (8 * c + 2 * k) * a.pe_s1;
        v[k] = (uint32_t)p[0] | (uint32_t)p[a.pe_s1] << 16;
      }
    }
    *reinterpret_cast<u32x4*>(a.rope + slot * R + 8 * c) = v;
  }
}

// A thread takes eight values of a row: a dword of codes and a scale byte, or 16
// bytes of rope. Slots outside the cache read as NaN.
template <int D, int R>
__global__ __launch_bounds__(kMx4RowThreads) void mx4_read_kernel(Mx4RowsArgs a) {
  constexpr int PER = (D + R) / 8;
  const int64_t i = mx4_row_thread();
  const int64_t row = i / PER;
  const int c = (int)(i % PER);
  if (row >= a.n) return;
  const int64_t slot = a.slots[row];
  u32x4 v = {0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
  if (slot >= 0 && slot < a.num_slots) {
    if (c < D / 8)
      v = mx4_values8(*reinterpret_cast<const uint32_t*>(a.codes + slot * (D / 2) + 4 * c),
                      a.scales[slot * (D / 32) + c / 4]);
    else
      v = *reinterpret_cast<const u32x4*>(a.rope + slot * R + 8 * (c - D / 8));
  }
  *reinterpret_cast<u32x4*>(a.out + row * a.out_st + 8 * c) = v;
}

}  // namespace rolaq

hipError_t rolaq_launch_mx4_write_plain(const rolaq::Mx4RowsArgs& a, int D, hipStream_t stream) {
  using namespace rolaq;
  const int R = D / 8;
  const dim3 grid = mx4_row_grid(a.n * ((D + R) / 8)), block(kMx4RowThreads);
  const int pe_vec = a.pe_s1 == 1 && a.pe_s0 % 8 == 0 && reinterpret_cast<uintptr_t>(a.k_pe) % 16 == 0;
  if (D == 512)
    hipLaunchKernelGGL((mx4_write_kernel<512, 64>), grid, block, 0, stream, a, pe_vec);
  else
    hipLaunchKernelGGL((mx4_write_kernel<256, 32>), grid, block, 0, stream, a, pe_vec);
  return hipGetLastError();
}

hipError_t rolaq_launch_mx4_read(const rolaq::Mx4RowsArgs& a, int D, hipStream_t stream) {
  using namespace rolaq;
  const int R = D / 8;
  const dim3 grid = mx4_row_grid(a.n * ((D + R) / 8)), block(kMx4RowThreads);
  if (D == 512)
    hipLaunchKernelGGL((mx4_read_kernel<512, 64>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((mx4_read_kernel<256, 32>), grid, block, 0, stream, a);
  return hipGetLastError();
}
