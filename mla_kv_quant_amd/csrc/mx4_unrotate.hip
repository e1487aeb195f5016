// MX4 cache rows back in the model's frame (gfx950): out = [X R_eff^T, rope] for gathered
// slots, X the stored rows (4-bit codes times 2^e for each 32), R_eff [D, D] bf16.
//
// The codes are an operand of v_mfma_scale_f32_16x16x128_f8f6f4 as they are, with the
// block scales as its scales; R_eff's rows are the other one, split exactly into two e4m3
// parts (mx4_split). So nothing is expanded, a row is D / 2 + D / 32 bytes of LDS, and
// R_eff can stay in registers for a block's life: a wave holds 16 NT of its rows (64 D NT
// bytes a wave, 128 registers at D = 512 and NT = 2) and walks 64-row tiles of X, which
// asynchronous copies bring to LDS a tile ahead.
//
// Two shapes. With many rows a block of eight waves covers 256 columns (half of D = 512,
// the other half's block on the same XCD), one block for each CU; what bounds it is R_eff's
// way in (18 us), then for each 64 rows 3.4 us between the stores (1.1) and the
// matrix instructions (D^2 products a row, twice, 1.7 us): 131072 rows at D = 512 in 71 us,
// 2.9 TB/s and 970 TFLOP/s. With few rows, where a wave's loads of R_eff are what takes
// time, a block is a wave of 16 columns: 8 rows in 5.2 us.
#include "mx4_codec.h"
#include "mx4_tile.h"

#include <algorithm>

namespace rolaq {

constexpr int kMx4BackRows = 64;  // rows of a tile

template <int D, int WV, int NT>
__global__ __launch_bounds__(64 * WV) void mx4_unrotate_kernel(Mx4RowsArgs a, int parts_of_rows) {
  constexpr int R = D / 8, NB = D / 32, KS = D / 128, CB = D / 2, T = kMx4BackRows;
  constexpr int SPLIT = D / (16 * NT * WV);  // blocks that share a row's columns
  constexpr int CT = T / WV;                 // rows that a wave copies
  constexpr int RC = 1024 / CB, LC = 64 / RC, LS = NB / 4;
  constexpr int NC = CT / RC;                    // its copies of codes
  constexpr int NSC = (CT * LS + 63) / 64;       // and of scales
  constexpr int NPE = (CT * R / 8 + 63) / 64;    // and its pieces of rope, 16 bytes a lane
  constexpr int TILE = T * CB + WV * NSC * 256;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2 * TILE];
  __shared__ int32_t s_slot[2][T];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  const int tid = threadIdx.x, lane = tid & 63, la = lane & 15, gq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // the column blocks of one part of the rows on one XCD (blocks go round the XCDs in turn)
  const int part = blockIdx.x / 8 % SPLIT, j = blockIdx.x / 8 / SPLIT * 8 + blockIdx.x % 8;
  const int64_t tiles = (a.n + T - 1) / T;
  const int k0 = __builtin_amdgcn_readfirstlane((int)(tiles * j / parts_of_rows));
  const int k1 = __builtin_amdgcn_readfirstlane((int)(tiles * (j + 1) / parts_of_rows));
  if (j >= parts_of_rows || k0 >= k1) return;

  // ---- copies: slots two tiles ahead, codes, scales and rope one tile ahead -------------
  // chunk c of row t goes to chunk c ^ f(t): 16 lanes that read one chunk of 16 rows meet all banks
  auto swz = [](int t) { return D == 512 ? t & 15 : (t >> 1) & 7; };
  auto load_slot = [&](int k) {  // slot of row lane % CT of this wave's
    return a.slots[min((int64_t)k * T + CT * wave + lane % CT, a.n - 1)];
  };
  u32x4 pe[NPE];
  auto mine = [&](int k) { return SPLIT == 1 || k % SPLIT == part; };  // (whose rope is stored here)
  auto ask = [&](int k, int64_t slot64) __attribute__((always_inline)) {
    const int slot = slot64 >= 0 && slot64 < a.num_slots ? (int)slot64 : -1;  // -1: outside the cache
    const uint32_t at = lds0 + (uint32_t)(k & 1) * TILE;
    if (lane < CT) s_slot[k & 1][CT * wave + lane] = slot;
    const int s0 = max(slot, 0);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int t = RC * i + lane / LC;
      const int64_t sl = __shfl(s0, t);
      copy16(a.codes + sl * CB + 16 * ((lane % LC) ^ swz(CT * wave + t)), at + wave * CT * CB + 1024 * i);
    }
#pragma unroll
    for (int i = 0; i < NSC; ++i) {
      const int t = (64 / LS * i + lane / LS) % CT;
      const int64_t sl = __shfl(s0, t);
      copy4(a.scales + sl * NB + 4 * (lane % LS), at + T * CB + (wave * NSC + i) * 256);
    }
    if (mine(k)) {
#pragma unroll
      for (int i = 0; i < NPE; ++i) {
        const int t = (64 / (R / 8) * i + lane / (R / 8)) % CT;
        const int64_t sl = __shfl(slot, t);
        pe[i] = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
        if (sl >= 0) pe[i] = gload<u32x4>(a.rope + sl * R + 8 * (lane % (R / 8)));
      }
    }
  };
  auto store_rope = [&](int k) {
#pragma unroll
    for (int i = 0; i < NPE; ++i) {
      const int t = 64 / (R / 8) * i + lane / (R / 8);
      const int64_t row = (int64_t)k * T + CT * wave + t;
      if (t < CT && row < a.n) *reinterpret_cast<u32x4*>(a.out + row * a.out_st + D + 8 * (lane % (R / 8))) = pe[i];
    }
  };
  int64_t slot = load_slot(k0);

  // ---- this wave's rows of R_eff ---------------------------------------------------------
  // Row m of its tile nt is column c0 + 8 (m / 4) + 4 nt + m % 4 of out (NT = 2), so that a
  // lane's results, rows 4 gq .. + 3 of each tile, are 8 columns in a row.
  const int c0 = 16 * NT * (WV * part + wave);
  i32x8 hi[NT][KS], lo[NT][KS];
  uint32_t rscale[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int col = NT == 2 ? c0 + 8 * (la >> 2) + 4 * nt + (la & 3) : c0 + la;
    u32x4 v[KS][2][2];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // K index 64 h + 16 gq + i of step s is feature 32 (KS kb + s) + 16 (gq & 1) + i, kb = 2 h + gq / 2
        const uint16_t* const p = a.rot + (int64_t)col * D + 32 * (KS * (2 * h + (gq >> 1)) + s) + 16 * (gq & 1);
        v[s][h][0] = gload<u32x4>(p);
        v[s][h][1] = gload<u32x4>(p + 8);
      }
    if (nt == 0) ask(k0, slot);  // (the first tile behind the first loads of R_eff)
    rscale[nt] = mx4_split<KS>(v, hi[nt], lo[nt]);
  }
  slot = load_slot(min(k0 + 1, k1 - 1));

  // ---- the tiles: turn k has tile k + 1's copies, tile k - 1's stores, tile k's products ----
  constexpr int STORES = T / 16;
  u32x2 res[STORES][NT];
  auto store = [&](int k, bool last) __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < STORES; ++m) {
      const int64_t row = (int64_t)k * T + 16 * m + la;
      if (last && row >= a.n) continue;
      uint16_t* const p = a.out + row * a.out_st + c0;
      if constexpr (NT == 2)
        *reinterpret_cast<u32x4*>(p + 8 * gq) = u32x4{res[m][0].x, res[m][0].y, res[m][1].x, res[m][1].y};
      else
        *reinterpret_cast<u32x2*>(p + 4 * gq) = res[m][0];
    }
  };
  auto turn = [&](int k, auto first) __attribute__((always_inline)) {
    // Tile k is in, and all reads of the other buffer are done. In flight here, the oldest
    // first, are tile k's copies (two or one of codes, one of scales), its rope if it is
    // stored here, the next slots; and behind them, from a block's third turn on, the
    // stores of the turn before, all STORES of them (only a part's last tile can
    // end early): these may go on. The first two turns have none behind their copies: the
    // first waits for everything here, the second where the loop begins.
    wait_loads<first ? 0 : STORES>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (mine(k)) store_rope(k);
    if (k + 1 < k1) {
      ask(k + 1, slot);
      slot = load_slot(min(k + 2, k1 - 1));
    }
    asm volatile("" ::: "memory");
    if (!first) store(k - 1, false);
    asm volatile("" ::: "memory");
    const uint8_t* const tile = smem + (k & 1) * TILE;
#pragma unroll
    for (int m = 0; m < T / 16; ++m) {
      const int t = 16 * m + la;
      const uint8_t* const sp = tile + T * CB + t / CT * (NSC * 256) + t % CT * NB + gq * KS;
      uint32_t sx = KS == 4 ? *reinterpret_cast<const uint32_t*>(sp) : *reinterpret_cast<const uint16_t*>(sp);
      if (s_slot[k & 1][t] < 0) sx = 0xffffffffu;  // (outside the cache: NaN)
      f32x4 acc[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) acc[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
      static_for<KS>([&](auto s) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(tile + t * CB + 16 * ((gq * KS + s) ^ swz(t)));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[nt] = mfma_fp8_fp4<0, s>(hi[nt][s], x, acc[nt], rscale[nt], sx);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[nt] = mfma_fp8_fp4<1, s>(lo[nt][s], x, acc[nt], rscale[nt], sx);
      });
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        res[m][nt] = u32x2{pack_bf16(acc[nt][0], acc[nt][1]), pack_bf16(acc[nt][2], acc[nt][3])};
    }
  };
  turn(k0, std::true_type{});
  wait_loads<0>();  // (tile k0 + 1's copies, with no stores behind them to count)
#pragma unroll 1
  for (int k = k0 + 1; k < k1; ++k) turn(k, std::false_type{});
  store(k1 - 1, true);
}

template <int D>
hipError_t launch_unrotate(const Mx4RowsArgs& a, int num_cus, hipStream_t stream) {
  const int64_t tiles = (a.n + kMx4BackRows - 1) / kMx4BackRows;
  const auto up8 = [](int64_t x) { return (x + 7) / 8 * 8; };
  // Few rows (4096 at D = 512, 8192 at 256 on 256 CUs): a wave's columns for a block. At D =
  // 512, of calls with the host's part: 2048 rows 11.6 us, 16.3 the other way; 4096 14.0 for
  // 16.7; 8192 25.0 for 17.5.
  if (tiles * (D / 16) <= 8 * (int64_t)num_cus) {
    const int64_t parts = up8(tiles);
    hipLaunchKernelGGL((mx4_unrotate_kernel<D, 1, 1>), dim3((unsigned)(parts * (D / 16))), dim3(64), 0, stream, a,
                       (int)tiles);
  } else {
    constexpr int SPLIT = D / 256;
    const int64_t parts = std::min(tiles, (int64_t)std::max(num_cus / SPLIT, 1));
    hipLaunchKernelGGL((mx4_unrotate_kernel<D, 8, 2>), dim3((unsigned)(up8(parts) * SPLIT)), dim3(512), 0, stream, a,
                       (int)parts);
  }
  return hipGetLastError();
}

}  // namespace rolaq

hipError_t rolaq_launch_mx4_unrotate(const rolaq::Mx4RowsArgs& a, int D, int num_cus, hipStream_t stream) {
  return D == 512 ? rolaq::launch_unrotate<512>(a, num_cus, stream) : rolaq::launch_unrotate<256>(a, num_cus, stream);
}
