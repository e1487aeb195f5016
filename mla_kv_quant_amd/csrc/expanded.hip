// Attention over expanded latent keys and values (gfx950): per head h
//   s_t = sm_scale (q_nope . k_nope_t,h + q_pe . k_pe_t),  o = sum_t softmax(s)_t v_t,h,
// k_nope and v side by side as kv_b_proj gives them, one k_pe for all heads; causal at the
// end of the keys, or all keys for all queries.
//
// A block has 128 query rows of one head, 32 to each of four waves, which hold their queries and outputs in
// registers and go through the keys in steps of 32 (64 at the small widths) that asynchronous copies
// bring to LDS, four steps ahead. Scores are formed transposed, S^T = K Q^T, so that a lane has one
// query's scores and they become the next product's operand, O^T += V^T P^T, where they are (values
// are read transposed from LDS). One stream of matrix instructions interleaves a step's scores with the
// output of the step before and has its weights formed in between: exp2 of scaled scores less a
// reference that moves only when a step's sum of weights passes 256, so that no maximum is formed.
// Weights are rounded to bf16, the type of the values that they are multiplied with (fp16 is three bits
// finer, but has no place for values above 65504, and two bf16 parts would double the second product); sums are of the
// weights as rounded, by which the output's weights add up to one. Outputs are off by 0.0019 to 0.0022 of their norm;
// rounded once from the exact ones they would be by 0.0017.
//
// Bound: matrix instructions at the clock that the power limit leaves, two waves to a SIMD: 16 heads of 4 x 4096
// queries 330 to 400 us by card (344 GFLOP, 0.86 to 1.04 PFLOP/s; a large library product reaches 1.24), 55 % of the
// cycles at 1.77 GHz with one under way; 40 heads of 4 x 2048 behind 14336, 64 wide, 1.57 to 1.61 ms (1.0). Without the
// weights' arithmetic it takes 20 to 30 % less, without the copies 15 %, without the reads of keys and values 6 %.
// 256 rows a block, 64 rows a wave (one wave to a SIMD), rings of 8 steps and operands read 9
// instructions ahead were no faster (480 us for 430 with 64 rows).
// Few rows behind long keys: bound by the keys' bytes (8 x 16 queries behind 4096, 16 heads: 59 us, 275 MB). A row block
// of up to 32 rows leaves three of its waves to copy alone.
// (Of the 256 registers a wave has, 6 to 120 are spilled, in the repeated pass of blocks with outputs that are not finite
// alone.)
#include "rolaq_common.h"
#include "mx4_request.h"
#include "mx4_tile.h"
#include "serve_args.h"

#include <algorithm>
#include <type_traits>

namespace rolaq {

typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

constexpr float kXNoRef = -0x1.fffffep127f;  // reference of a row that has seen no score
constexpr float kXMost = 256.f;              // a step's sum of weights above which its row's reference is looked at

template <int DN>
struct XGeo {
  static constexpr int DR = DN / 2, DK = DN + DR;
  static constexpr int W = 4;                     // waves
  static constexpr int ROWS = 32 * W;             // query rows of a block
  static constexpr int TK = DN == 128 ? 32 : 64;  // keys of a step
  static constexpr int U = TK / 32;               // units of 32 keys
  static constexpr int NB = 2 * DN, PB = 2 * DR;  // bytes of a nope or value row, and of a rope row
  static constexpr int NTILE = TK * NB, PTILE = TK * PB, KTILE = NTILE + PTILE;
  static constexpr int RING = 4;                  // steps whose keys, and values, lie in LDS
  static constexpr int V0 = RING * KTILE;         // where the values start
  static constexpr int LDS = V0 + RING * NTILE;
  static constexpr int KS = DK / 16, KN = DN / 16;  // K-steps of the scores, those of the nope part
  static constexpr int ND = DN / 32;                // output column blocks
  static constexpr int SM = KS * U, OM = 2 * ND * U, SL = SM + OM;  // MFMAs of a step
  static constexpr int COPIES = 5;  // a wave's, of 1 KB each: two pieces of nope, one of rope, two of values
  static_assert(NTILE == 2048 * W && PTILE == 1024 * W && 2 * LDS <= 160 * 1024, "pieces of a step, two blocks a CU");
};

__device__ __forceinline__ f32x16 mfma32x32x16_bf16(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ float x_max_halves(float v) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
}
__device__ __forceinline__ float x_add_halves(float v) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

// Chunk c (16 bytes) of row r of a tile lies at chunk c ^ swz(r): 16 rows of one column (a quarter
// wave of a score read), and 4 rows x 64 bytes (half a wave of a transposed read), fall
// on 16 chunk positions each. BYTES: of a row.
template <int BYTES>
__device__ __forceinline__ int k_swz(int r) { return BYTES == 256 ? r & 15 : BYTES == 128 ? (r >> 1) & 7 : (r >> 2) & 3; }
template <int BYTES>
__device__ __forceinline__ int v_swz(int r) { return BYTES == 256 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); }

__device__ __forceinline__ float x_sum2(uint32_t v, float acc) {  // acc + both bf16 values of v
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, v), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), acc,
                                         false);
}

// The largest of the lanes' v, none negative (DPP as in wave_scan).
__device__ __forceinline__ int wave_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
  return __builtin_amdgcn_readlane(v, 63);
}

struct XPlace {
  int b, rb;           // request (-1: none), row block
  int q0, nq, past;    // first query, queries computed, keys before the first query's own
  int k0, nk;          // first key row, key rows
  int parts;           // parts of the keys of every row block
};
// What a launch takes, in us, of `blocks` row blocks of `longest` steps at most, `mean` in the mean, in `parts`: a
// step of one block on a CU, and of each of several; split keys cost their rows' partials, written and read
// (`partial` a part), and a second launch.
__device__ __host__ inline float x_cost(float blocks, float cus, float longest, float mean, float partial, int parts) {
  const float each = ceilf(blocks * (float)parts / cus);
  return fmaxf(0.65f * longest, 0.6f * each * mean) / (float)parts + (parts > 1 ? 6.f + partial * (float)parts : 0.f);
}
// The `want`-th row block of the batch: a request's run together, as they share its keys, the last (which sees most)
// first, and of up to 64 requests those of more than half the most keys before the others, so that the blocks that
// a launch ends with are short.
// (Row blocks of all requests by their number of keys: 10 prompts of 800, 128 heads, 610 us against 540.)
// Where the launch has room for parts (a.splits > 1), their number follows from the lengths.
template <int ROWS, int TK>
__device__ __forceinline__ XPlace x_place(const ExpandedArgs& a, uint32_t want) {
  const int lane = threadIdx.x & 63;
  const auto clampq = [&](int i) { return min(max(a.qo_indptr[i], 0), a.T); };
  const auto clampk = [&](int i) { return min(max(a.kv_indptr[i], 0), a.N); };
  XPlace p{-1, 0, 0, 0, 0, 0, 0, 1};
  uint32_t before = 0;
  for (int c = 0; c < a.B; c += 64) {
    const int i = min(c + lane, a.B - 1);
    const int q0 = clampq(i), nq_all = max(clampq(i + 1) - q0, 0), nq = min(nq_all, a.max_q_len);
    const int k0 = clampk(i), nk = max(clampk(i + 1) - k0, 0), past = nk - nq_all;
    const int n = c + lane < a.B ? (nq + ROWS - 1) / ROWS : 0;
    uint32_t start = 0;  // row blocks before this lane's request's
    if (a.B <= 64) {
      const int most = wave_max(n ? nk : 0);
      const uint32_t longer = nk > most / 2 ? (uint32_t)n : 0u, rest = (uint32_t)n - longer;
      const uint32_t to = wave_scan(longer), behind = wave_scan(rest);  // (by all lanes)
      const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)to, 63);
      start = longer ? to - longer : first + behind - rest;
      if (a.splits > 1) {
        const float steps = (float)((nk + TK - 1) / TK), longest = (float)((most + TK - 1) / TK);
        // (a causal request's row blocks see ever fewer keys)
        float all = (float)n * steps - (a.causal ? 0.5f * (float)n * (float)(n - 1) * (float)(ROWS / TK) : 0.f);
        all = fmaxf(all, (float)n);
        float blocks = (float)n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) all += __shfl_xor(all, o), blocks += __shfl_xor(blocks, o);
        // lane s - 1 has s parts, of four steps at least
        float us = lane < a.splits && (lane == 0 || 4.f * (float)(lane + 1) <= longest)
                       ? x_cost(blocks * (float)a.H, (float)a.cus, longest, all / fmaxf(blocks, 1.f), a.partial, lane + 1)
                       : INFINITY;
        int parts = lane + 1;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const float u = __shfl_xor(us, o);
          const int q = __shfl_xor(parts, o);
          if (u < us || (u == us && q < parts)) us = u, parts = q;
        }
        p.parts = __builtin_amdgcn_readfirstlane(parts);
      }
    } else {
      const uint32_t incl = wave_scan((uint32_t)n);
      start = before + incl - (uint32_t)n;
      before += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    }
    const uint64_t hit = __builtin_amdgcn_ballot_w64(start <= want && want < start + (uint32_t)n);
    const int rb = n - 1 - (int)(want - start);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      p.b = c + l;
      p.rb = __builtin_amdgcn_readlane(rb, l);
      p.q0 = __builtin_amdgcn_readlane(q0, l);
      p.nq = __builtin_amdgcn_readlane(nq, l);
      p.past = __builtin_amdgcn_readlane(past, l);
      p.k0 = __builtin_amdgcn_readlane(k0, l);
      p.nk = __builtin_amdgcn_readlane(nk, l);
      return p;
    }
  }
  return p;
}

// Copies of 16 bytes a lane to lds and lds + 1024: from base + o0 and base + 1024 + o1 (the
// instruction's offset counts on both sides).
__device__ __forceinline__ void x_copy2(const void* base, uint32_t o0, uint32_t o1, uint32_t lds) {
  asm volatile(
      "s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %3\n\t"
      "global_load_lds_dwordx4 %2, %3 offset:1024" ::"s"(lds),
      "v"(o0), "v"(o1), "s"(base)
      : "memory", "m0");
}

// One block's work. LSE: for calls that ask for it, the sum of the weights before their rounding as well. CARE: with
// a look at values that rows may not see (see clean); without, true, and nothing written, where outputs are
// not finite.
template <int DN, bool LSE, bool CARE>
__device__ __forceinline__ bool expanded_block(const ExpandedArgs& a) {
  using G = XGeo<DN>;
  constexpr int NB = G::NB, PB = G::PB, TK = G::TK, KS = G::KS, KN = G::KN, ND = G::ND, U = G::U, RING = G::RING;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  int tid = threadIdx.x;
  if (CARE) asm volatile("" : "+v"(tid));  // (nothing formed the first time is kept in registers for this)
  const int lane = tid & 63, la32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // ---- head, row block and part of the keys ---------------------------------------
  // Where every block is resident at once, none waits for a CU to fall idle: the second one on each CU is
  // taken from the short end, so that a CU's two take as long as another's.
  uint32_t item = blockIdx.x;
  const uint32_t cus = (uint32_t)a.cus;
  if (gridDim.x > cus && gridDim.x <= 2 * cus && item >= cus) item = gridDim.x - 1 - (item - cus);
  const int h = item % (uint32_t)a.H;
  const uint32_t rest = item / (uint32_t)a.H;
  const int part = rest / (uint32_t)a.blocks;
  const XPlace at = x_place<G::ROWS, TK>(a, rest - (uint32_t)part * (uint32_t)a.blocks);
  const int parts = at.parts;
  if (at.b < 0 || part >= parts) return false;
  if (a.splits > 1 && item == 0 && tid == 0)  // (for the second launch)
    reinterpret_cast<int*>(a.ws)[(int64_t)a.splits * a.T * a.H * (DN + 2)] = parts;
  // Row blocks are full from the last query back, so that a short one is the first, which sees the fewest
  // keys (10 prompts of 800, 128 heads: 540 us full from the first query on, 520 so).
  const int q0 = at.q0, k0 = at.k0, nk = at.nk, short_rows = (at.nq - 1) % G::ROWS + 1;
  const int row0 = at.rb == 0 ? 0 : short_rows + G::ROWS * (at.rb - 1);
  const int nq = short_rows + G::ROWS * at.rb;  // rows up to this block's end
  // keys that row r sees
  const auto sees = [&](int r) { return a.causal ? min(max(at.past + r + 1, 0), nk) : nk; };
  const int tiles = (sees(nq - 1) + TK - 1) / TK;
  const int t0 = (int)((int64_t)tiles * part / parts), n = (int)((int64_t)tiles * (part + 1) / parts) - t0;
  const int first_key = TK * t0;  // keys and steps are counted from here

  // ---- tile copies ------------------------------------------------------------------
  // This wave's pieces of a step: two of nope, one of rope, two of values, 64 chunks each.
  // Every step issues the same copies: past the last tile that one again, to places that nothing reads any
  // more; rows past the last key read that one.
  constexpr int NC = NB / 16, PC = PB / 16;  // chunks of a row
  const uint32_t kv_row = 2 * (uint32_t)a.kv_st, pe_row = 2 * (uint32_t)a.pe_st;  // bytes
  // (1024 bytes before the first row, so that no offset is negative)
  const uint8_t* const kv =
      reinterpret_cast<const uint8_t*>(a.kv + (int64_t)(k0 + first_key) * a.kv_st + (int64_t)h * a.kv_sh) - 1024;
  const uint8_t* const pe = reinterpret_cast<const uint8_t*>(a.pe + (int64_t)(k0 + first_key) * a.pe_st);
  const auto n_row = [&](int j) { return (64 * (2 * wave + j) + lane) / NC; };
  const int p_row = (64 * wave + lane) / PC;
  uint32_t noff[2], voff[2], poff = p_row * pe_row + 16 * ((lane % PC) ^ k_swz<PB>(p_row));
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = n_row(j), c = lane % NC;
    noff[j] = r * kv_row + 1024 * (1 - j) + 16 * (c ^ k_swz<NB>(r));
    voff[j] = r * kv_row + 1024 * (1 - j) + NB + 16 * (c ^ v_swz<NB>(r));
  }
  const auto past_last = [&](int r) { return (uint32_t)max(r - (nk - 1 - first_key - TK * (n - 1)), 0); };
  const auto tile_of = [&](const uint8_t* p, uint32_t row, int t) {
    return p + (uint64_t)(uint32_t)min(t, n - 1) * (uint64_t)(TK * row);
  };
  const auto copy_nope = [&](int t, int slot) __attribute__((always_inline)) {
    if (__builtin_expect(t == n - 1, 0)) {  // (once: the later ones are this tile again)
      asm volatile("");
#pragma unroll
      for (int j = 0; j < 2; ++j) noff[j] -= past_last(n_row(j)) * kv_row;
      poff -= past_last(p_row) * pe_row;
    }
    x_copy2(tile_of(kv, kv_row, t), noff[0], noff[1], lds0 + slot * G::KTILE + 2048 * wave);
  };
  const auto copy_rope = [&](int t, int slot) __attribute__((always_inline)) {
    copy16(tile_of(pe, pe_row, t), poff, lds0 + slot * G::KTILE + G::NTILE + 1024 * wave);
  };
  const auto copy_values = [&](int t, int slot) __attribute__((always_inline)) {
    if (__builtin_expect(t == n - 1, 0)) {
      asm volatile("");
#pragma unroll
      for (int j = 0; j < 2; ++j) voff[j] -= past_last(n_row(j)) * kv_row;
    }
    x_copy2(tile_of(kv, kv_row, t), voff[0], voff[1], lds0 + G::V0 + slot * G::NTILE + 2048 * wave);
  };

  // ---- query rows -------------------------------------------------------------------
  const int row = min(row0 + 32 * wave + la32, nq - 1);  // (rows past the last: that one again)
  u32x4 qf[KS];
  {
    const uint16_t* const p = a.q + (int64_t)(q0 + row) * a.q_st + (int64_t)h * a.q_sh + 8 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = gload<u32x4>(p + 16 * s);
  }
  // The first tiles go out behind the query's loads, which are waited for here, so that no wait for
  // them is left behind the copies.
  if (n > 0) {
#pragma unroll
    for (int t = 0; t < RING; ++t) {
      copy_nope(t, t);
      copy_rope(t, t);
    }
#pragma unroll
    for (int t = 0; t < RING - 2; ++t) copy_values(t, t);
  }
#pragma unroll
  for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qf[s]));
  const int vis = sees(row) - first_key;       // keys that the row sees, from first_key on
  const int vis_min = sees(row0) - first_key;  // seen by every row of the block
  // steps of which this wave has rows that see something: in the others it only copies
  const int row_last = min(row0 + 32 * wave + 31, nq - 1);
  const int own = row0 + 32 * wave >= nq ? 0 : min(max((sees(row_last) - first_key + TK - 1) / TK, 0), n);

  f32x16 O[ND];  // O^T: columns 32 d + 8 (j / 4) + 4 g + j % 4 of the lane's row
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) O[d][j] = 0.f;
  float ref = kXNoRef, sum = 0.f, usum = 0.f;  // usum (LSE): of the weights as they were
  float most = kXMost;                         // the largest sum of a step that needs no look at the reference
  const float c2 = a.sm_scale * kLog2e;

  // ---- LDS operands -----------------------------------------------------------------
  const int la = lane & 15;
  uint32_t kbase[KS], vbase[ND];
#pragma unroll
  for (int s = 0; s < KS; ++s)
    kbase[s] = s < KN ? la32 * NB + 16 * ((2 * s + g) ^ k_swz<NB>(la32))
                      : G::NTILE + la32 * PB + 16 * ((2 * (s - KN) + g) ^ k_swz<PB>(la32));
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    const int r = 4 * g + (la >> 2);
    vbase[d] = G::V0 + r * NB + 16 * ((4 * d + 2 * ((lane >> 4) & 1) + ((la & 3) >> 1)) ^ v_swz<NB>(r)) + 8 * (la & 1);
  }
  // K-step s of unit u of the keys in `slot`
  const auto kread = [&](int slot, int u, int s) __attribute__((always_inline)) {
    return *reinterpret_cast<const u32x4*>(smem + kbase[s] + slot * G::KTILE + u * 32 * (s < KN ? NB : PB));
  };
  // columns 32 d .. of 16 keys m of the values in `slot`, transposed
  const auto vread = [&](int slot, int m, int d) __attribute__((always_inline)) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const uint8_t* const p = smem + vbase[d] + slot * G::NTILE + 16 * m * NB;
    const u32x2 v0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p)));
    const u32x2 v1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * NB)));
    return u32x4{v0.x, v0.y, v1.x, v1.y};
  };

  // ---- the parts of a step ------------------------------------------------------------
  // MFMA i of a step's scores: units in turns, so that chains of one unit are apart
  const auto score = [&](f32x16 (&S)[U], int i, u32x4 k) __attribute__((always_inline)) {
    const int u = i % U, s = i / U;
    f32x16 zero;
#pragma unroll
    for (int j = 0; j < 16; ++j) zero[j] = 0.f;
    S[u] = mfma32x32x16_bf16(k, qf[s], s == 0 ? zero : S[u]);
  };
  const auto output = [&](const u32x4 (&P)[2 * U], int i, u32x4 v) __attribute__((always_inline)) {
    O[i % ND] = mfma32x32x16_bf16(v, P[i / ND], O[i % ND]);
  };
  // positions that a row does not see
  const auto mask = [&](f32x16 (&S)[U], int t) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int lim = vis - TK * t - 32 * u - 4 * g;
#pragma unroll
      for (int j = 0; j < 16; ++j) S[u][j] = 8 * (j / 4) + j % 4 < lim ? S[u][j] : -INFINITY;
    }
  };
  // Weights of a step in OPS operations for each of 8 U pairs of keys
  float e0, e1, us[2], uu;
  constexpr int OPS = LSE ? 8 : 6;
  const auto weigh = [&](const f32x16 (&S)[U], u32x4 (&P)[2 * U], int o) __attribute__((always_inline)) {
    const int e = o / OPS, m = e / 4, d = e % 4, j = 8 * (m % 2) + 2 * d, op = o % OPS;
    if (op == 0) e0 = fmaf(S[m / 2][j], c2, -ref);
    if (op == 1) e1 = fmaf(S[m / 2][j + 1], c2, -ref);
    if (op == 2) e0 = __builtin_amdgcn_exp2f(e0);
    if (op == 3) e1 = __builtin_amdgcn_exp2f(e1);
    if (op == 4) {
      uint32_t w = pack_bf16(e0, e1);
      asm volatile("" : "+v"(w));  // formed here, not where a later step uses it
      P[m][d] = w;
    }
    if (op == 6) uu += e0;
    if (op == 7) {
      uu += e1;
      asm volatile("" : "+v"(uu));
    }
    if (op == 5) {
      us[e % 2] = x_sum2(P[m][d], us[e % 2]);
      asm volatile("" : "+v"(us[e % 2]));
    }
  };
  // A step's sum says whether a weight passed the slack (or was the row's first): then the
  // reference moves to the largest score so far, what was summed before is scaled, and the
  // step's weights are formed again, by a difference of rounded scores, which holds
  // for scores of any size. (No maximum is formed otherwise.)
  const auto settle = [&](const f32x16 (&S)[U], u32x4 (&P)[2 * U]) __attribute__((always_inline)) {
    float got = us[0] + us[1];
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(got > most) != 0, 0)) {
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 16; ++j) mx = fmaxf(mx, S[u][j]);
      mx = x_max_halves(mx) * c2;
      const bool over = x_max_halves(got) > most;
      const float to = over ? fmaxf(mx, ref) : ref;
      // (nothing was summed before the first reference, but an infinite value may be in O)
      const float f = ref == kXNoRef ? 1.f : __builtin_amdgcn_exp2f(ref - to);
      ref = to;
      if (over) most = fabsf(to) < 0x1p24f ? kXMost : -1.f;
      sum *= f;
      usum *= f;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) O[d][j] *= f;
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int m = 0; m < 2 * U; ++m)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const float x0 = S[m / 2][8 * (m % 2) + 2 * d], x1 = S[m / 2][8 * (m % 2) + 2 * d + 1];
          float p0, p1;
          {
#pragma clang fp contract(off)
            p0 = __builtin_amdgcn_exp2f(x0 * c2 - to);
            p1 = __builtin_amdgcn_exp2f(x1 * c2 - to);
          }
          const uint32_t w = over ? pack_bf16(p0, p1) : P[m][d];
          P[m][d] = w;
          s0 += bf16_lo(w) + bf16_hi(w);
          s1 += p0 + p1;
        }
      got = over ? s0 : got;
      if (LSE) uu = over ? s1 : uu;
    }
    sum += got;
    if (LSE) usum += uu;
  };
  // Values of a tile of which a row may not see all may be anything where it does not see them, and 0
  // times what is not finite is NaN, which stays. So a block whose outputs are not finite goes through its
  // keys again, with care: before such a tile's output every wave looks for a value that is not finite;
  // where there is one, all agree, each clears those of its own pieces, and what they add to the rows that
  // see them comes from memory. (With care at once: a prompt of 333, 16 heads, 15.5 us for 14.4, ragged
  // prompts of 128 heads 852 for 834.)
  const auto clean = [&](int slot, int t) __attribute__((always_inline)) {
    u16x2_t big = {0, 0};
    uint8_t* const v = smem + G::V0 + slot * G::NTILE + 16 * lane;
#pragma unroll
    for (int k = 0; k < G::NTILE / 1024; ++k) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(v + 1024 * k);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2_t, w[e] & 0x7fff7fffu));
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(big[0] >= 0x7f80 || big[1] >= 0x7f80) == 0, 1)) return;
    __syncthreads();
#pragma unroll
    for (int k = 2 * wave; k < 2 * wave + 2; ++k) {
      u32x4 w = *reinterpret_cast<const u32x4*>(v + 1024 * k);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u;
        if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0xffffu;
      }
      *reinterpret_cast<u32x4*>(v + 1024 * k) = w;
    }
    __syncthreads();
#pragma unroll 1
    for (int k = TK * t; k < min(TK * (t + 1), nk - first_key); ++k) {
      const uint8_t* const vr = kv + (int64_t)k * kv_row + 1024 + NB + 8 * g;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const u32x2 w = gload<u32x2>(vr + 64 * d + 16 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float y = e % 2 ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2]);
            if (k < vis && !(fabsf(y) < INFINITY)) O[d][4 * q + e] += y;
          }
        }
    }
  };

  // Step t, in ring slot I of t: the matrix cores form the scores of step t + 1 and the output of
  // step t - 1 while the vector units turn the scores S of step t into weights. Its operands
  // come in a ring of AHEAD + 1, of 5 in a row the second and the fourth the output's;
  // where the last of them are under way it meets the other waves and turns to the next step's.
  // (The first step has zero weights for its output, and zero values: slot RING - 1 is cleared.)
  constexpr int AHEAD = 4, SL = G::SL;
  static_assert(G::SM * 2 == G::OM * 3 && SL % (AHEAD + 1) == 0, "three of the scores to two of the output");
  u32x4 f[AHEAD + 1];
  const auto fetch = [&](auto I, int y) __attribute__((always_inline)) {
    constexpr int i = decltype(I)::value;
    const int k = 2 * (y / 5) + y % 5 / 2, s = 3 * (y / 5) + y % 5 / 2;
    f[y % (AHEAD + 1)] = y % 5 % 2 == 0 ? kread((i + 1) % RING, s % U, s / U) : vread((i + RING - 1) % RING, k / ND, k % ND);
  };
  // Before step t: K t + 1 and V t - 1 are there (two steps' copies may be under way), and no wave
  // reads K t and V t - 2 any more.
  const auto meet = [&](int slot, int t) __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((RING - 2) * G::COPIES) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (CARE && __builtin_expect(TK * t > vis_min && t > 0, 0)) clean((slot + RING - 1) % RING, t - 1);
  };
  const auto step = [&](auto I, int t, f32x16 (&S)[U], f32x16 (&Sn)[U], u32x4 (&P)[2 * U], const u32x4 (&Pb)[2 * U])
                        __attribute__((always_inline)) {
    constexpr int i = decltype(I)::value;
    const std::integral_constant<int, (i + 1) % RING> next;
    if (__builtin_expect(TK * (t + 1) > vis_min, 0)) mask(S, t);
    us[0] = us[1] = uu = 0.f;
    static_for<SL>([&](auto Y) __attribute__((always_inline)) {
      constexpr int y = decltype(Y)::value, k = 2 * (y / 5) + y % 5 / 2, ALL = 8 * U * OPS;
      if constexpr (y == 1) copy_nope(t + RING, i);
      if constexpr (y == 6) copy_rope(t + RING, i);
      if constexpr (y == 11) copy_values(t + RING - 2, (i + RING - 2) % RING);
      if constexpr (y == SL - AHEAD) meet((i + 1) % RING, t + 1);
      if constexpr (y + AHEAD < SL)
        fetch(I, y + AHEAD);
      else
        fetch(next, y + AHEAD - SL);
      if constexpr (y % 5 % 2 == 0)
        score(Sn, 3 * (y / 5) + y % 5 / 2, f[y % (AHEAD + 1)]);
      else
        output(Pb, k, f[y % (AHEAD + 1)]);
      constexpr int o0 = y * ALL / SL, o1 = (y + 1) * ALL / SL;
      static_for<o1 - o0>([&](auto o) __attribute__((always_inline)) { weigh(S, P, o0 + decltype(o)::value); });
      __builtin_amdgcn_sched_barrier(0);
    });
    settle(S, P);
  };

  if (n > 0) {
    f32x16 SA[U], SB[U];
    u32x4 PA[2 * U], PB_[2 * U];
#pragma unroll
    for (int m = 0; m < 2 * U; ++m) PB_[m] = PA[m] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (int k = 0; k < 2; ++k)
      *reinterpret_cast<u32x4*>(smem + G::V0 + (RING - 1) * G::NTILE + 1024 * (2 * wave + k) + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
    wait_loads<0>();
    __syncthreads();
    if (own > 0) {
#pragma unroll
      for (int x = 0; x < G::SM; ++x) {
        score(SA, x, kread(0, x % U, x / U));
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __syncthreads();  // (K 0 is no longer read)
    int t = 0;
    if (own > 0) {
      static_for<AHEAD>([&](auto Y) __attribute__((always_inline)) { fetch(std::integral_constant<int, 0>{}, decltype(Y)::value); });
      for (;;) {
        step(std::integral_constant<int, 0>{}, t, SA, SB, PA, PB_);
        if (++t == own) break;
        step(std::integral_constant<int, 1>{}, t, SB, SA, PB_, PA);
        if (++t == own) break;
        step(std::integral_constant<int, 2>{}, t, SA, SB, PA, PB_);
        if (++t == own) break;
        step(std::integral_constant<int, 3>{}, t, SB, SA, PB_, PA);
        if (++t == own) break;
      }
      // the last step's output (its values were met for)
      if ((own & 1) == 0) {
#pragma unroll
        for (int m = 0; m < 2 * U; ++m) PA[m] = PB_[m];
      }
#pragma unroll
      for (int x = 0; x < G::OM; ++x) {
        output(PA, x, vread((own - 1) % RING, x / ND, x % ND));
        if (x % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    }
    for (; t < n; ++t) {  // steps of other waves
      copy_nope(t + RING, t % RING);
      copy_rope(t + RING, t % RING);
      copy_values(t + RING - 2, (t + RING - 2) % RING);
      meet((t + 1) % RING, t + 1);
    }
    wait_loads<0>();  // no copy may outlive the block's LDS
    if constexpr (!CARE) {
      float all = 0.f;  // not finite where an output is not
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int j = 0; j < 16; ++j) all += O[d][j];
      const bool bad = __builtin_amdgcn_ballot_w64(!(fabsf(all) < INFINITY)) != 0;
      __syncthreads();  // (nothing is read from LDS any more)
      uint32_t* const of = reinterpret_cast<uint32_t*>(smem);
      if (lane == 0) of[wave] = bad;
      __syncthreads();
      const u32x4 b = *reinterpret_cast<const u32x4*>(of);
      if (__builtin_amdgcn_readfirstlane((int)(b[0] | b[1] | b[2] | b[3]))) {
        __syncthreads();
        return true;
      }
    }
  }

  // ---- normalise and store -----------------------------------------------------------------
  const bool ok = row0 + 32 * wave + la32 < nq;
  const float l = x_add_halves(sum);
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
  const float ul = LSE ? x_add_halves(usum) : 0.f;
  const int64_t to = (int64_t)(q0 + row) * a.H + h;
  if (parts > 1) {
    const int64_t total = (int64_t)a.T * a.H;
    float* const po = a.ws + (part * total + to) * DN + 4 * g;
    if (ok) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4*>(po + 32 * d + 8 * q) =
              f32x4{O[d][4 * q] * inv, O[d][4 * q + 1] * inv, O[d][4 * q + 2] * inv, O[d][4 * q + 3] * inv};
      float* const pl = a.ws + a.splits * total * DN + part * total + to;
      if (g == 0) *pl = l == 0.f ? -INFINITY : ref + __log2f(l);
      if (LSE && g == 0) pl[a.splits * total] = ul == 0.f ? -INFINITY : ref + __log2f(ul);
    }
    return false;
  }
  if (LSE && ok && g == 0) a.lse[to] = ul == 0.f ? -INFINITY : (ref + __log2f(ul)) * kLn2;
  uint16_t* const dst = a.out + (int64_t)(q0 + row) * a.o_st + (int64_t)h * a.o_sh;
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    uint32_t w[4][2];  // columns 32 d + 8 q + 4 g + (0..3)
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int k = 0; k < 2; ++k) w[q][k] = pack_bf16(O[d][4 * q + 2 * k] * inv, O[d][4 * q + 2 * k + 1] * inv);
    // the halves' pieces joined to 8 consecutive columns a lane: 32 d + 16 p + 8 g + (0..7)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const auto y = __builtin_amdgcn_permlane32_swap(w[2 * p][0], w[2 * p + 1][0], false, false);
      const auto z = __builtin_amdgcn_permlane32_swap(w[2 * p][1], w[2 * p + 1][1], false, false);
      if (ok) *reinterpret_cast<u32x4*>(dst + 32 * d + 16 * p + 8 * g) = u32x4{y[0], z[0], y[1], z[1]};
    }
  }
  return false;
}

template <int DN, bool LSE>
__global__ __launch_bounds__(256, 2) void expanded_kernel(ExpandedArgs a) {
  if (__builtin_expect(expanded_block<DN, LSE, false>(a), 0)) expanded_block<DN, LSE, true>(a);
}

// Partials of split keys: out = sum_s 2^(lse_s - M) O_s / sum_s 2^(lse_s - M).
template <int DN>
__global__ __launch_bounds__(256) void expanded_merge_kernel(ExpandedArgs a) {
  constexpr int LPR = DN / 4;  // lanes of a row
  const int64_t total = (int64_t)a.T * a.H;
  const int parts = min(reinterpret_cast<const int*>(a.ws)[a.splits * total * (DN + 2)], a.splits);
  if (parts <= 1) return;  // (written in its place)
  const int c = threadIdx.x % LPR;
  const int base = (threadIdx.x & 63) - c;  // the row's first lane
  const auto over = [](float v, auto f) {   // over the row's lanes
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) v = f(v, __shfl_xor(v, o));
    return v;
  };
  const auto max2 = [](float x, float y) { return fmaxf(x, y); };
  const auto add2 = [](float x, float y) { return x + y; };
  for (int64_t at = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR; at < total;
       at += (int64_t)gridDim.x * (256 / LPR)) {
    const int t = (int)(at / a.H), h = (int)(at - (int64_t)t * a.H);
    // rows that belong to no request, or to none of its first max_q_len, have no partials
    float there = 0.f;
    for (int b = c; b < a.B; b += LPR) {
      const int lo = min(max(a.qo_indptr[b], 0), a.T), hi = min(max(a.qo_indptr[b + 1], 0), a.T);
      if (t >= lo && t < min((int64_t)hi, (int64_t)lo + a.max_q_len)) there = 1.f;
    }
    if (over(there, max2) == 0.f) continue;
    // (parts s = c, c + LPR .. are this lane's)
    const float* const lse = a.ws + a.splits * total * DN + at;
    float M = -INFINITY;
    for (int s = c; s < parts; s += LPR) M = fmaxf(M, lse[s * total]);
    M = over(M, max2);
    float den = 0.f, sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < parts; s0 += LPR) {
      const int mine = s0 + c;
      const float l = mine < parts ? lse[mine * total] : -INFINITY;
      const float wl = l == -INFINITY ? -1.f : __builtin_amdgcn_exp2f(l - M);  // (-1: a part without keys)
      if (l != -INFINITY) den += wl;
      if (a.lse && mine < parts) {
        const float ul = lse[(a.splits + mine) * total];
        if (ul != -INFINITY) sum += __builtin_amdgcn_exp2f(ul - M);
      }
      const int n = min(LPR, parts - s0);
#pragma unroll 8
      for (int i = 0; i < n; ++i) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.ws + ((s0 + i) * total + at) * DN + 4 * c);
        const float w = __shfl(wl, base + i);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = w == -1.f ? o[k] : fmaf(w, v[k], o[k]);
      }
    }
    den = over(den, add2);
    const float inv = den == 0.f ? 0.f : 1.f / den;
    if (a.lse) {
      sum = over(sum, add2);
      if (c == 0) a.lse[at] = sum == 0.f ? -INFINITY : (M + __log2f(sum)) * kLn2;
    }
    *reinterpret_cast<u32x2*>(a.out + (int64_t)t * a.o_st + (int64_t)h * a.o_sh + 4 * c) =
        u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
  }
}

constexpr int kXMostSplits = 64;
struct XPlan {
  int64_t blocks;  // row blocks of the batch at most
  int splits;      // parts of the keys at most
  float partial;   // us of a part's partials
};
// The lengths are known on the device alone. There is room for as many parts as pay for one request of all
// the keys, where row blocks are fewer than the two a CU that run together (more end close together: the longest
// come first) and requests fewer than the lanes that find them; at most four blocks a CU in all.
XPlan expanded_plan(int64_t T, int64_t N, int B, int H, int DN, int max_q_len, int num_cus) {
  constexpr int rows = XGeo<128>::ROWS;
  XPlan p{std::min<int64_t>((int64_t)B * ((max_q_len + rows - 1) / rows), T / rows + B), 1, 0.f};
  p.partial = (float)(8.0 * (double)T * H * DN / 5e6);  // written and read at 5 TB/s
  const int64_t all = std::max<int64_t>(p.blocks * H, 1), room = all < 2 * (int64_t)num_cus ? 4 * (int64_t)num_cus / all : 1;
  const float steps = (float)(N / (DN == 128 ? XGeo<128>::TK : XGeo<64>::TK));
  if (B > 64) return p;
  float best = x_cost(1.f, (float)num_cus, steps, steps, p.partial, 1);
  for (int s = 2; s <= std::min<int64_t>(room, kXMostSplits) && 4.f * s <= steps; ++s) {
    const float us = x_cost(1.f, (float)num_cus, steps, steps, p.partial, s);
    if (us < best) best = us, p.splits = s;
  }
  return p;
}

template <int DN, bool LSE>
hipError_t launch_expanded(ExpandedArgs a, int num_cus, hipStream_t stream) {
  using G = XGeo<DN>;
  const XPlan p = expanded_plan(a.T, a.N, a.B, a.H, DN, a.max_q_len, num_cus);
  a.splits = p.splits;
  a.blocks = (int)p.blocks;
  a.partial = p.partial;
  a.cus = num_cus;
  hipError_t e = hipFuncSetAttribute((const void*)expanded_kernel<DN, LSE>, hipFuncAttributeMaxDynamicSharedMemorySize, G::LDS);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((expanded_kernel<DN, LSE>), dim3((unsigned)(p.blocks * a.H * a.splits)), dim3(256), G::LDS, stream, a);
  e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  const int64_t rows = (int64_t)a.T * a.H, per = 256 / (DN / 4);
  hipLaunchKernelGGL((expanded_merge_kernel<DN>), dim3((unsigned)std::min<int64_t>((rows + per - 1) / per, 8 * num_cus)),
                     dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace rolaq

int64_t rolaq_expanded_ws_bytes(int64_t T, int64_t N, int B, int H, int DN, int max_q_len, int num_cus) {
  const int s = rolaq::expanded_plan(T, N, B, H, DN, max_q_len, num_cus).splits;
  return s > 1 ? (int64_t)s * T * H * (DN + 2) * 4 + 16 : 0;
}

hipError_t rolaq_launch_expanded(const rolaq::ExpandedArgs& a, int DN, int num_cus, hipStream_t stream) {
  using namespace rolaq;
  if (DN == 128)
    return a.lse ? launch_expanded<128, true>(a, num_cus, stream) : launch_expanded<128, false>(a, num_cus, stream);
  if (DN == 64)
    return a.lse ? launch_expanded<64, true>(a, num_cus, stream) : launch_expanded<64, false>(a, num_cus, stream);
  return hipErrorInvalidValue;
}
