// Absorbed MLA attention over the 4-bit (MX4) latent cache (gfx950): decode,
// verification of a few drafted tokens and chunked prefill with one kernel.
//
// For a query row (token i of n, head) over the positions t <= len - n + i:
//   s_t = sm_scale (q_lat . x_t + q_pe . r_t),  O = sum_t softmax(s)_t x_t,
// x_t the stored latent row (4-bit codes times 2^e for each 32 of them), r_t the
// bf16 rope row.
//
// A block of four waves walks 64-position tiles for 16 G query rows (G = 1, 2, 4
// groups of 16). Tiles are copied by asynchronous loads straight into an LDS ring
// as they lie in the cache: 4-bit codes stay 4-bit up to the matrix core.
// * Scores: wave w takes group w % G and the positions 16 G (w / G) .. of a tile.
//   The codes are the A operand of v_mfma_scale_f32_16x16x128_f8f6f4 as they
//   are, with the block scales as its A scales, so nothing is expanded. The bf16
//   query is split into two e4m3 parts, hi + lo / 16, with one power of two for
//   a row: eight significant bits are two times four, so the split is exact
//   for values down to 2^-13 of the row's largest and off by less than 2^-21 of
//   it below. Rope terms are bf16 MFMAs into the same FP32 accumulators.
// * Softmax in FP32, log2 domain, against a whole-number reference for each
//   row: a tile's largest score rounded up, moved only when a later score passes
//   it by more than 2^8 (bf16 probabilities have FP32's range). A reference
//   then moves by whole powers of two, exact in the accumulators as in P. P is
//   rounded to bf16, into whose exponents the block scales go; O is divided by the sum of
//   the rounded P (v_dot2_f32_bf16, a chain for each sub-tile), so that weights add up
//   to one and a row that is seen alone comes back as it is. The LSE, where a
//   call asks for it, takes the sum of the P before rounding.
// * Output: wave w takes the features D/4 w .. of all G groups. The codes come
//   out of LDS transposed (ds_read_b64_tr_b4: 16 positions of one feature), become
//   bf16 pairs by v_cvt_scalef32_pk_bf16_fp4 (one instruction for two values) and
//   meet P in bf16 MFMAs. The block scales go into exponents, two at a time and
//   exactly. With one group (few rows) they are taken from P's: P 2^(s - 159)
//   (v_pk_sub_u16, saturating at zero), O 2^-32 of its value. With more they are
//   added to the values', once for all groups: x 2^(s - 63) (v_pk_add_u16; a zero
//   becomes 2^(s - 190), 2^-126 of the smallest level), O 2^64 times its value.
//   Masked positions have P = 0 and finite values (a scale byte that is none counts
//   as one), so what they hold does not reach O.
// One barrier a tile: the scores of tile i + 1 and the output of tile i lie between
// two barriers, so that matrix, vector and LDS work of both can overlap. With one
// group the loop waits for HBM (5.8 TB/s in it); with four at 512 features a turn takes
// 5100 cycles, of which matrix instructions are 2200, vector ones some 1300 and LDS reads some
// 1700 (every wave reads the whole tile's keys for its group): none of them is the bound, but
// with one wave on a SIMD and a barrier a turn they follow each other.
//
// Measured, kernel alone: 32 x 16384 positions, 16 heads, D = 512: 49 us (4.3 TB/s); 24 ragged
// requests with 128 heads: 71 us (690 TFLOP/s); 64 x 16384, 40 heads, D = 256: 89 us; chunks of 4 x
// 2048 behind 14336, 40 heads, D = 256: 4.7 ms (1.16 PFLOP/s).
//
// Work: the tiles of all (request, row block) pairs, each behind an allowance for its
// start and end, lie on one line that is cut into equal parts, a part for each block;
// a pair cut by a border leaves partials that mx4_merge_kernel joins. With many row
// blocks each has a block of its own.
#include "rolaq_common.h"
#include "mx4_args.h"
#include "mx4_tile.h"

#include <algorithm>

namespace rolaq {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;

constexpr int kMx4Tile = 64;           // positions in a tile
constexpr int kMx4Idx = 4;             // tiles whose page numbers are held (ring slots - 1 at least)
constexpr float kMx4NoRef = -0x1.fffffep127f;  // reference of a row that has seen no score
constexpr float kMx4Slack = 8.f;       // log2 by which a score may pass its row's reference: sums of
                                       // 2^21 such P times 6 2^96, the largest value held, stay below 2^128

// Packed saturating subtraction of two 16-bit fields.
__device__ __forceinline__ uint32_t sub_sat(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t,
                            __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// One group's output accumulators times f where need is not 0, in
// place in AGPRs (the branch is inside, so the compiler sees no join and adds no
// copies of them; the waits cover the MFMAs before and behind).
__device__ __forceinline__ void scale_acc8(f32x4 (&o)[8], float f, uint32_t need) {
  float t0, t1, t2, t3;
  asm volatile(
      "s_cmp_lg_u32 %13, 0\n\t"
      "s_cbranch_scc0 1f\n\t"
      "s_nop 7\n\ts_nop 7\n\t"
      "ROLAQ_ACC_SCALE %0, %8, %9, %10, %11, %12, %12, %12, %12\n\t"
      "ROLAQ_ACC_SCALE %1, %8, %9, %10, %11, %12, %12, %12, %12\n\t"
      "ROLAQ_ACC_SCALE %2, %8, %9, %10, %11, %12, %12, %12, %12\n\t"
      "ROLAQ_ACC_SCALE %3, %8, %9, %10, %11, %12, %12, %12, %12\n\t"
      "ROLAQ_ACC_SCALE %4, %8, %9, %10, %11, %12, %12, %12, %12\n\t"
      "ROLAQ_ACC_SCALE %5, %8, %9, %10, %11, %12, %12, %12, %12\n\t"
      "ROLAQ_ACC_SCALE %6, %8, %9, %10, %11, %12, %12, %12, %12\n\t"
      "ROLAQ_ACC_SCALE %7, %8, %9, %10, %11, %12, %12, %12, %12\n\t"
      "s_nop 7\n"
      "1:"
      : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3]), "+a"(o[4]), "+a"(o[5]), "+a"(o[6]), "+a"(o[7]),
        "=&v"(t0), "=&v"(t1), "=&v"(t2), "=&v"(t3)
      : "v"(f), "s"(need)
      : "scc");
}

// acc + both values of a packed pair of bf16 (exact products by one).
__device__ __forceinline__ float sum_bf16x2(uint32_t v, float acc) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, v), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), acc,
                                         false);
}

// Sum of two 16-bit fields each (no carry between them).
__device__ __forceinline__ uint32_t add16(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(u16x2, a) + __builtin_bit_cast(u16x2, b));
}

// Eight 4-bit codes -> eight bf16 values, in order.
__device__ __forceinline__ u32x4 fp4x8_to_bf16(uint32_t v) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, 1.0f, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, 1.0f, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, 1.0f, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, 1.0f, 3))};
}

template <int D, int R, int G>
struct Mx4Geo {
  static constexpr int W = 4;         // waves
  static constexpr int ROWS = 16 * G;
  static constexpr int NB = D / 32;   // scale blocks of a row
  static constexpr int KS = D / 128;  // K-steps of the latent scores; also blocks per lane group
  static constexpr int CB = D / 2;    // code bytes of a row
  static constexpr int FW = D / W;    // features of a wave
  static constexpr int FT = FW / 16;  // its output tiles
  static constexpr int TW = W / G;    // waves that share a group's positions
  static constexpr int MT = 4 / TW;   // 16-position sub-tiles of a wave's scores
  static constexpr int CT = kMx4Tile / W;  // positions that a wave copies
  static constexpr int CODES = kMx4Tile * CB, ROPE = kMx4Tile * 2 * R, SCALES = 256 * W;
  static constexpr int TILE = CODES + ROPE + SCALES;  // a ring slot
  static constexpr int S = D == 512 ? 5 : 4;          // ring slots
  static constexpr int OCC = D == 512 ? 1 : 2;        // blocks on a CU
  static constexpr bool ACC = D == 512 && G >= 2;     // over 256 registers: O in AGPRs
  // A turn in two parts, tile k + 1's products beside tile k's expansion, then tile k's
  // output beside tile k + 1's softmax: it holds the whole expanded tile, for which 256
  // features and four groups have no registers (two blocks on a CU). Per step of 24
  // requests with 128 heads, 512 features: 86 us, 94 without; of 64 x 16384 positions with
  // 40 heads, 256 features: 100 us, 89 without.
  static constexpr bool MIX = D == 512 && G >= 2;
  // Halves of P that the other turn holds at a time: with four groups one, 92 us for
  // both at the latter step's 96; with fewer both, 56.4 us for one's 57.4 (32 x 16384, 16 heads, 512).
  static constexpr int PH = G == 4 ? 1 : 2;
  // Block scales to V's exponents, not to P's: 16 additions for 32 features against 8 G. At
  // G = 1 the other way round takes 56.4 us for 55.8.
  static constexpr bool VSIDE = G >= 2;
  static constexpr float UNIT = VSIDE ? 0x1p-64f : 0x1p32f;  // of O
  // A pair's start (query, first tiles) and end (output or partial) count as so many tiles
  // where the work is cut, so that a block with two of them has fewer. us, 0 / 3 / 6 / 10: 24 ragged
  // requests with 128 heads 86.7 / 81.2 / 76.5 / 77.1; 16 with 2 .. 4 queries 54.9 / 49.0 / 45.2 / 44.9; 400 short
  // ones, 16 heads, 100.8 / 83.8 / 79.3 / 80.7; ragged chunks 882 / 866 / 847 / 854; D = 256, 64 ragged requests,
  // 16 heads 29.4 / 27.0 / 25.5 / 25.8; and ragged chunks, where nothing is gained, 376 / 373 / 379 / 377.
  static constexpr int PRE = 6;
  static constexpr int LOADS = (CODES + ROPE) / (1024 * W) + 1;  // a wave's copies for a tile
  // LDS offsets
  static constexpr int P = S * TILE;                        // [2][ROWS][64] bf16, 16-byte chunks swizzled
  static constexpr int ES = P + 2 * ROWS * 128;             // [2][NB][64] exponent fields of the scales
  static constexpr int IDX = ES + 2 * NB * 128;             // [kMx4Idx][W][64] page numbers
  static constexpr int FLAG = IDX + kMx4Idx * 256 * W;      // [2][W]
  static constexpr int WREF = FLAG + 8 * W;                 // [2][W][16]
  static constexpr int LSUM = WREF + 128 * W;               // [W][16] of two sums
  static constexpr int LDS = LSUM + 128 * W;
  static_assert(LDS * OCC <= 160 * 1024, "LDS of a CU");
  static_assert(S - 1 <= kMx4Idx, "page numbers in flight");
  static_assert(TW >= 1 && TW <= 4 && FT % 2 == 0, "a wave's scores and features");
  static constexpr int SLOT = ROWS * (D + 3) * 4;  // bytes of a partial: O, (reference, sum of rounded P) by row, sum of P by row
};

// What the attend kernel leaves for the merge at the start of the workspace, by pair
// (request and row block), or by block where there are more pairs than kMx4Jobs.
struct Mx4Job {
  int parts;       // blocks that hold partials of the pair, from block `first` on; 0: nothing to join
  int first;
  int second;      // block `first`'s is its second segment (else its first, as all others')
  int row0, rows;  // first row of the pair, rows of the request
  int q0;          // first query of the request
  int pad[2];
};
constexpr int kMx4Jobs = 4096;
constexpr int kMx4WsHead = kMx4Jobs * sizeof(Mx4Job);

// A request's part of the batch.
struct Mx4Request {
  int q0, nq;        // first query, queries (max_q_len at most)
  int past;          // positions before the first query's own (negative: the first ones see nothing)
  int len;           // cached positions
  int list;          // first entry of its page list
};

__device__ __forceinline__ Mx4Request mx4_request(const Mx4AttendArgs& a, int b) {
  Mx4Request r;
  // (every offset within its range before any difference, which could wrap)
  const auto query = [&](int i) { return min(max(a.qo_indptr ? a.qo_indptr[i] : i, 0), a.T); };
  r.q0 = query(b);
  const int nq = max(query(b + 1) - r.q0, 0);
  r.nq = min(nq, a.max_q_len);
  r.list = max(a.kv_indptr[b], 0);
  const int64_t end = min((int64_t)max(a.kv_indptr[b + 1], 0), a.n_indices);
  const int64_t pages = max(end - r.list, (int64_t)0);
  const int64_t most = pages << a.page_shift;  // positions that the list reaches
  r.len = (int)max(min(min(a.kv_lens[b], most), (int64_t)0x3fffffff), (int64_t)0);
  r.past = r.len - nq;
  return r;
}

__device__ __forceinline__ int mx4_row_blocks(const Mx4Request& r, int H, int rows) { return (r.nq * H + rows - 1) / rows; }
__device__ __forceinline__ int mx4_tiles(const Mx4Request& r) { return max((r.len + kMx4Tile - 1) / kMx4Tile, 1); }

// Outputs v times f (one over the row's sum) as bf16. What is below 2^-94 is 0: there P with
// a scale taken from its exponents saturates at zero, and zeros with a scale added to
// theirs have gone into v as at most 2^-95.
template <bool FLUSH>
__device__ __forceinline__ u32x2 finish(f32x4 v, float f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] *= f;
    if (FLUSH && fabsf(v[i]) < 0x1p-94f) v[i] = 0.f;
  }
  return u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
}

// Inclusive sum over the lanes up to this one (DPP: shifts within rows of 16, then
// the rows' last lanes to the rows behind).
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);  // row_shr:1
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);  // row_bcast:15, rows 1 and 3
  v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);  // row_bcast:31, rows 2 and 3
  return v;
}

// Unit range of block j of n over `units`: [units j / n, units (j + 1) / n).
__device__ __forceinline__ uint32_t mx4_first_unit(uint32_t units, uint32_t j, uint32_t n) {
  return (uint32_t)((uint64_t)units * j / n);
}
// The block that has unit u.
__device__ __forceinline__ uint32_t mx4_block_of(uint32_t u, uint32_t units, uint32_t n) {
  return (uint32_t)((((uint64_t)u + 1) * n - 1) / units);
}

// PAGED: pages of 16 positions or more. A wave copies CT = 64 / W positions, 16 or 8,
// which then lie in one page: its number is a scalar, and the copies' offsets are the
// same for every tile. Otherwise the positions' page numbers come through LDS.
// LSE: for calls that ask for it, the sum of P before its rounding as well. In one
// kernel for both the largest prefill takes 4875 us for 4768, ragged chunks 844 for 821.
template <int D, int R, int G, bool PAGED, bool LSE>
__global__ __launch_bounds__(256, (Mx4Geo<D, R, G>::ACC ? 1 : 2)) void mx4_attend_kernel(Mx4AttendArgs a) {
  using Ge = Mx4Geo<D, R, G>;
  if constexpr (Ge::ACC) define_acc_macros();
  constexpr int W = Ge::W;
  constexpr int NB = Ge::NB, KS = Ge::KS, CB = Ge::CB, FT = Ge::FT, TW = Ge::TW, MT = Ge::MT, CT = Ge::CT, S = Ge::S;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_u8*)smem;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int la = lane & 15, gq = lane >> 4;
  const int gw = wave % G, tw = wave / G;  // this wave's group and its share of a tile's positions

  // ---- which units are this block's --------------------------------------------
  uint32_t u = 0, u_end = 1;
  uint32_t u_req = 0;  // first unit of request b
  uint32_t all_units = 0, all_blocks = 0;
  Mx4Job* jobs = nullptr;
  int b = 0, rb_only = 0;
  uint32_t pre = Ge::PRE;  // units before a pair's tiles, for its start and end
  Mx4Request rq = {};
  if (a.blocks > 0) {
    // Tiles of all requests, summed by every wave for itself (a request a lane, 256
    // requests' loads in one round trip), then the request that has the first unit.
    const auto units_of = [&](const Mx4Request& r, int i) {
      return i < a.B ? (uint32_t)mx4_row_blocks(r, a.H, Ge::ROWS) * ((uint32_t)mx4_tiles(r) + pre) : 0u;
    };
    Mx4Request r4[4];
    uint32_t n4[4], at4[4], units = 0;
    const auto load4 = [&](int c) {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k == 0 || c + 64 * k < a.B) r4[k] = mx4_request(a, min(c + 64 * k + lane, a.B - 1));
      if (a.B <= 256) {
        // pairs of one size that fill whole blocks, or blocks that fill whole pairs, stay so
        const uint32_t rb0 = __builtin_amdgcn_readfirstlane(mx4_row_blocks(r4[0], a.H, Ge::ROWS));
        const uint32_t nt0 = __builtin_amdgcn_readfirstlane(mx4_tiles(r4[0]));
        uint64_t other = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k == 0 || 64 * k < a.B)
            other |= __builtin_amdgcn_ballot_w64(64 * k + lane < a.B &&
                                                 ((uint32_t)mx4_row_blocks(r4[k], a.H, Ge::ROWS) != rb0 ||
                                                  (uint32_t)mx4_tiles(r4[k]) != nt0));
        const uint32_t pairs = a.B * rb0, n = min((uint32_t)a.blocks, pairs * nt0);
        if (other == 0 && pairs > 0 && (n % pairs == 0 || pairs % n == 0)) pre = 0;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        n4[k] = at4[k] = 0;
        if (k > 0 && c + 64 * k >= a.B) continue;
        n4[k] = units_of(r4[k], c + 64 * k + lane);
        const uint32_t incl = wave_scan(n4[k]);
        at4[k] = units + incl - n4[k];
        units += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
      }
    };
    for (int c = 0; c < a.B; c += 256) load4(c);
    const uint32_t nblk = min((uint32_t)a.blocks, units);
    // consecutive parts on one XCD (blocks go round the XCDs in turn): they share pages
    const uint32_t per = gridDim.x / 8;
    const uint32_t j = gridDim.x % 8 == 0 ? (blockIdx.x % 8) * per + blockIdx.x / 8 : blockIdx.x;
    jobs = reinterpret_cast<Mx4Job*>(a.ws);
    if (j >= nblk) {  // (also without any unit)
      if (!a.by_pair && tid == 0) jobs[j].parts = 0;
      return;
    }
    u = mx4_first_unit(units, j, nblk);
    u_end = mx4_first_unit(units, j + 1, nblk);
    a.blocks = (int)j;  // (from here on: this block's number)
    all_units = units;
    all_blocks = nblk;
    const bool again = a.B > 256;  // only the last 256 requests' sums are held
    if (again) units = 0;
    for (int c = 0; c < a.B; c += 256) {
      if (again) load4(c);  // (its running sum starts again)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint64_t hit = __builtin_amdgcn_ballot_w64(at4[k] <= u && u < at4[k] + n4[k]);
        if (hit) {
          const int l = __builtin_ctzll(hit);
          b = c + 64 * k + l;
          u_req = (uint32_t)__builtin_amdgcn_readlane((int)at4[k], l);
          rq.q0 = __builtin_amdgcn_readlane(r4[k].q0, l);
          rq.nq = __builtin_amdgcn_readlane(r4[k].nq, l);
          rq.past = __builtin_amdgcn_readlane(r4[k].past, l);
          rq.len = __builtin_amdgcn_readlane(r4[k].len, l);
          rq.list = __builtin_amdgcn_readlane(r4[k].list, l);
        }
      }
    }
  } else {
    // a block for each (request, row block), the later row blocks of a request,
    // which see most positions, first; request by request, so that each is
    // spread over the XCDs (blocks go round them in turn; requests in turn, in a multiple
    // of 8, would each lie on one: 32 ragged chunks, 40 heads, D = 256 8.9 ms for 3.9)
    const uint32_t j = blockIdx.y * gridDim.x + blockIdx.x;
    b = j / (uint32_t)a.row_blocks;
    if (b >= a.B) return;
    rb_only = a.row_blocks - 1 - (int)(j % (uint32_t)a.row_blocks);
    rq = mx4_request(a, b);
  }
  const bool shared = a.ws != nullptr;

  const uint32_t max_page = (uint32_t)((a.num_slots - 1) >> a.page_shift), max_slot = (uint32_t)(a.num_slots - 1);
  const uint32_t page_mask = (1u << a.page_shift) - 1;
  const float c2 = a.sm_scale * kLog2e;
  int nth = 0;  // segments done
  // A wave's copies of CT positions: RC (RR) rows of codes (rope) at a time, LC (LR)
  // lanes a row; chunk c of row t goes to chunk c ^ f(t), so that 16 lanes that read
  // one chunk of 16 rows, or 16 rows' parts of one block, meet all banks.
  constexpr int RC = 1024 / CB, LC = 64 / RC, RR = 1024 / (2 * R), LR = 64 / RR, LS = NB / 4;
  auto code_swz = [](int t) { return D == 512 ? t & 15 : (t >> 1) & 7; };
  auto rope_swz = [](int t) { return R == 64 ? (t >> 1) & 7 : (t >> 2) & 3; };
  auto code_off = [&](int j) {  // byte of copy j's piece within the CT rows
    const int t = RC * j + lane / LC;
    return t * CB + 16 * ((lane % LC) ^ code_swz(CT * wave + t));
  };
  auto rope_off = [&](int j) {
    const int t = RR * j + lane / LR;
    return t * 2 * R + 16 * ((lane % LR) ^ rope_swz(CT * wave + t));
  };
  const int scale_off = ((lane / LS) % CT) * NB + 4 * (lane % LS);

  while (u < u_end) {
    // ---- the next segment: tiles [t0, t1) of a row block of request b ---------------
    int rb, t0, t1, ntiles = mx4_tiles(rq);
    if (shared) {
      const uint32_t done = u - u_req, span = ntiles + pre;
      const int nrb = mx4_row_blocks(rq, a.H, Ge::ROWS), i = done / span;
      if (i >= nrb) {  // on to the next request (one without queries has no units)
        if (++b >= a.B) break;
        u_req = u;
        rq = mx4_request(a, b);
        continue;
      }
      // first and last row blocks in turns: the later ones see more positions
      rb = i & 1 ? nrb - 1 - (i >> 1) : i >> 1;
      const uint32_t at = done - i * span, n = min(span - at, u_end - u), u0 = u - at + pre;  // u0: its first tile
      u += n;
      t0 = max((int)(at - pre), 0);
      t1 = (int)(at + n - pre);
      if (t1 <= 0) continue;  // its tiles begin in the next block
      // The merge's job for this pair: by the block that begins it, or (by block) by the
      // one that takes it over from there.
      if (tid == 0 && (a.by_pair ? t0 == 0 : nth == 0)) {
        const uint32_t j1 = mx4_block_of(u0 + ntiles - 1, all_units, all_blocks);
        const uint32_t j0 = a.by_pair ? (uint32_t)a.blocks : mx4_block_of(u0, all_units, all_blocks);
        const bool cut = a.by_pair ? j1 > j0 : t0 > 0 && (int)j0 + 1 == a.blocks;
        jobs[a.by_pair ? b * a.row_blocks + rb : a.blocks] =
            Mx4Job{cut ? (int)(j1 - j0 + 1) : 0, (int)j0, mx4_first_unit(all_units, j0, all_blocks) < u0 - pre, rb * Ge::ROWS,
                   rq.nq * a.H, rq.q0, {0, 0}};
      }
    } else {
      u = u_end;
      rb = rb_only;
      if (rb >= mx4_row_blocks(rq, a.H, Ge::ROWS)) return;
      t0 = 0;
      t1 = ntiles;
    }
    const bool whole = t0 == 0 && t1 == ntiles;
    const int rows = rq.nq * a.H, row0 = rb * Ge::ROWS;
    // queries and heads of rows row0 + x, x < 64: one division, then exact products (row0 % H + x < 192)
    const int tok0 = row0 / a.H, head0 = row0 - tok0 * a.H;
    auto tok_of = [&](int x) { return tok0 + (((head0 + x) * a.h_inv) >> 16); };
    // positions that a row sees: its causal limit; rows past the last see none
    const int last_row = min(row0 + Ge::ROWS, rows) - 1;
    const int vis_all = rq.past + tok0 + 1;                // seen by every row of the block
    const int vis_most = rq.past + tok_of(last_row - row0) + 1;  // by any
    const int my_row = row0 + 16 * gw + la;
    const int my_tok = tok_of(16 * gw + la);
    const int vis = my_row < rows ? rq.past + my_tok + 1 : 0;
    const bool full_rows = row0 + Ge::ROWS <= rows;
    const int t_end = min(t1, (vis_most + kMx4Tile - 1) / kMx4Tile);
    const int nt = max(t_end - t0, 0);  // tiles to walk
    const int pos_last = max(rq.len - 1, 0);

    __syncthreads();  // the last segment's LDS reads are done

    // ---- page numbers and tiles, asynchronously ---------------------------------------
    const int list_last = pos_last & ~(CT - 1);  // (PAGED) first of the last CT positions
    auto page_of = [&](int k) -> uint32_t {  // PAGED: page of this wave's CT positions of tile k
      const int pos = min(kMx4Tile * (t0 + k) + CT * wave, list_last);
      return *(const __attribute__((address_space(4))) uint32_t*)(a.kv_indices + rq.list + (pos >> a.page_shift));
    };
    auto copy_idx = [&](int k) {
      const int pos = min(kMx4Tile * (t0 + k) + CT * wave + la % CT, pos_last);
      copy4(a.kv_indices + rq.list + (pos >> a.page_shift),
            lds0 + Ge::IDX + ((k & (kMx4Idx - 1)) * W + wave) * 256);
    };
    // Copies of tile k to the ring slot at byte `at`; `slot(x)`: cache slot of position x of this wave's CT.
    auto copy_slots = [&](uint32_t at, auto&& slot) {
      uint32_t sl[CT / RC + CT / RR + 1];
#pragma unroll
      for (int j = 0; j < CT / RC; ++j) sl[j] = slot(RC * j + lane / LC);
#pragma unroll
      for (int j = 0; j < CT / RR; ++j) sl[CT / RC + j] = slot(RR * j + lane / LR);
      sl[CT / RC + CT / RR] = slot((lane / LS) % CT);
#pragma unroll
      for (int j = 0; j < CT / RC; ++j)
        copy16(a.codes + (uint64_t)sl[j] * CB + code_off(j) % CB, at + CT * wave * CB + 1024 * j);
#pragma unroll
      for (int j = 0; j < CT / RR; ++j)
        copy16(reinterpret_cast<const uint8_t*>(a.rope) + (uint64_t)sl[CT / RC + j] * (2 * R) + rope_off(j) % (2 * R),
               at + Ge::CODES + CT * wave * 2 * R + 1024 * j);
      copy4(a.scales + (uint64_t)sl[CT / RC + CT / RR] * NB + 4 * (lane % LS), at + Ge::CODES + Ge::ROPE + 256 * wave);
    };
    auto copy_tile = [&](int k, uint32_t at, uint32_t page) {
      at += lds0;
      if constexpr (PAGED) {
        const int pos = min(kMx4Tile * (t0 + k) + CT * wave, list_last);
        const uint32_t s0 = (min(page, max_page) << a.page_shift) + ((uint32_t)pos & page_mask);
        if (__builtin_expect(s0 + CT - 1 <= max_slot, 1)) {
          const uint8_t* const c = a.codes + (uint64_t)s0 * CB;
          const uint8_t* const r = reinterpret_cast<const uint8_t*>(a.rope) + (uint64_t)s0 * (2 * R);
#pragma unroll
          for (int j = 0; j < CT / RC; ++j) copy16(c, (uint32_t)code_off(j), at + CT * wave * CB + 1024 * j);
#pragma unroll
          for (int j = 0; j < CT / RR; ++j)
            copy16(r, (uint32_t)rope_off(j), at + Ge::CODES + CT * wave * 2 * R + 1024 * j);
          copy4(a.scales + (uint64_t)s0 * NB, (uint32_t)scale_off, at + Ge::CODES + Ge::ROPE + 256 * wave);
        } else {  // the cache ends inside the page
          copy_slots(at, [&](int x) { return min(s0 + (uint32_t)x, max_slot); });
        }
      } else {
        const uint8_t* const idx = smem + Ge::IDX + ((k & (kMx4Idx - 1)) * W + wave) * 256;
        copy_slots(at, [&](int x) {
          const uint32_t p = *reinterpret_cast<const uint32_t*>(idx + 4 * x);
          const int pos = min(kMx4Tile * (t0 + k) + CT * wave + x, pos_last);
          return min((min(p, max_page) << a.page_shift) + ((uint32_t)pos & page_mask), max_slot);
        });
      }
    };

    // ---- the query rows of this wave's group: e4m3 hi and lo parts, rope ---------------
    i32x8 qhi[KS], qlo[KS];
    u32x4 qpe[R / 32];
    uint32_t qscale;
    u32x4 v[KS][2][2];
    {
      const bool mine = my_row < rows;  // (rows past the last: the pair's first row)
      const int tok = mine ? my_tok : tok0, head = mine ? head0 + 16 * gw + la - (my_tok - tok0) * a.H : head0;
      const uint16_t* q = a.q + (int64_t)(rq.q0 + tok) * a.q_st + (int64_t)head * a.q_sh;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // K index 64 h + 16 gq + i of step s is feature 32 (KS kb + s) + 16 (gq & 1) + i, kb = 2 h + gq / 2
          const uint16_t* p = q + 32 * (KS * (2 * h + (gq >> 1)) + s) + 16 * (gq & 1);
          v[s][h][0] = gload<u32x4>(p);
          v[s][h][1] = gload<u32x4>(p + 8);
        }
#pragma unroll
      for (int k = 0; k < R / 32; ++k) qpe[k] = gload<u32x4>(q + D + 32 * k + 8 * gq);
    }
    // The first tiles are asked for behind the query's loads; those are waited for here,
    // with the page numbers, so that no wait for them is left behind the tiles.
    uint32_t page = 0;  // PAGED: of the next tile to ask for
    if (nt > 0) {
      if constexpr (PAGED) {
        page = page_of(0);
      } else {
#pragma unroll 1
        for (int k = 0; k < S - 2; ++k) copy_idx(k);
      }
    }
    wait_loads<0>();
#pragma unroll
    for (int s = 0; s < KS; ++s)
      asm volatile("" : "+v"(v[s][0][0]), "+v"(v[s][0][1]), "+v"(v[s][1][0]), "+v"(v[s][1][1]));
#pragma unroll
    for (int k = 0; k < R / 32; ++k) asm volatile("" : "+v"(qpe[k]));
    uint32_t ask_at = 0;  // ring slot of the next tile to ask for
    auto next = [](uint32_t at) { return at + Ge::TILE == S * Ge::TILE ? 0u : at + Ge::TILE; };
    auto ask_tile = [&](int k) {
      if (k < nt) {
        const uint32_t p = page;
        if constexpr (PAGED) page = page_of(k + 1);
        copy_tile(k, ask_at, p);
        ask_at = next(ask_at);
      }
    };
    if (nt > 0) {
#pragma unroll 1
      for (int k = 0; k < S - 2; ++k) {
        if constexpr (!PAGED) copy_idx(k + S - 2);
        ask_tile(k);
      }
    }
    qscale = mx4_split<KS>(v, qhi, qlo);

    f32x4 o[G][FT];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < FT; ++j) o[g][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float ref[G];  // reference of row la of each group, the same in every wave
#pragma unroll
    for (int g = 0; g < G; ++g) ref[g] = kMx4NoRef;
    // this lane's sums (its positions of row la of group gw): of P as it is rounded, and (LSE) of P
    float psum = 0.f, ptile = 0.f, lsum = 0.f, ltile = 0.f, wref = kMx4NoRef;

    // The operands of 16 positions' scores (sub-tile m of this wave's MT) from the ring slot `at`.
    struct Keys {
      u32x4 code[KS], pe[R / 32];
      uint32_t scale;
    };
    auto read_keys = [&](uint32_t at, int m) {
      const uint8_t* const slot = smem + at;
      const int t = 16 * (tw * MT + m) + la;
      Keys kv;
#pragma unroll
      for (int s = 0; s < KS; ++s)
        kv.code[s] = *reinterpret_cast<const u32x4*>(slot + t * CB + 16 * ((gq * KS + s) ^ code_swz(t)));
      const uint8_t* const sp = slot + Ge::CODES + Ge::ROPE + 256 * (t / CT) + t % CT * NB + gq * KS;
      kv.scale = KS == 4 ? *reinterpret_cast<const uint32_t*>(sp) : *reinterpret_cast<const uint16_t*>(sp);
#pragma unroll
      for (int j = 0; j < R / 32; ++j)
        kv.pe[j] = *reinterpret_cast<const u32x4*>(slot + Ge::CODES + t * 2 * R + 16 * ((4 * j + gq) ^ rope_swz(t)));
      return kv;
    };
    // Their products with the query rows of this wave's group: the latent ones on e4m3
    // hi and lo, the rope ones on bf16. With a single sub-tile two chains take turns.
    auto products = [&](const Keys& kv) {
      f32x4 c = {0.f, 0.f, 0.f, 0.f}, d2 = {0.f, 0.f, 0.f, 0.f};
      f32x4& d = MT == 1 ? d2 : c;
      static_for<KS>([&](auto s) {
        c = mfma_fp4_fp8<s, 0>(kv.code[s], qhi[s], c, kv.scale, qscale);
        d = mfma_fp4_fp8<s, 1>(kv.code[s], qlo[s], d, kv.scale, qscale);
      });
#pragma unroll
      for (int j = 0; j < R / 32; ++j) d = mfma16x16x32(kv.pe[j], qpe[j], d);
      return MT == 1 ? c + d : c;
    };
    // Exponent fields of the scales of this wave's CT copied positions, (s - 63) << 7 or
    // (159 - s) << 7, to LDS buffer k & 1.
    auto scale_fields = [&](int k, uint32_t at) {
      if (CT * LS == 64 || lane < CT * LS) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(smem + at + Ge::CODES + Ge::ROPE + 256 * wave + 4 * lane);
        uint16_t* const es =
            reinterpret_cast<uint16_t*>(smem + Ge::ES + (k & 1) * NB * 128) + 4 * (lane % LS) * 64 + CT * wave + lane / LS;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = (int)((w >> (8 * i)) & 255u);
          es[64 * i] = (uint16_t)((Ge::VSIDE ? min(max(c - kMx4Low, 0), kMx4High - kMx4Low) : max(kMx4High - c, 0)) << 7);
        }
      }
    };
    // What is rare about tile k's scores: positions that not every row sees, and a
    // score that passes its row's reference by more than the slack. The wave's flag
    // and its reference go to LDS buffer k & 1.
    auto look = [&](int k, f32x4 (&acc)[MT]) {
      const int p0 = kMx4Tile * (t0 + k), buf = k & 1;
      if (__builtin_expect(!full_rows || p0 + kMx4Tile > vis_all, 0)) {
        asm volatile("");  // (a branch: most tiles have nothing to mask)
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (p0 + 16 * (tw * MT + m) + 4 * gq + i >= vis) acc[m][i] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, acc[m][i]);
      mx *= c2;
      wref = ref[gw];
      const bool moved = __builtin_amdgcn_ballot_w64(mx > wref + kMx4Slack) != 0;
      if (__builtin_expect(moved, 0)) {
        const float top = wave_max_over_groups(mx);
        if (top > wref + kMx4Slack) wref = ceilf(top);
        if (gq == 0) *reinterpret_cast<float*>(smem + Ge::WREF + 64 * W * buf + 64 * wave + 4 * la) = wref;
      }
      if (lane == 0) *reinterpret_cast<uint32_t*>(smem + Ge::FLAG + 4 * W * buf + 4 * wave) = moved;
    };
    // Probabilities of tile k, to LDS buffer k & 1.
    auto softmax = [&](int k, const f32x4 (&acc)[MT]) {
      // (the score rounded before the difference, as in the reference: fused, one of
      // 2^31 and more could pass its own maximum by 2^7)
#pragma clang fp contract(off)
      ltile = ptile = 0.f;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p[i] = __builtin_amdgcn_exp2f(acc[m][i] * c2 - wref);
          if constexpr (LSE) ltile += p[i];
        }
        const u32x2 w = {pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3])};
        ptile += sum_bf16x2(w.y, sum_bf16x2(w.x, 0.f));
        // chunk (8 positions) c of a row at c ^ (row & 7)
        const int c = 2 * (tw * MT + m) + (gq >> 1);
        *reinterpret_cast<u32x2*>(smem + Ge::P + (k & 1) * Ge::ROWS * 128 + (16 * gw + la) * 128 + 16 * (c ^ (la & 7)) +
                                  8 * (gq & 1)) = w;
      }
    };
    // P of tile k: row la of group g, positions 16 gq + 8 h .. + 7.
    auto read_p = [&](int k, int g, int h) {
      return *reinterpret_cast<const u32x4*>(smem + Ge::P + (k & 1) * Ge::ROWS * 128 + (16 * g + la) * 128 +
                                             16 * ((2 * gq + h) ^ (la & 7)));
    };
    struct Flags {
      uint32_t of[W];
    };
    auto read_flags = [&](int k) {
      Flags f;
#pragma unroll
      for (int w = 0; w < W; ++w) f.of[w] = reinterpret_cast<const uint32_t*>(smem + Ge::FLAG + 4 * W * (k & 1))[w];
      return f;
    };
    // The common references of tile k: where a wave has moved one (not 0 returned), all
    // go to the largest, and what was computed against smaller ones is scaled down
    // by powers of two, earlier sums here, P by `lower` with `down`.
    uint32_t down[G];  // by how many powers of two a group's P of this lane's positions falls
    auto agree = [&](int k, const Flags& fl) {
      const int buf = k & 1;
      uint32_t any = 0;
#pragma unroll
      for (int w = 0; w < W; ++w) any |= fl.of[w];
      const uint32_t moved = __builtin_amdgcn_readfirstlane(any);
      float fall[G];  // factor by which a group's earlier sums fall
#pragma unroll
      for (int g = 0; g < G; ++g) fall[g] = 1.f;
#pragma unroll
      for (int g = 0; g < G; ++g) down[g] = 0;
      if (__builtin_expect(moved != 0, 0)) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float mine[TW], top = ref[g];
#pragma unroll
          for (int w = 0; w < TW; ++w) {
            const int wv = w * G + g;
            const float r = *reinterpret_cast<const float*>(smem + Ge::WREF + 64 * W * buf + 64 * wv + 4 * la);
            mine[w] = fl.of[wv] ? r : ref[g];
            top = fmaxf(top, mine[w]);
          }
          fall[g] = __builtin_amdgcn_exp2f(ref[g] - top);
          if constexpr (!Ge::ACC) {
#pragma unroll
            for (int j = 0; j < FT; ++j) o[g][j] *= fall[g];
          }
          float r = mine[0];  // of the wave that made this lane's 16 positions
#pragma unroll
          for (int w = 1; w < TW; ++w) r = gq * TW / 4 == w ? mine[w] : r;
          const uint32_t d = (uint32_t)fminf(top - r, 511.f) << 7;
          down[g] = d | d << 16;
          if (g == gw) {
            const float f = __builtin_amdgcn_exp2f(wref - top);
            psum *= fall[g];
            ptile *= f;
            if constexpr (LSE) {
              lsum *= fall[g];
              ltile *= f;
            }
          }
          ref[g] = top;
        }
      }
      if constexpr (Ge::ACC) {
#pragma unroll
        for (int g = 0; g < G; ++g) scale_acc8(o[g], fall[g], moved);
      }
      if constexpr (LSE) lsum += ltile;
      psum += ptile;
      return moved;
    };
    auto lower = [&](u32x4& p, uint32_t d) {
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = sub_sat(p[i], d);
    };
    // (MIX) 32 of this wave's features of tile k (scale block bb of its FT / 2), as they lie in the
    // ring slot `at`, and as bf16 with the scales in their exponents: positions 16 gq .. + 15
    // (two halves) of feature la of two output tiles.
    struct Raw {
      u32x4 e[2];
      i32x2 v[2];
    };
    auto read_raw = [&](int k, uint32_t at, int bb) {
      const int t = 16 * gq + la, nb = wave * (FT / 2) + bb;
      const u32x4* const es = reinterpret_cast<const u32x4*>(smem + Ge::ES + (k & 1) * NB * 128 + nb * 128 + 32 * gq);
      Raw r;
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        r.e[f] = es[f];
        r.v[f] = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
            (__attribute__((address_space(3))) i32x2*)(smem + at + t * CB + 16 * (nb ^ code_swz(t)) + 8 * f));
      }
      return r;
    };
    auto expand = [&](const Raw& r, u32x4 (&x0)[2], u32x4 (&x1)[2]) {
      x0[0] = fp4x8_to_bf16((uint32_t)r.v[0].x);
      x0[1] = fp4x8_to_bf16((uint32_t)r.v[0].y);
      x1[0] = fp4x8_to_bf16((uint32_t)r.v[1].x);
      x1[1] = fp4x8_to_bf16((uint32_t)r.v[1].y);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x0[h][i] = add16(x0[h][i], r.e[h][i]);
          x1[h][i] = add16(x1[h][i], r.e[h][i]);
        }
    };
    // O^T += X^T P^T of tile k, with N halves (8 of a lane's 16 positions) of P at a time.
    auto outputs = [&](int k, uint32_t at) {
      constexpr int N = Ge::PH;
      u32x4 p[G][N];
      auto read_ps = [&](int h0) {
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int h = 0; h < N; ++h) p[g][h] = read_p(k, g, h0 + h);
      };
      const Flags fl = read_flags(k);
      read_ps(0);
      const uint32_t moved = agree(k, fl);
      const int t = 16 * gq + la;
      u32x2 x[FT];  // 16 positions of feature la of each output tile
      auto read_x = [&](int j) {
        x[j] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr4_b64_v2i32(
            (__attribute__((address_space(3))) i32x2*)(smem + at + t * CB + 16 * ((wave * (FT / 2) + j / 2) ^ code_swz(t)) +
                                                       8 * (j % 2))));
      };
      if constexpr (N == 1) {
#pragma unroll
        for (int j = 0; j < FT; ++j) read_x(j);
      }
#pragma unroll
      for (int h0 = 0; h0 < 2; h0 += N) {
        if (h0) read_ps(h0);
        if (__builtin_expect(moved != 0, 0)) {
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int h = 0; h < N; ++h) lower(p[g][h], down[g]);
        }
#pragma unroll
        for (int bb = 0; bb < FT / 2; ++bb) {
          if constexpr (N == 2) {
            read_x(2 * bb);
            read_x(2 * bb + 1);
          }
          const uint8_t* const es = smem + Ge::ES + (k & 1) * NB * 128 + (wave * (FT / 2) + bb) * 128 + 32 * gq + 16 * h0;
#pragma unroll
          for (int h = 0; h < N; ++h) {
            const u32x4 e = *reinterpret_cast<const u32x4*>(es + 16 * h);
            const uint32_t w0 = x[2 * bb][h0 + h], w1 = x[2 * bb + 1][h0 + h];
            u32x4 x0 = fp4x8_to_bf16(w0), x1 = fp4x8_to_bf16(w1);
            if constexpr (Ge::VSIDE) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                x0[i] = add16(x0[i], e[i]);
                x1[i] = add16(x1[i], e[i]);
              }
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
              u32x4 q = p[g][h];
              if constexpr (!Ge::VSIDE) {
#pragma unroll
                for (int i = 0; i < 4; ++i) q[i] = sub_sat(q[i], e[i]);
              }
              o[g][2 * bb] = mfma16x16x32(x0, q, o[g][2 * bb]);
              o[g][2 * bb + 1] = mfma16x16x32(x1, q, o[g][2 * bb + 1]);
            }
          }
        }
      }
    };

    // ---- the tile loop -------------------------------------------------------------
    // Copies in order: before the loop tiles 0 .. S - 3, in turn k (after barrier k)
    // tile k + S - 1, each (without PAGED) behind the page numbers of the tile S - 2
    // later. Barrier k waits until tile k + 1 is in; then tiles k + 2 .. k + S - 2 may
    // be on their way. Turn k has tile k's output and tile k + 1's scores.
    constexpr int IC = PAGED ? 0 : S - 3;  // page number copies behind tile k + 1
    uint32_t here = 0, ahead = 0;          // ring slots of tiles k and k + 1
    auto meet = [&](int k) {
      const int there = nt - 2 - k;  // tiles past k + 1
      if (there >= S - 3) {
        wait_loads<IC + (S - 3) * Ge::LOADS>();
      } else if (S > 4 && there == 1) {
        wait_loads<IC + Ge::LOADS>();
      } else {
        wait_loads<IC>();
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };
    auto ask = [&](int k) {
      if constexpr (!PAGED) copy_idx(k + 2 * S - 3);
      ask_tile(k + S - 1);
    };
    if (nt > 0) {
      f32x4 acc[MT];
      meet(-1);
      ask(-1);
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[m] = products(read_keys(0, m));
      scale_fields(0, 0);
      look(0, acc);
      softmax(0, acc);
#pragma unroll 1
      for (int k = 0; k < nt - 1; ++k) {
        here = ahead;
        ahead = next(ahead);
        meet(k);
        if constexpr (Ge::MIX) {
          constexpr int STEPS = MT > FT / 2 ? MT : FT / 2;
          u32x4 p[G][2], x[FT][2];
          // first part: the LDS reads of a step go out a step ahead of it
          const Flags fl = read_flags(k);
#pragma unroll
          for (int g = 0; g < G; ++g)
#pragma unroll
            for (int h = 0; h < 2; ++h) p[g][h] = read_p(k, g, h);
          Keys keys = read_keys(ahead, 0);
          Raw raw = read_raw(k, here, 0);
          ask(k);
          if (__builtin_expect(agree(k, fl) != 0, 0)) {
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
              for (int h = 0; h < 2; ++h) lower(p[g][h], down[g]);
          }
#pragma unroll
          for (int i = 0; i < STEPS; ++i) {
            Keys keys2;
            Raw raw2;
            if (i + 1 < MT) keys2 = read_keys(ahead, i + 1);
            if (i + 1 < FT / 2) raw2 = read_raw(k, here, i + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (i < MT) acc[i] = products(keys);
            if (i < FT / 2) expand(raw, x[2 * i], x[2 * i + 1]);
            if (i + 1 == STEPS) scale_fields(k + 1, ahead);
            if (i + 1 < MT) keys = keys2;
            if (i + 1 < FT / 2) raw = raw2;
          }
          // second part
          look(k + 1, acc);
#pragma unroll
          for (int j = 0; j < FT; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int g = 0; g < G; ++g) o[g][j] = mfma16x16x32(x[j][h], p[g][h], o[g][j]);
          softmax(k + 1, acc);
        } else {
          ask(k);
          outputs(k, here);
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m] = products(read_keys(ahead, m));
          scale_fields(k + 1, ahead);
          look(k + 1, acc);
          softmax(k + 1, acc);
        }
      }
      meet(nt - 1);
      outputs(nt - 1, ahead);
    }
    if constexpr (!PAGED) wait_loads<0>();  // (page numbers asked for past the end)

    // ---- the rows' sums, then the output or a partial --------------------------------
    if constexpr (LSE) lsum = wave_sum_over_groups(lsum);
    psum = wave_sum_over_groups(psum);
    if (gq == 0) *reinterpret_cast<f32x2*>(smem + Ge::LSUM + 128 * wave + 8 * la) = f32x2{lsum, psum};
    __syncthreads();
#pragma unroll
    for (int g = 0; g < G; ++g) {
      f32x2 l = {0.f, 0.f};
#pragma unroll
      for (int w = 0; w < TW; ++w) {
        const f32x2 v = *reinterpret_cast<const f32x2*>(smem + Ge::LSUM + 128 * (w * G + g) + 8 * la);
        l = f32x2{l.x + v.x, l.y + v.y};
      }
      const int r = row0 + 16 * g + la;
      if (r >= rows) continue;
      const int tq = tok_of(16 * g + la), tok = rq.q0 + tq, head = head0 + 16 * g + la - (tq - tok0) * a.H;
      if (whole) {
        const float inv = l.y == 0.f ? 0.f : Ge::UNIT / l.y;
        uint16_t* const out = a.out + (int64_t)tok * a.o_st + (int64_t)head * a.o_sh + Ge::FW * wave + 4 * gq;
#pragma unroll
        for (int j = 0; j < FT; ++j) {
          *reinterpret_cast<u32x2*>(out + 16 * j) = finish<Ge::VSIDE>(o[g][j], inv);
        }
        if (LSE && wave == 0 && gq == 0)
          a.lse[(int64_t)tok * a.H + head] = l.x == 0.f ? -INFINITY : (ref[g] + log2f(l.x)) * kLn2;
      } else {
        uint8_t* const part = a.ws + kMx4WsHead + ((int64_t)2 * a.blocks + (nth > 0)) * Ge::SLOT;
        float* const po = reinterpret_cast<float*>(part) + (16 * g + la) * D + Ge::FW * wave + 4 * gq;
#pragma unroll
        for (int j = 0; j < FT; ++j) *reinterpret_cast<f32x4*>(po + 16 * j) = o[g][j] * Ge::UNIT;
        if (wave == 0 && gq == 0) {
          reinterpret_cast<f32x2*>(part + Ge::ROWS * D * 4)[16 * g + la] = f32x2{ref[g], l.y};
          if constexpr (LSE) reinterpret_cast<float*>(part + Ge::ROWS * (D + 2) * 4)[16 * g + la] = l.x;
        }
      }
    }
    ++nth;
  }
  if (shared && !a.by_pair && nth == 0 && tid == 0) jobs[a.blocks].parts = 0;
}

// Joins the partials of the pairs that were cut: a block for a job, 4 C columns and
// THREADS / (C PARTS) rows, C threads for each of PARTS shares of a row's partials, four
// of them in flight for each. What bounds it is latency (the job, then the partials), so
// blocks are small enough to be on the card all at once.
template <int D, int C, int PARTS, int THREADS>
__global__ __launch_bounds__(THREADS) void mx4_merge_kernel(Mx4AttendArgs a, int rows_per_block) {
  constexpr int N = 4, RM = THREADS / C / PARTS;
  static_assert(PARTS == 1 || RM == 1, "blocks with several shares leave as one");
  __shared__ f32x4 s_o[PARTS][C];
  __shared__ f32x2 s_ml[PARTS];
  __shared__ float s_ls[PARTS];
  const Mx4Job job = reinterpret_cast<const Mx4Job*>(a.ws)[blockIdx.x];
  if (a.by_pair) {  // (pairs that there are not: their jobs are not written)
    const int b = blockIdx.x / a.row_blocks;
    const Mx4Request rq = mx4_request(a, b);
    if ((int)(blockIdx.x % a.row_blocks) >= mx4_row_blocks(rq, a.H, rows_per_block)) return;
  }
  const int c = threadIdx.x % C, col = 4 * (C * blockIdx.z + c);
  const int unit = C % 64 == 0 ? __builtin_amdgcn_readfirstlane(threadIdx.x / C) : threadIdx.x / C;
  const int part = unit % PARTS, rl = blockIdx.y * RM + unit / PARTS, r = job.row0 + rl;
  if (job.parts == 0 || r >= job.rows || rl >= rows_per_block) return;
  const int64_t slot = (int64_t)rows_per_block * (D + 3) * 4;
  const uint8_t* const parts = a.ws + kMx4WsHead + 2 * job.first * slot;
  float m = kMx4NoRef, l = 0.f, lse = 0.f;  // reference, sums of P as it was rounded and (for an LSE) of P
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int j = part; j < job.parts; j += N * PARTS) {
    f32x2 ml[N];
    float ls[N];
    f32x4 v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int jj = min(j + i * PARTS, job.parts - 1);
      const uint8_t* const p = parts + (2 * jj + (jj == 0 ? job.second : 0)) * slot;
      ml[i] = gload<f32x2>(p + (int64_t)rows_per_block * D * 4 + 8 * rl);
      ls[i] = a.lse ? gload<float>(p + (int64_t)rows_per_block * (D + 2) * 4 + 4 * rl) : 0.f;
      v[i] = gload<f32x4>(p + ((int64_t)rl * D + col) * 4);
    }
    float top = m;
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, ml[i].x);
    const float f = __builtin_amdgcn_exp2f(m - top);
    l *= f;
    lse *= f;
    o *= f;
    m = top;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (j + i * PARTS < job.parts) {
        const float w = __builtin_amdgcn_exp2f(ml[i].x - top);
        l = fmaf(w, ml[i].y, l);
        lse = fmaf(w, ls[i], lse);
        o += v[i] * w;
      }
    }
  }
  if constexpr (PARTS > 1) {
    s_o[part][c] = o;
    if (c == 0) {
      s_ml[part] = f32x2{m, l};
      s_ls[part] = lse;
    }
    __syncthreads();
    if (part) return;
    float top = m;
#pragma unroll
    for (int i = 1; i < PARTS; ++i) top = fmaxf(top, s_ml[i].x);
    const float f = __builtin_amdgcn_exp2f(m - top);
    l *= f;
    lse *= f;
    o *= f;
    m = top;
#pragma unroll
    for (int i = 1; i < PARTS; ++i) {
      const float w = __builtin_amdgcn_exp2f(s_ml[i].x - top);
      l = fmaf(w, s_ml[i].y, l);
      lse = fmaf(w, s_ls[i], lse);
      o += s_o[i][c] * w;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int tok = job.q0 + r / a.H, head = r % a.H;
  *reinterpret_cast<u32x2*>(a.out + (int64_t)tok * a.o_st + (int64_t)head * a.o_sh + col) = finish<true>(o, inv);
  if (a.lse && col == 0) a.lse[(int64_t)tok * a.H + head] = lse == 0.f ? -INFINITY : (m + log2f(lse)) * kLn2;
}

template <int D, int R, int G, bool PAGED, bool LSE>
hipError_t launch_attend(Mx4AttendArgs a, int num_cus, hipStream_t stream) {
  using Ge = Mx4Geo<D, R, G>;
  const int64_t rows = (int64_t)a.max_q_len * a.H;
  a.row_blocks = (int)((rows + Ge::ROWS - 1) / Ge::ROWS);
  a.h_inv = (65536 + a.H - 1) / a.H;
  // Shared out, but for more requests than a block's sums hold, more tiles than 32 bits
  // count, and, where two blocks run on a CU, more than 4 row blocks for each CU: those
  // have a block each. What sharing costs is a block's sums, an even batch's cuts and, in
  // chunks without a prefix, tiles that a row block does not see; what it brings is even
  // work, the more the fewer row blocks there are to even it out, and lengths are not known here.
  // us, shared out / a block each, by row blocks for a CU, 256 CUs. D = 256, 40 heads: ragged
  // chunks behind prefixes 2.0 215 / 240, 2.5 266 / 328, 3.9 334 / 388, 7.6 653 / 675, 9.2
  // 798 / 738, 21 2186 / 1982; of one length 2.0 185 / 182, 4.0 332 / 320, 8 592 / 567, 24
  // 1916 / 1796; from their start 2.0 27.7 / 21.7, 4.0 43.6 / 41.6, 11 122 / 104; decode 1.3
  // 132 / 154, 2.5 241 / 271; 16 heads, ragged 2.6 196 / 223, 3.7 337 / 341, 5.4 526 / 499,
  // 16 1770 / 1578. D = 512: 128 heads, ragged 1.0 213 / 302, 2.9 471 / 539, 7.6 1237 / 1330,
  // 16 2537 / 2600; of one length 1.0 180 / 172, 4.0 586 / 582, 12 1752 / 1764; from their
  // start 1.0 28.5 / 19.9, 4.0 77 / 72, 8 147 / 149; decode 2.0 216 / 274, 8 791 / 871; 16
  // heads, ragged 2.4 440 / 435, 6.9 1414 / 1473, 20 4005 / 3599.
  const int64_t items = ((int64_t)a.T * a.H + Ge::ROWS - 1) / Ge::ROWS;
  const int64_t most_tiles = (a.n_indices << a.page_shift) / kMx4Tile + (int64_t)(1 + Ge::PRE) * a.B;
  const bool shared = a.B <= kMx4Requests && (Ge::OCC == 1 || items <= 4 * (int64_t)num_cus) && most_tiles < ((int64_t)1 << 32) / a.row_blocks;
  const hipError_t e = hipFuncSetAttribute((const void*)mx4_attend_kernel<D, R, G, PAGED, LSE>,
                                           hipFuncAttributeMaxDynamicSharedMemorySize, Ge::LDS);
  if (e != hipSuccess) return e;
  if (!shared) {
    a.ws = nullptr;
    a.blocks = 0;
    // (in two dimensions: 2^24 blocks of 256 threads are too many for one)
    const int64_t blocks = (int64_t)a.row_blocks * a.B, x = std::min<int64_t>(blocks, 1 << 22);
    hipLaunchKernelGGL((mx4_attend_kernel<D, R, G, PAGED, LSE>), dim3((unsigned)x, (unsigned)((blocks + x - 1) / x)), dim3(256),
                       Ge::LDS, stream, a);
    return hipGetLastError();
  }
  a.blocks = std::min(num_cus * Ge::OCC, kMx4Jobs);
  const int64_t pairs = (int64_t)a.B * a.row_blocks;
  a.by_pair = pairs <= a.blocks;
  hipLaunchKernelGGL((mx4_attend_kernel<D, R, G, PAGED, LSE>), dim3(a.blocks), dim3(256), Ge::LDS, stream, a);
  hipError_t rc = hipGetLastError();
  if (rc != hipSuccess) return rc;
  // Partials of a row: 16 and more in U shares of whole rows, 16 U and more (a few pairs) in 16
  // shares of 128 columns, fewer in one. Both kernels at D = 512, 16 heads, 8192 positions, by the last two: 1
  // request 21.5 us for 40.8, 8 20.3 for 24.7, 16 24.4 for 26.1, 32 34.8 for 35.1, and 32 with 128
  // heads 99.7 for 93.2; by the first two: 1 request 16.9 for 21.2 (of 16384 positions 19.5
  // for 29.3), 4 17.3 for 18.7, 8 20.3 for 20.2, 16 25.2 for 24.2.
  const int64_t there = std::min<int64_t>(rows, Ge::ROWS), jobs = a.by_pair ? pairs : a.blocks;
  constexpr int RM = 256 / (D / 4), U = 512 / (D / 4);
  if (pairs * 16 * U <= a.blocks)
    hipLaunchKernelGGL((mx4_merge_kernel<D, 32, 16, 512>), dim3(jobs, there, D / 128), dim3(512), 0, stream, a, Ge::ROWS);
  else if (pairs * 16 <= a.blocks)
    hipLaunchKernelGGL((mx4_merge_kernel<D, D / 4, U, 512>), dim3(jobs, there), dim3(512), 0, stream, a, Ge::ROWS);
  else
    hipLaunchKernelGGL((mx4_merge_kernel<D, D / 4, 1, 256>), dim3(jobs, (there + RM - 1) / RM), dim3(256), 0, stream, a,
                       Ge::ROWS);
  return hipGetLastError();
}

template <int D, int R, int G>
hipError_t launch_paged(const Mx4AttendArgs& a, int num_cus, hipStream_t stream) {
  if (a.lse)
    return a.page_shift >= 4 ? launch_attend<D, R, G, true, true>(a, num_cus, stream)
                             : launch_attend<D, R, G, false, true>(a, num_cus, stream);
  return a.page_shift >= 4 ? launch_attend<D, R, G, true, false>(a, num_cus, stream)
                           : launch_attend<D, R, G, false, false>(a, num_cus, stream);
}

}  // namespace rolaq

int64_t rolaq_mx4_attend_ws_bytes(int D, int num_cus) {
  using namespace rolaq;
  // two partials of 64 rows a block
  return kMx4WsHead + (D == 512 ? (int64_t)2 * num_cus * Mx4Geo<512, 64, 4>::OCC * Mx4Geo<512, 64, 4>::SLOT
                                : (int64_t)2 * num_cus * Mx4Geo<256, 32, 4>::OCC * Mx4Geo<256, 32, 4>::SLOT);
}

hipError_t rolaq_launch_mx4_attend(const rolaq::Mx4AttendArgs& a, int D, int num_cus, hipStream_t stream) {
  using namespace rolaq;
  const int64_t rows = (int64_t)a.max_q_len * a.H;
  // As few groups as hold a request's rows. us, of 32 x 4096 positions, for four groups' kernel:
  // 16 rows at D = 512 24.5 / 36.3, at 256 17.5 / 22.8; 32 rows 31.7 / 39.4 and 22.4 / 25.5.
#define ROLAQ_MX4(DD, RR)                                                    \
  if (D == DD) {                                                             \
    if (rows <= 16) return launch_paged<DD, RR, 1>(a, num_cus, stream);      \
    if (rows <= 32) return launch_paged<DD, RR, 2>(a, num_cus, stream);      \
    return launch_paged<DD, RR, 4>(a, num_cus, stream);                      \
  }
  ROLAQ_MX4(512, 64)
  ROLAQ_MX4(256, 32)
#undef ROLAQ_MX4
  return hipErrorInvalidValue;
}
