// Attention weight of every cached position of the MX4 latent cache (gfx950), summed over a
// request's query rows (queries and heads):
//   acc_t (+)= sum over the rows that see t of exp(sm_scale (q_lat . x_t + q_pe . r_t) - lse),
// lse the row's log sum of exponentials as the attention call returned it.
//
// The positions are what a wave holds: it loads the codes of 16 MT positions straight into
// registers, expands them to bf16 (v_cvt_scalef32_pk_bf16_fp4, exact) and goes through the query
// rows, which lie in LDS as they are, 16 at a time, on bf16 MFMA. A position's sum stays in its
// lanes until the rows are through, so that each is written once, by one lane, in an
// order that no other request or launch shape changes (but for parts of many rows, whose sums are joined in
// their order). (The scores of the attention itself, 4-bit
// codes against a query split into two e4m3 parts, are off by 2^-18 of the largest: the weights
// were off by 1e-5, now by 3e-7.)
//
// Few rows (64 at most, a decode step): a block keeps them in LDS and walks a range of the batch's
// tiles, expanding as it multiplies; bound by the cache's bytes: 49 us for 32 requests of 16384
// positions under 16 heads of width 512, 210 MB at 4.3 TB/s. Many rows (the last queries of prompts): a
// wave keeps its positions expanded in registers, and the rows come to LDS 64 at a time (32 of width
// 512) while the last ones are in use, the weights of 16 rows between the products of the next 16; bound by
// the matrix instructions, their operands' reads and the exponentials in turn: 88 to 91 us (95 under the profiler) for
// 32 queries of 40 heads of width 256 in 8 requests of 8192 to 16384 positions, 69 GFLOP; 73 with the products alone,
// 17 with one step alone (139 with 16 rows at a time and tiles of 256 positions a block, of which a part of
// the blocks had one and the rest two). At width 256 46 registers are spilled there, which steps load before their
// products; none within them.
#include "rolaq_common.h"
#include "mx4_args.h"
#include "mx4_request.h"
#include "mx4_tile.h"

#include <algorithm>
#include <cmath>

namespace rolaq {

typedef __attribute__((address_space(3))) uint8_t lds_byte;

template <int D, int R>
struct WGeo {
  static constexpr int W = 4;  // waves
  static constexpr int NB = D / 32, CB = D / 2;
  static constexpr int JS = D / 128;        // code loads of a position: lane group gq has block 4 j + gq
  static constexpr int RS = R / 32;         // K-steps of the rope scores
  static constexpr int RC = (D + R) / 8;    // 16-byte chunks of a query row
  static constexpr int QT = 16 * 16 * RC;   // bytes of 16 query rows
  static constexpr int QR = D == 512 ? 32 : 64;  // rows in LDS at a time where they are streamed
  static constexpr int STEP = QR / 16 * QT;      // their bytes
  static_assert(STEP == 9 * W * 1024, "nine copies of 1 KB a wave, of whole rows");
};
constexpr int kWeightsFew = 64;  // the most rows of a request that stay in LDS

// Chunk c of query row r (of 16) lies at chunk c ^ w_swz(r): the 16 rows of a chunk meet all banks.
template <int D>
__device__ __forceinline__ int w_swz(int r) { return D == 512 ? (r >> 1) & 7 : (r >> 2) & 3; }

// Eight codes -> eight bf16 values, times f.
__device__ __forceinline__ u32x4 w_expand(uint32_t v, float f) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, f, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, f, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, f, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, f, 3))};
}

// Sum over the 16 lanes of a row of lanes, the same bits on each of them: both sides of an exchange add the same
// two sums. (Which lane writes a position follows from where its tile starts, so from the batch; sums of rotated lanes
// differed by lane in their last bit.)
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float row_sum16(float v) {
  v = add_dpp<0xB1>(v);     // quad_perm 1, 0, 3, 2
  v = add_dpp<0x4E>(v);     // quad_perm 2, 3, 0, 1
  v = add_dpp<0x141>(v);    // row_half_mirror: the other four of eight
  return add_dpp<0x140>(v);  // row_mirror: the other eight
}

// QT > 0: at most 16 QT rows a request, kept in LDS; 0: any number, streamed.
template <int D, int R, int MOST, int QT>
__global__ __launch_bounds__(256, 2) void mx4_weights_kernel(Mx4WeightsArgs a) {
  using G = WGeo<D, R>;
  constexpr int NB = G::NB, CB = G::CB, RS = G::RS, W = G::W, JS = G::JS, RC = G::RC;
  // A batch is shared out among the blocks in units of positions: whole tiles of MOST sub-tiles a wave where the rows
  // are few; single sub-tiles a wave where they are many, for blocks to end together.
  constexpr int TILE = 16 * W * (QT > 0 ? MOST : 1);
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_byte*)smem;
  const int lane = threadIdx.x & 63, la = lane & 15, gq = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // ---- this block's part of the batch's tiles -------------------------------------
  // positions of request i that count
  const auto places = [&](int i, const Mx4Request& r) {
    const int64_t row = a.req_idx ? a.req_idx[i] : i;
    return row >= 0 && row < a.acc_rows ? (int)min((int64_t)r.len, a.acc_cols) : 0;
  };
  const auto tiles_of = [&](int i) {
    return i < a.B ? (uint32_t)((places(i, mx4_request(a, i)) + TILE - 1) / TILE) : 0u;
  };
  // what one of them costs: many rows, the steps over them
  const auto cost_of = [&](int i) {
    if (QT > 0 || i >= a.B) return 1u;
    const int steps = (mx4_request(a, i).nq * a.H + G::QR - 1) / G::QR;
    return (uint32_t)(steps >> a.cost_shift) + 1u;
  };
  uint32_t total = 0;
  for (int c = 0; c < a.B; c += 64)
    total += (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(tiles_of(c + lane) * cost_of(c + lane)), 63);
  // (each part of the rows is all blocks' over again; neighbours on one XCD: they read the same query rows)
  const uint32_t blocks = QT > 0 ? gridDim.x : gridDim.x / (uint32_t)a.parts, per = blocks / 8;
  const uint32_t part = QT > 0 ? 0u : blockIdx.x / blocks, in_part = blockIdx.x - part * blocks;
  const uint32_t j = blocks % 8 == 0 ? (in_part % 8) * per + in_part / 8 : in_part;
  const uint32_t nb = min(blocks, total);
  if (j >= nb) return;
  // The units of a request (n, from `start` in the batch's cost) that are this block's. Few rows: an even part of
  // the batch. Many: a block that took a request's last units and the next one's first would go through two
  // requests' rows and end last, so each request has blocks of its own, as many as its part of the cost says, and
  // one too small for that goes to the block before which it ends.
  const auto share = [&](uint32_t start, uint32_t n, uint32_t cost, uint32_t& t0, uint32_t& t1) {
    if constexpr (QT > 0) {
      const uint32_t lo = (uint32_t)((uint64_t)total * j / nb), hi = (uint32_t)((uint64_t)total * (j + 1) / nb);
      t0 = max(lo, start) - start;
      t1 = min(max(hi, start) - start, n);
    } else {
      const uint64_t at = 2 * (uint64_t)start * nb + total;
      const uint32_t b0 = min((uint32_t)(at / (2 * (uint64_t)total)), nb - 1);
      const uint32_t b1 = min((uint32_t)((at + 2 * (uint64_t)n * cost * nb) / (2 * (uint64_t)total)), nb);
      const uint32_t blocks = b1 > b0 ? b1 - b0 : 1, k = j - b0;
      t0 = k < blocks ? (uint32_t)((uint64_t)n * k / blocks) : n;
      t1 = k < blocks ? (uint32_t)((uint64_t)n * (k + 1) / blocks) : 0u;
    }
  };
  // where a lane finds its operands of 16 rows: x = 4 s + i is block 4 s + gq's i-th quarter, x = 4 JS + s rope
  // (the swizzle is within a block and a half, so s is a plain offset)
  uint32_t q_at[4], pe_at[RS];
#pragma unroll
  for (int i = 0; i < 4; ++i) q_at[i] = 16 * (la * RC + ((4 * gq + i) ^ w_swz<D>(la)));
#pragma unroll
  for (int s = 0; s < RS; ++s) pe_at[s] = 16 * (la * RC + D / 8 + ((4 * s + gq) ^ w_swz<D>(la)));
  const auto operand = [&](uint32_t rows16, int x) __attribute__((always_inline)) {
    const uint32_t at = x < 4 * JS ? q_at[x % 4] + 256 * (x / 4) : pe_at[x < 4 * JS ? 0 : x - 4 * JS];
    return *reinterpret_cast<const u32x4*>(smem + rows16 + at);
  };
  const uint32_t max_page = (uint32_t)((a.num_slots - 1) >> a.page_shift), max_slot = (uint32_t)(a.num_slots - 1);
  const uint32_t page_mask = (1u << a.page_shift) - 1;

  uint32_t before = 0;
  for (int chunk = 0; chunk < a.B; chunk += 64) {
    const uint32_t units = tiles_of(chunk + lane), cost = cost_of(chunk + lane), incl = wave_scan(units * cost);
    uint32_t part0, part1;
    share(before + incl - units * cost, units, cost, part0, part1);
    before += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    for (uint64_t hit = __builtin_amdgcn_ballot_w64(part0 < part1); hit; hit &= hit - 1) {
      const int l = __builtin_ctzll(hit), b = chunk + l;
      const uint32_t t_begin = (uint32_t)__builtin_amdgcn_readlane((int)part0, l);
      const uint32_t t_end = (uint32_t)__builtin_amdgcn_readlane((int)part1, l);
      const Mx4Request rq = mx4_request(a, b);
      const int n = places(b, rq);  // positions
      const int rows = rq.nq * a.H, qtiles = (rows + 15) / 16;
      float* const acc = a.acc + (a.req_idx ? a.req_idx[b] : b) * a.acc_st;
      // Copies of 16 bytes a lane of rows r0 .. r0 + 16 N - 1, N times 16 rows, to LDS at `at`, nine a wave
      // for every 16 * 9 W / COPIES rows (past the last row: that one again).
      const int64_t q_row0 = (int64_t)rq.q0 * a.q_st;
      const auto copy_piece = [&](int r0, int k, uint32_t at) __attribute__((always_inline)) {
        const int ci = 64 * k + lane, r = ci / RC, c = (ci - r * RC) ^ w_swz<D>(r & 15);
        const uint32_t row = (uint32_t)min(r0 + r, rows - 1), tok = row / (uint32_t)a.H, head = row - tok * a.H;
        copy16(a.q + q_row0 + (int64_t)tok * a.q_st + (int64_t)head * a.q_sh + 8 * c, at + 1024 * k);
      };
      // lse of row la of 16, and the positions that it sees; a row that saw nothing (lse -inf, whatever its query
      // holds), or one past the last, sees none
      struct Row {
        float lse;
        int vis;
      };
      const auto row_of = [&](int qt) {
        const int row = 16 * qt + la;
        const uint32_t rc = (uint32_t)min(row, rows - 1), tok = rc / (uint32_t)a.H, head = rc - tok * a.H;
        const float lse = a.lse[(int64_t)(rq.q0 + (int)tok) * a.H + head];
        return Row{lse, row < rows && lse != -INFINITY ? rq.past + (int)tok + 1 : 0};
      };
      Row qrow[QT > 0 ? QT : 1];
      if constexpr (QT > 0) {
        __syncthreads();  // the last request's rows are no longer read
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
          if (qt < qtiles) {
            for (int k = wave; k < G::QT / 1024; k += W) copy_piece(16 * qt, k, lds0 + qt * G::QT);
            qrow[qt] = row_of(qt);
          } else {
            qrow[qt] = Row{INFINITY, 0};
          }
        wait_loads<0>();
        __syncthreads();
      }
      // a tile from unit t: MT sub-tiles of 16 positions for each wave
      const auto tile = [&](uint32_t t, auto Sub) __attribute__((always_inline)) {
        constexpr int MT = decltype(Sub)::value;
        const int p0 = (int)t * TILE + 16 * MT * wave;  // this wave's positions
        // ---- the keys --------------------------------------------------------------------
        u32x4 code[MT][JS], pe[MT][RS];
        float scale[MT][JS];
        uint32_t nan = 0;
        uint32_t slot[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const int pos = min(p0 + 16 * m + la, n - 1);
          const uint32_t page = (uint32_t)a.kv_indices[rq.list + (pos >> a.page_shift)];
          slot[m] = min((min(page, max_page) << a.page_shift) + ((uint32_t)pos & page_mask), max_slot);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const uint8_t* const c = a.codes + (uint64_t)slot[m] * CB + 16 * gq;
#pragma unroll
          for (int s = 0; s < JS; ++s) code[m][s] = gload<u32x4>(c + 64 * s);
          const uint8_t* const r = reinterpret_cast<const uint8_t*>(a.rope) + (uint64_t)slot[m] * (2 * R) + 16 * gq;
#pragma unroll
          for (int s = 0; s < RS; ++s) pe[m][s] = gload<u32x4>(r + 64 * s);
          const uint8_t* const sp = a.scales + (uint64_t)slot[m] * NB;
          uint32_t w[JS];
          if constexpr (JS == 4) {
            const u32x4 v = gload<u32x4>(sp);
            w[0] = v[0], w[1] = v[1], w[2] = v[2], w[3] = v[3];
          } else {
            const u32x2 v = gload<u32x2>(sp);
            w[0] = v[0], w[1] = v[1];
          }
#pragma unroll
          for (int s = 0; s < JS; ++s) {
            const uint32_t e = (w[s] >> (8 * gq)) & 255u;  // of block 4 s + gq
            scale[m][s] = __uint_as_float(e << 23);
            nan |= e == (uint32_t)kMx4NaN ? 1u << (JS * m + s) : 0u;
          }
        }
        float sum[MT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[m][i] = 0.f;
        // dword i of the codes of block 4 s + gq of sub-tile m, as values
        const auto values = [&](int m, int s, int i) {
          u32x4 v = w_expand(code[m][s][i], scale[m][s]);
          const uint32_t bad = nan >> (JS * m + s) & 1u ? 0x7fc07fc0u : 0u;
#pragma unroll
          for (int k = 0; k < 4; ++k) v[k] |= bad;
          return v;
        };
        // the scores of 16 rows, C[position 4 gq + i][row la], to weights
        const auto weigh = [&](const f32x4 (&c)[MT], const Row& r) {
          // positions that not every row sees
          const bool edge = __builtin_amdgcn_ballot_w64(r.vis < p0 + 16 * MT) != 0;
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float w = __builtin_amdgcn_exp2f(fmaf(c[m][i], a.sm_scale, -r.lse) * kLog2e);
              if (edge) w = p0 + 16 * m + 4 * gq + i < r.vis ? w : 0.f;
              sum[m][i] += w;
            }
        };
        const auto add_weight = [&](float c, float lse, float& to) __attribute__((always_inline)) {
          to += __builtin_amdgcn_exp2f(fmaf(c, a.sm_scale, -lse) * kLog2e);
          asm volatile("" : "+v"(to));  // added here, between the products
        };
        if constexpr (QT > 0) {
          if (p0 < n) {
            f32x4 c[QT][MT];
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
#pragma unroll
              for (int m = 0; m < MT; ++m) c[qt][m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < JS; ++s)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                u32x4 k[MT];
#pragma unroll
                for (int m = 0; m < MT; ++m) k[m] = values(m, s, i);
#pragma unroll
                for (int qt = 0; qt < QT; ++qt) {
                  const u32x4 q = operand(qt * G::QT, 4 * s + i);
#pragma unroll
                  for (int m = 0; m < MT; ++m) c[qt][m] = mfma16x16x32(k[m], q, c[qt][m]);
                }
              }
#pragma unroll
            for (int s = 0; s < RS; ++s)
#pragma unroll
              for (int qt = 0; qt < QT; ++qt) {
                const u32x4 q = operand(qt * G::QT, 4 * JS + s);
#pragma unroll
                for (int m = 0; m < MT; ++m) c[qt][m] = mfma16x16x32(pe[m][s], q, c[qt][m]);
              }
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
              if (QT == 1 || qt < qtiles) weigh(c[qt], qrow[qt]);
          }
        } else {
          // rows that see none of the tile's positions come first: from the first token that does
          const int tok0 = max((int)t * TILE - rq.past, 0);
          constexpr int QR = G::QR, SUB = QR / 16;
          const int all = (rows + QR - 1) / QR, steps = (int)((int64_t)all * (part + 1) / a.parts);
          const int s0 = (int)min(max((int64_t)tok0 * a.H / QR, (int64_t)all * part / a.parts), (int64_t)steps);
          // Whose rows lie one behind the other: a step's copies are the last one's, so much further on.
          const bool flat = a.q_st == (int64_t)a.H * a.q_sh && a.q_sh < (1 << 22);
          uint32_t off[9];
#pragma unroll
          for (int k = 0; k < 9; ++k) {
            const int ci = 64 * (9 * wave + k) + lane, r = ci / RC;
            off[k] = (uint32_t)(2 * (r * (int)a.q_sh + 8 * ((ci - r * RC) ^ w_swz<D>(r & 15))));
          }
          const auto copy_step = [&](int s) __attribute__((always_inline)) {
            const uint32_t at = lds0 + (uint32_t)(s & 1) * G::STEP;
            if (flat && QR * (s + 1) <= rows) {
              const uint16_t* const from = a.q + q_row0 + (int64_t)QR * s * a.q_sh;
#pragma unroll
              for (int k = 0; k < 9; ++k) copy16(from, off[k], at + 1024 * (9 * wave + k));
            } else {
#pragma unroll 1
              for (int k = 0; k < 9; ++k) copy_piece(QR * s, 9 * wave + k, at);
            }
          };
          // lse of the rows la of a step (rows as q0 H + row in a.lse)
          float next[SUB];
          const auto load_lse = [&](int s) __attribute__((always_inline)) {
#pragma unroll
            for (int q = 0; q < SUB; ++q)
              next[q] = a.lse[(int64_t)rq.q0 * a.H + min(QR * s + 16 * q + la, rows - 1)];
          };
          if (s0 < steps) {
            copy_step(s0);
            load_lse(s0);
          }
          u32x4 k[MT][JS][4];
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int s = 0; s < JS; ++s)
#pragma unroll
              for (int i = 0; i < 4; ++i) k[m][s][i] = values(m, s, i);
          for (int step = s0; step < steps; ++step) {
            wait_loads<0>();
            __syncthreads();  // these rows are there; the last ones are no longer read
            float lse[SUB];
            bool none = false;
#pragma unroll
            for (int q = 0; q < SUB; ++q) {
              lse[q] = next[q];
              none = none || lse[q] == -INFINITY;
            }
            const bool all_weigh = __builtin_amdgcn_ballot_w64(none) == 0;
            if (step + 1 < steps) {
              copy_step(step + 1);
              load_lse(step + 1);
            }
            const uint32_t rows_at = (uint32_t)(step & 1) * G::STEP;
            const int first_row = QR * step;
            constexpr int NS = 4 * JS + RS, AHEAD = 3;  // operands of 16 rows; how many come ahead of their use
            const auto product = [&](f32x4 (&c)[MT], int x, u32x4 y) __attribute__((always_inline)) {
#pragma unroll
              for (int m = 0; m < MT; ++m)
                c[m] = mfma16x16x32(x < 4 * JS ? k[m][x / 4 % JS][x % 4] : pe[m][x < 4 * JS ? 0 : x - 4 * JS], y,
                                    x == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : c[m]);
            };
            if (__builtin_expect(all_weigh && rq.past + first_row / a.H + 1 >= p0 + 16 * MT && first_row + QR <= rows, 1)) {
              // every row sees every position: the weights of 16 rows between the products of the next 16
              f32x4 c[2][MT];
              u32x4 ring[AHEAD + 1];
              static_for<AHEAD>([&](auto Y) __attribute__((always_inline)) { ring[Y] = operand(rows_at, Y); });
              static_for<SUB * NS>([&](auto Y) __attribute__((always_inline)) {
                constexpr int y = decltype(Y)::value, q = y / NS, x = y % NS, ahead = y + AHEAD;
                if constexpr (ahead < SUB * NS)
                  ring[ahead % (AHEAD + 1)] = operand(rows_at + ahead / NS * G::QT, ahead % NS);
                product(c[q % 2], x, ring[y % (AHEAD + 1)]);
                if constexpr (q > 0) {
                  constexpr int v0 = x * 4 * MT / NS, v1 = (x + 1) * 4 * MT / NS;
#pragma unroll
                  for (int v = v0; v < v1; ++v)
                    add_weight(c[(q + 1) % 2][v / 4][v % 4], lse[q > 0 ? q - 1 : 0], sum[v / 4][v % 4]);
                }
                __builtin_amdgcn_sched_barrier(0);
              });
#pragma unroll
              for (int v = 0; v < 4 * MT; ++v) add_weight(c[(SUB - 1) % 2][v / 4][v % 4], lse[SUB - 1], sum[v / 4][v % 4]);
            } else {
#pragma unroll
              for (int q = 0; q < SUB; ++q) {
                if (first_row + 16 * q >= rows) break;
                f32x4 c[MT];
#pragma unroll
                for (int x = 0; x < NS; ++x) {
                  product(c, x, operand(rows_at + q * G::QT, x));
                  if (x % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
                const int row = first_row + 16 * q + la;
                weigh(c, Row{lse[q], row < rows && lse[q] != -INFINITY
                                         ? rq.past + (int)((uint32_t)row / (uint32_t)a.H) + 1 : 0});
              }
            }
          }
          __syncthreads();
        }
        // ---- sums over the rows, a position to each lane that writes ------------------------
        float out = 0.f;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float s = row_sum16(sum[m][i]);
            if (la == 4 * m + i) out = s;
          }
        static_assert(MT <= 4, "a lane for each position");
        const int pos = p0 + 16 * (la >> 2) + 4 * gq + (la & 3);
        if (la < 4 * MT && pos < n) {
          if (QT == 0 && a.parts > 1)
            a.ws[part * a.ws_part + ((int64_t)rq.list << a.page_shift) + pos] = out;
          else
            acc[pos] = a.add ? acc[pos] + out : out;
        }
      };
      for (uint32_t t = t_begin; t < t_end;) {
        if constexpr (QT > 0) {
          tile(t, std::integral_constant<int, MOST>{});
          ++t;
        } else {
          const uint32_t left = t_end - t, tiles = (left + MOST - 1) / MOST, sub = (left + tiles - 1) / tiles;
          if constexpr (MOST >= 4) {
            if (sub == 4) tile(t, std::integral_constant<int, 4>{});
            if (sub == 3) tile(t, std::integral_constant<int, 3>{});
          }
          if (sub == 2) tile(t, std::integral_constant<int, 2>{});
          if (sub == 1) tile(t, std::integral_constant<int, 1>{});
          t += sub;
        }
      }
    }
  }
}

// Sums of the rows' parts, in their order.
__global__ __launch_bounds__(256) void mx4_weights_join_kernel(Mx4WeightsArgs a) {
  const int each = gridDim.x / a.B, b = blockIdx.x / each;  // blocks of a request
  const Mx4Request rq = mx4_request(a, b);
  const int64_t row = a.req_idx ? a.req_idx[b] : b;
  if (row < 0 || row >= a.acc_rows) return;
  const int n = (int)min((int64_t)rq.len, a.acc_cols);
  const float* const ws = a.ws + ((int64_t)rq.list << a.page_shift);
  float* const acc = a.acc + row * a.acc_st;
  for (int pos = (blockIdx.x - b * each) * 256 + threadIdx.x; pos < n; pos += each * 256) {
    float sum = a.add ? acc[pos] : 0.f;
#pragma unroll 8
    for (int p = 0; p < a.parts; ++p) sum += ws[p * a.ws_part + pos];
    acc[pos] = sum;
  }
}

// Many rows: units of 64 positions at most, and parts of the rows. A unit's steps over its request's rows come one after
// another, so that a launch takes as long as the longest request's, or as all units' on the blocks that run
// at once: parts bring the first down to the second, of three steps at least, if that saves three (a step takes
// two microseconds, a second launch and what it reads six). 7 requests of 51 to 172 positions and up
// to 51 queries of 128 heads: 238 us in one part, 29 in parts of a few steps; 12 of 21 positions, 20 queries of 48
// heads: 39 and 24.
struct WeightsPlan {
  int64_t units;
  int parts;
};
static WeightsPlan weights_plan(int64_t n_indices, int page_shift, int B, int64_t all_rows, int64_t rows, int step,
                                int num_cus) {
  // (positions stay below 2^30 a request, the units of all below 2^30 as the sums would not fit the memory)
  const int64_t positions = std::min<int64_t>(n_indices, int64_t(1) << 40 >> page_shift) << page_shift;
  WeightsPlan p{std::min<int64_t>(positions / 64 + B, 1 << 30), 1};
  if (rows <= kWeightsFew || B == 0) return p;
  const int64_t steps = (rows + step - 1) / step;
  const double mean = std::min((double)steps, (double)all_rows / B / step + 0.5);
  const double each = std::max(3.0, (double)p.units * mean / (2.0 * num_cus));
  const int64_t parts = (int64_t)std::ceil((double)steps / each);
  if (parts > 1 && (double)steps - std::max(each, (double)steps / parts) > 3.0)
    p.parts = (int)std::min<int64_t>(parts, 2 * num_cus);
  return p;
}

template <int D, int R, int MT, int QT>
hipError_t launch_weights(const Mx4WeightsArgs& a, int64_t blocks, hipStream_t stream) {
  constexpr int lds = QT > 0 ? QT * WGeo<D, R>::QT : 2 * WGeo<D, R>::STEP;
  if constexpr (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)mx4_weights_kernel<D, R, MT, QT>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((mx4_weights_kernel<D, R, MT, QT>), dim3((unsigned)blocks), dim3(256), lds, stream, a);
  return hipGetLastError();
}

template <int D, int R>
hipError_t launch_weights_rows(const Mx4WeightsArgs& a, int num_cus, hipStream_t stream) {
  const int64_t rows = (int64_t)a.max_q_len * a.H, tiles = (a.n_indices << a.page_shift) / 128 + a.B;
  static_assert(kWeightsFew == 64, "four groups of rows");
  // Few rows: as many blocks as their LDS leaves room for, four a CU at most (32 requests of 16384, 16 heads: 48.2 us
  // with four, 51.4 with three, 55.6 with eight; 40 heads of width 512 28 with the two that fit, 35 with more).
  const auto few = [&](int groups) {
    const int64_t cu = std::min<int64_t>(4, (160 << 10) / (groups * WGeo<D, R>::QT));
    return std::min<int64_t>(tiles, cu * num_cus);
  };
  if (rows <= 16) return launch_weights<D, R, 2, 1>(a, few(1), stream);
  if (rows <= 32) return launch_weights<D, R, 2, 2>(a, few(2), stream);
  // (40 heads of width 256: 20.2 us with three groups, 21.2 with four)
  if (rows <= 48) return launch_weights<D, R, 2, 3>(a, few(3), stream);
  if (rows <= 64) return launch_weights<D, R, 2, 4>(a, few(4), stream);
  Mx4WeightsArgs m = a;
  const WeightsPlan p = weights_plan(a.n_indices, a.page_shift, a.B, (int64_t)a.T * a.H, rows, WGeo<D, R>::QR, num_cus);
  m.parts = a.ws ? p.parts : 1;
  m.ws_part = a.n_indices << a.page_shift;
  // (a batch's cost in 32 bits)
  while (p.units * ((rows / WGeo<D, R>::QR >> m.cost_shift) + 2) >= (int64_t(1) << 32)) ++m.cost_shift;
  const int64_t blocks = std::min<int64_t>(p.units, 2 * num_cus / m.parts);
  const hipError_t e = launch_weights<D, R, D == 512 ? 2 : 4, 0>(m, blocks * m.parts, stream);
  if (e != hipSuccess || m.parts == 1) return e;
  const int64_t each = std::max<int64_t>(1, std::min<int64_t>((m.ws_part + 255) / 256, 2048 / a.B));
  hipLaunchKernelGGL(mx4_weights_join_kernel, dim3((unsigned)(each * a.B)), dim3(256), 0, stream, m);
  return hipGetLastError();
}

}  // namespace rolaq

int64_t rolaq_mx4_weights_ws_bytes(int64_t n_indices, int page_shift, int B, int64_t all_rows, int64_t rows, int D,
                                   int num_cus) {
  using namespace rolaq;
  const int step = D == 512 ? WGeo<512, 64>::QR : WGeo<256, 32>::QR;
  const int parts = weights_plan(n_indices, page_shift, B, all_rows, rows, step, num_cus).parts;
  return parts > 1 ? parts * (n_indices << page_shift) * 4 : 0;
}

hipError_t rolaq_launch_mx4_weights(const rolaq::Mx4WeightsArgs& a, int D, int num_cus, hipStream_t stream) {
  using namespace rolaq;
  if (D == 512) return launch_weights_rows<512, 64>(a, num_cus, stream);
  if (D == 256) return launch_weights_rows<256, 32>(a, num_cus, stream);
  return hipErrorInvalidValue;
}
