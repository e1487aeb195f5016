// Attention weight of every cached position of the MX4 latent cache (gfx950), summed over a
// request's query rows (queries and heads):
//   acc_t (+)= sum over the rows that see t of exp(sm_scale (q_lat . x_t + q_pe . r_t) - lse),
// lse the row's log sum of exponentials as the attention call returned it.
//
// The positions are what a wave holds: it loads the codes of 16 MT positions straight into
// registers, expands them to bf16 (v_cvt_scalef32_pk_bf16_fp4, exact) and goes through the query
// rows, which lie in LDS as they are, 16 at a time, on bf16 MFMA. A position's sum stays in its
// lanes until the rows are through, so that each is written once, by one lane, in an
// order that no other request or launch shape changes. (The scores of the attention itself, 4-bit
// codes against a query split into two e4m3 parts, are off by 2^-18 of the largest: the weights
// were off by 1e-5, now by 3e-7.)
//
// Few rows (64 at most, a decode step): a block keeps them in LDS and walks a range of the batch's
// tiles, expanding as it multiplies; bound by the cache's bytes. Many rows (the last
// queries of prompts): a wave keeps its positions expanded, and the rows come to LDS 16 at a time
// while the last 16 are in use; bound by the matrix instructions.
#include "rolaq_common.h"
#include "mx4_args.h"
#include "mx4_request.h"
#include "mx4_tile.h"

#include <algorithm>

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
  static constexpr int COPIES = QT / 1024;
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

// Sum over the 16 lanes of a row of lanes, on each of them.
template <int CTRL>
__device__ __forceinline__ float add_ror(float v) {
  return v + __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float row_sum16(float v) {
  v = add_ror<0x121>(v);
  v = add_ror<0x122>(v);
  v = add_ror<0x124>(v);
  return add_ror<0x128>(v);
}

// QT > 0: at most 16 QT rows a request, kept in LDS; 0: any number, streamed.
template <int D, int R, int MT, int QT>
__global__ __launch_bounds__(256, 2) void mx4_weights_kernel(Mx4WeightsArgs a) {
  using G = WGeo<D, R>;
  constexpr int NB = G::NB, CB = G::CB, RS = G::RS, W = G::W, JS = G::JS, RC = G::RC;
  constexpr int TILE = 16 * MT * W;  // positions of a block's tile
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
  uint32_t total = 0;
  for (int c = 0; c < a.B; c += 64) total += (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(tiles_of(c + lane)), 63);
  // (neighbours on one XCD: they read the same query rows)
  const uint32_t per = gridDim.x / 8;
  const uint32_t j = gridDim.x % 8 == 0 ? (blockIdx.x % 8) * per + blockIdx.x / 8 : blockIdx.x;
  const uint32_t nb = min(gridDim.x, total);
  if (j >= nb) return;
  uint32_t u = (uint32_t)((uint64_t)total * j / nb);
  const uint32_t u_end = (uint32_t)((uint64_t)total * (j + 1) / nb);
  int b = 0;
  uint32_t first = 0;  // first tile of request b
  {
    uint32_t before = 0;
    for (int c = 0; c < a.B; c += 64) {
      const uint32_t n = tiles_of(c + lane), incl = wave_scan(n), start = before + incl - n;
      const uint64_t hit = __builtin_amdgcn_ballot_w64(start <= u && u < start + n);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        b = c + l;
        first = (uint32_t)__builtin_amdgcn_readlane((int)start, l);
        break;
      }
      before += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    }
  }
  const uint32_t max_page = (uint32_t)((a.num_slots - 1) >> a.page_shift), max_slot = (uint32_t)(a.num_slots - 1);
  const uint32_t page_mask = (1u << a.page_shift) - 1;

  while (u < u_end && b < a.B) {
    const Mx4Request rq = mx4_request(a, b);
    const int n = places(b, rq);  // positions
    const uint32_t mine = (uint32_t)((n + TILE - 1) / TILE);
    if (u - first >= mine) {
      first += mine;
      ++b;
      continue;
    }
    const uint32_t t_end = min(mine, u_end - first);
    const int rows = rq.nq * a.H, qtiles = (rows + 15) / 16;
    float* const acc = a.acc + (a.req_idx ? a.req_idx[b] : b) * a.acc_st;
    // copies of this wave's share of rows 16 qt .. to LDS at `at` (past the last row: that one again)
    const auto copy_rows = [&](int qt, uint32_t at) {
      for (int k = wave; k < G::COPIES; k += W) {
        const int ci = 64 * k + lane, r = ci / RC, c = (ci - r * RC) ^ w_swz<D>(r);
        const uint32_t row = (uint32_t)min(16 * qt + r, rows - 1), tok = row / (uint32_t)a.H, head = row - tok * a.H;
        copy16(a.q + (int64_t)(rq.q0 + (int)tok) * a.q_st + (int64_t)head * a.q_sh + 8 * c, at + 1024 * k);
      }
    };
    // lse of row la of 16, and the positions that it sees; a row that saw nothing (lse
    // -inf), or one past the last, weighs nothing
    struct Row {
      float lse;
      int vis;
    };
    const auto row_of = [&](int qt) {
      const int row = 16 * qt + la;
      const uint32_t rc = (uint32_t)min(row, rows - 1), tok = rc / (uint32_t)a.H, head = rc - tok * a.H;
      Row r{a.lse[(int64_t)(rq.q0 + (int)tok) * a.H + head], row < rows ? rq.past + (int)tok + 1 : 0};
      if (r.lse == -INFINITY) r.lse = INFINITY;
      return r;
    };
    Row qrow[QT > 0 ? QT : 1];
    if constexpr (QT > 0) {
      __syncthreads();  // the last request's rows are no longer read
#pragma unroll
      for (int qt = 0; qt < QT; ++qt)
        if (qt < qtiles) {
          copy_rows(qt, lds0 + qt * G::QT);
          qrow[qt] = row_of(qt);
        } else {
          qrow[qt] = Row{INFINITY, 0};
        }
      wait_loads<0>();
      __syncthreads();
    }
    for (uint32_t t = u - first; t < t_end; ++t) {
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
        // positions that not every row sees (a row past the last sees none)
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
      const auto query = [&](const uint8_t* rows16, int c) {
        return *reinterpret_cast<const u32x4*>(rows16 + 16 * (la * RC + (c ^ w_swz<D>(la))));
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
                const u32x4 q = query(smem + qt * G::QT, 16 * s + 4 * gq + i);
#pragma unroll
                for (int m = 0; m < MT; ++m) c[qt][m] = mfma16x16x32(k[m], q, c[qt][m]);
              }
            }
#pragma unroll
          for (int s = 0; s < RS; ++s)
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
              const u32x4 q = query(smem + qt * G::QT, D / 8 + 4 * s + gq);
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
        const int qt0 = (int)min((int64_t)tok0 * a.H / 16, (int64_t)qtiles);
        Row next{};
        if (qt0 < qtiles) {
          copy_rows(qt0, lds0 + (qt0 & 1) * G::QT);
          next = row_of(qt0);
        }
        u32x4 k[MT][JS][4];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int s = 0; s < JS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) k[m][s][i] = values(m, s, i);
        for (int qt = qt0; qt < qtiles; ++qt) {
          wait_loads<0>();
          __syncthreads();  // these rows are there; the last ones are no longer read
          const Row now = next;
          if (qt + 1 < qtiles) {
            copy_rows(qt + 1, lds0 + ((qt + 1) & 1) * G::QT);
            next = row_of(qt + 1);
          }
          const uint8_t* const q16 = smem + (qt & 1) * G::QT;
          f32x4 c[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m) c[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < JS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const u32x4 q = query(q16, 16 * s + 4 * gq + i);
#pragma unroll
              for (int m = 0; m < MT; ++m) c[m] = mfma16x16x32(k[m][s][i], q, c[m]);
            }
#pragma unroll
          for (int s = 0; s < RS; ++s) {
            const u32x4 q = query(q16, D / 8 + 4 * s + gq);
#pragma unroll
            for (int m = 0; m < MT; ++m) c[m] = mfma16x16x32(pe[m][s], q, c[m]);
          }
          weigh(c, now);
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
      if (la < 4 * MT && pos < n) acc[pos] = a.add ? acc[pos] + out : out;
    }
    u = first + t_end;
  }
}

template <int D, int R, int MT, int QT>
hipError_t launch_weights(const Mx4WeightsArgs& a, int most_blocks, hipStream_t stream) {
  constexpr int lds = (QT > 0 ? QT : 2) * WGeo<D, R>::QT;
  const hipError_t e = hipFuncSetAttribute((const void*)mx4_weights_kernel<D, R, MT, QT>,
                                           hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  const int64_t tiles = (a.n_indices << a.page_shift) / (64 * MT) + a.B;
  hipLaunchKernelGGL((mx4_weights_kernel<D, R, MT, QT>), dim3((unsigned)std::min<int64_t>(tiles, most_blocks)), dim3(256),
                     lds, stream, a);
  return hipGetLastError();
}

template <int D, int R>
hipError_t launch_weights_rows(const Mx4WeightsArgs& a, int num_cus, hipStream_t stream) {
  const int64_t rows = (int64_t)a.max_q_len * a.H;
  static_assert(kWeightsFew == 64, "four groups of rows");
  if (rows <= 16) return launch_weights<D, R, 2, 1>(a, 4 * num_cus, stream);
  if (rows <= 32) return launch_weights<D, R, 2, 2>(a, 4 * num_cus, stream);
  if (rows <= 64) return launch_weights<D, R, 2, 4>(a, 2 * num_cus, stream);
  return launch_weights<D, R, D == 512 ? 2 : 4, 0>(a, 2 * num_cus, stream);
}

}  // namespace rolaq

hipError_t rolaq_launch_mx4_weights(const rolaq::Mx4WeightsArgs& a, int D, int num_cus, hipStream_t stream) {
  using namespace rolaq;
  if (D == 512) return launch_weights_rows<512, 64>(a, num_cus, stream);
  if (D == 256) return launch_weights_rows<256, 32>(a, num_cus, stream);
  return hipErrorInvalidValue;
}
