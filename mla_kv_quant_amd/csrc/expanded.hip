// Attention over expanded latent keys and values (gfx950): per head h
//   s_t = sm_scale (q_nope . k_nope_t,h + q_pe . k_pe_t),  o = sum_t softmax(s)_t v_t,h,
// k_nope and v side by side as kv_b_proj gives them, one k_pe for all heads; causal at the
// end of the keys, or all keys for all queries.
#include "rolaq_common.h"
#include "mx4_request.h"
#include "mx4_tile.h"
#include "serve_args.h"

#include <algorithm>

namespace rolaq {

constexpr float kXNoRef = -0x1.fffffep127f;  // reference of a row that has seen no score
constexpr float kXSlack = 8.f;               // log2 by which a score may pass its row's reference

template <int DN, int RG_>
struct XGeo {
  static constexpr int DR = DN / 2, DK = DN + DR;
  static constexpr int RG = RG_;          // groups of 32 query rows of a wave
  static constexpr int W = 4;             // waves
  static constexpr int ROWS = 32 * RG * W;
  static constexpr int KT = 64;           // keys of a tile
  static constexpr int KB = 2 * DK, VB = 2 * DN;    // bytes of a key and of a value row
  static constexpr int KC = KB / 16, VC = VB / 16;  // their 16-byte chunks
  static constexpr int TILE = KT * (KB + VB);
  static constexpr int NBUF = 2;
  static constexpr int KS = DK / 16;  // K-steps of the scores
  static constexpr int ND = DN / 32;  // output column blocks
  static constexpr int KCOP = KT * KC / (64 * W), VCOP = KT * VC / (64 * W);  // a wave's 1 KB copies of a tile
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

// Chunk c of key row r lies at chunk c ^ k_swz(r), of value row r at c ^ v_swz(r): 16 rows of
// one column (a quarter wave of a score read), and 4 rows x 64 bytes (half a wave of a transposed
// read), fall on 16 chunk positions each.
template <int DN>
__device__ __forceinline__ int k_swz(int r) { return DN == 128 ? (r >> 1) & 7 : (r >> 2) & 3; }
template <int DN>
__device__ __forceinline__ int v_swz(int r) { return DN == 128 ? 4 * (r & 3) : 4 * ((r >> 1) & 1); }

// LSE: for calls that ask for it, the sum of the weights before their rounding as well.
template <int DN, int RG, bool LSE>
__global__ __launch_bounds__(256, RG == 1 ? 2 : 1) void expanded_kernel(ExpandedArgs a) {
  using G = XGeo<DN, RG>;
  constexpr int KB = G::KB, VB = G::VB, KC = G::KC, VC = G::VC, KT = G::KT, KS = G::KS, ND = G::ND;
  extern __shared__ __attribute__((aligned(1024))) uint8_t smem[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  const int tid = threadIdx.x, lane = tid & 63, la32 = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // ---- head, row block and part of the keys ---------------------------------------
  const uint32_t item = blockIdx.x;
  const int h = item % (uint32_t)a.H;
  const uint32_t rest = item / (uint32_t)a.H;
  const int part = rest % (uint32_t)a.splits;
  const uint32_t want = rest / (uint32_t)a.splits;  // row block of the batch
  const auto clampq = [&](int i) { return min(max(a.qo_indptr[i], 0), a.T); };
  const auto clampk = [&](int i) { return min(max(a.kv_indptr[i], 0), a.N); };
  int b = -1, rb = 0;
  {
    uint32_t before = 0;
    for (int c = 0; c < a.B; c += 64) {
      const int i = min(c + lane, a.B - 1);
      const int nq = min(max(clampq(i + 1) - clampq(i), 0), a.max_q_len);
      const uint32_t n = c + lane < a.B ? (uint32_t)((nq + G::ROWS - 1) / G::ROWS) : 0u;
      const uint32_t incl = wave_scan(n), start = before + incl - n;
      const uint64_t hit = __builtin_amdgcn_ballot_w64(start <= want && want < start + n);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        b = c + l;
        rb = __builtin_amdgcn_readlane((int)n, l) - 1 - (int)(want - (uint32_t)__builtin_amdgcn_readlane((int)start, l));
        break;
      }
      before += (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    }
  }
  if (b < 0) return;
  const int q0 = __builtin_amdgcn_readfirstlane(clampq(b)), k0 = __builtin_amdgcn_readfirstlane(clampk(b));
  const int nq_all = max(__builtin_amdgcn_readfirstlane(clampq(b + 1)) - q0, 0), nq = min(nq_all, a.max_q_len);
  const int nk = max(__builtin_amdgcn_readfirstlane(clampk(b + 1)) - k0, 0);
  const int row0 = rb * G::ROWS;
  const int past = nk - nq_all;
  // keys that row r sees
  const auto sees = [&](int r) { return a.causal ? min(max(past + r + 1, 0), nk) : nk; };
  const int last = min(row0 + G::ROWS, nq) - 1;
  const int kend_all = sees(last);
  const int tiles_all = (kend_all + KT - 1) / KT;
  const int t0 = (int)((int64_t)tiles_all * part / a.splits), t1 = (int)((int64_t)tiles_all * (part + 1) / a.splits);

  // ---- query rows -------------------------------------------------------------------
  int vis[RG];
  u32x4 qf[RG][KS];
#pragma unroll
  for (int r = 0; r < RG; ++r) {
    const int row = row0 + 32 * (RG * wave + r) + la32;
    vis[r] = sees(min(row, nq - 1));
    const uint16_t* const p = a.q + (int64_t)(q0 + min(row, nq - 1)) * a.q_st + (int64_t)h * a.q_sh + 8 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[r][s] = gload<u32x4>(p + 16 * s);
  }
  const int vis_min = sees(row0);  // seen by every row of the block

  f32x16 O[RG][ND];
#pragma unroll
  for (int r = 0; r < RG; ++r)
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < 16; ++j) O[r][d][j] = 0.f;
  float ref[RG], sum[RG], usum[RG];  // usum (LSE): of the weights as they were
#pragma unroll
  for (int r = 0; r < RG; ++r) ref[r] = kXNoRef, sum[r] = usum[r] = 0.f;
  const float c2 = a.sm_scale * kLog2e;

  // ---- tile copies --------------------------------------------------------------------
  const uint8_t* const kv = reinterpret_cast<const uint8_t*>(a.kv + (int64_t)k0 * a.kv_st + (int64_t)h * a.kv_sh);
  const uint8_t* const pe = reinterpret_cast<const uint8_t*>(a.pe + (int64_t)k0 * a.pe_st);
  const auto copy = [&](int t) {
    const uint32_t at = lds0 + (uint32_t)(t & 1) * G::TILE;
#pragma unroll
    for (int j = 0; j < G::KCOP; ++j) {
      const int ci = 64 * (G::KCOP * wave + j) + lane, row = ci / KC, c = (ci - row * KC) ^ k_swz<DN>(row);
      const int64_t key = min(KT * t + row, nk - 1);
      const uint8_t* const src = c < VC ? kv + key * (2 * a.kv_st) + 16 * c : pe + key * (2 * a.pe_st) + 16 * (c - VC);
      copy16(src, at + 1024 * (G::KCOP * wave + j));
    }
#pragma unroll
    for (int j = 0; j < G::VCOP; ++j) {
      const int ci = 64 * (G::VCOP * wave + j) + lane, row = ci / VC, c = (ci - row * VC) ^ v_swz<DN>(row);
      const int64_t key = min(KT * t + row, nk - 1);
      copy16(kv + key * (2 * a.kv_st) + VB + 16 * c, at + KT * KB + 1024 * (G::VCOP * wave + j));
    }
  };

  if (t0 < t1) copy(t0);
  for (int t = t0; t < t1; ++t) {
    wait_loads<0>();
    __syncthreads();
    if (t + 1 < t1) copy(t + 1);
    const uint8_t* const kt = smem + (t & 1) * G::TILE;
    const uint8_t* const vt = kt + KT * KB;
    // ---- scores of 64 keys: S[r][u], u: 32 keys ----
    f32x16 S[RG][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int r = 0; r < RG; ++r)
#pragma unroll
        for (int j = 0; j < 16; ++j) S[r][u][j] = 0.f;
      const int row = 32 * u + la32;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(kt + row * KB + 16 * ((2 * s + g) ^ k_swz<DN>(row)));
#pragma unroll
        for (int r = 0; r < RG; ++r) S[r][u] = mfma32x32x16_bf16(kf, qf[r][s], S[r][u]);
      }
    }
    const bool edge = KT * (t + 1) > vis_min;
    u32x4 P[RG][4];
#pragma unroll
    for (int r = 0; r < RG; ++r) {
      if (edge) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (KT * t + 32 * u + 8 * (j / 4) + 4 * g + j % 4 >= vis[r]) S[r][u][j] = -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 16; ++j) mx = fmaxf(mx, S[r][u][j]);
      mx = x_max_halves(mx) * c2;
      const bool over = mx > ref[r] + kXSlack;
      if (__builtin_amdgcn_ballot_w64(over)) {
        const float to = over ? mx : ref[r];
        const float f = __builtin_amdgcn_exp2f(ref[r] - to);
        ref[r] = to;
        sum[r] *= f;
        if constexpr (LSE) usum[r] *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int j = 0; j < 16; ++j) O[r][d][j] *= f;
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(S[r][u][8 * m + 2 * i], c2, -ref[r]));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(S[r][u][8 * m + 2 * i + 1], c2, -ref[r]));
            const uint32_t w = pack_bf16(p0, p1);
            if constexpr (LSE) usum[r] += p0 + p1;
            P[r][2 * u + m][i] = w;
            sum[r] += bf16_lo(w);
            sum[r] += bf16_hi(w);
          }
    }
    // ---- output ----
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int la = lane & 15;
    bool odd = false;  // a value that is not finite, on a tile that not every row sees
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        u32x2 v[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int row = 16 * m + 8 * half + 4 * g + (la >> 2);
          const int c = (4 * d + 2 * ((lane >> 4) & 1) + ((la & 3) >> 1)) ^ v_swz<DN>(row);
          const uint8_t* const p = vt + row * VB + 16 * c + 8 * (la & 1);
          v[half] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p)));
        }
        u32x4 vf = {v[0].x, v[0].y, v[1].x, v[1].y};
        if (edge) {
          // (weight 0 times such a value would be NaN: it counts for the rows that see it, below)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool lo = (vf[i] & 0x7f80u) == 0x7f80u, hi = (vf[i] & 0x7f800000u) == 0x7f800000u;
            odd |= lo | hi;
            vf[i] &= (lo ? 0xffff0000u : 0xffffffffu) & (hi ? 0xffffu : 0xffffffffu);
          }
        }
#pragma unroll
        for (int r = 0; r < RG; ++r) O[r][d] = mfma32x32x16_bf16(vf, P[r][m], O[r][d]);
      }
    }
    if (edge && __builtin_amdgcn_ballot_w64(odd)) {
#pragma unroll 1
      for (int k = 0; k < KT; ++k) {
        const uint8_t* const vr = vt + k * VB;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int f = 32 * d + 8 * (j / 4) + 4 * g + j % 4;
            const float v = bf16_to_float(
                *reinterpret_cast<const uint16_t*>(vr + 16 * ((f / 8) ^ v_swz<DN>(k)) + 2 * (f % 8)));
            const bool bad = !(fabsf(v) < INFINITY);
#pragma unroll
            for (int r = 0; r < RG; ++r)
              if (bad && KT * t + k < vis[r]) O[r][d][j] += v;
          }
      }
    }
  }

  // ---- normalise and store -----------------------------------------------------------------
#pragma unroll
  for (int r = 0; r < RG; ++r) {
    const int row = row0 + 32 * (RG * wave + r) + la32;
    const bool ok = row < nq;
    const float l = x_add_halves(sum[r]);
    const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
    const float ul = LSE ? x_add_halves(usum[r]) : 0.f;
    const int64_t at = (int64_t)(q0 + min(row, nq - 1)) * a.H + h;
    if (a.splits > 1) {
      const int64_t total = (int64_t)a.T * a.H;
      float* const po = a.ws + (part * total + at) * DN + 4 * g;
      if (ok) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4*>(po + 32 * d + 8 * q) =
                f32x4{O[r][d][4 * q] * inv, O[r][d][4 * q + 1] * inv, O[r][d][4 * q + 2] * inv, O[r][d][4 * q + 3] * inv};
        float* const pl = a.ws + a.splits * total * DN + part * total + at;
        if (g == 0) *pl = l == 0.f ? -INFINITY : ref[r] + __log2f(l);
        if (LSE && g == 0) pl[a.splits * total] = ul == 0.f ? -INFINITY : ref[r] + __log2f(ul);
      }
      continue;
    }
    if (LSE && ok && g == 0) a.lse[at] = ul == 0.f ? -INFINITY : (ref[r] + __log2f(ul)) * kLn2;
    uint16_t* const dst = a.out + (int64_t)(q0 + min(row, nq - 1)) * a.o_st + (int64_t)h * a.o_sh;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      uint32_t w[4][2];  // columns 32 d + 8 q + 4 g + (0..3)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int k = 0; k < 2; ++k) w[q][k] = pack_bf16(O[r][d][4 * q + 2 * k] * inv, O[r][d][4 * q + 2 * k + 1] * inv);
      // the halves' pieces joined to 8 consecutive columns a lane: 32 d + 16 p + 8 g + (0..7)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const auto x = __builtin_amdgcn_permlane32_swap(w[2 * p][0], w[2 * p + 1][0], false, false);
        const auto y = __builtin_amdgcn_permlane32_swap(w[2 * p][1], w[2 * p + 1][1], false, false);
        if (ok) *reinterpret_cast<u32x4*>(dst + 32 * d + 16 * p + 8 * g) = u32x4{x[0], y[0], x[1], y[1]};
      }
    }
  }
}

// Partials of split keys: out = sum_s 2^(lse_s - M) O_s / sum_s 2^(lse_s - M).
template <int DN>
__global__ __launch_bounds__(256) void expanded_merge_kernel(ExpandedArgs a) {
  constexpr int LPR = DN / 4;  // lanes of a row
  const int64_t total = (int64_t)a.T * a.H, at = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  if (at >= total) return;
  const int t = (int)(at / a.H), h = (int)(at - (int64_t)t * a.H), c = threadIdx.x % LPR;
  // rows that belong to no request, or to none of its first max_q_len, have no partials
  bool there = false;
  for (int b = 0; b < a.B; ++b) {
    const int lo = min(max(a.qo_indptr[b], 0), a.T), hi = min(max(a.qo_indptr[b + 1], 0), a.T);
    there |= t >= lo && t < min((int64_t)hi, (int64_t)lo + a.max_q_len);
  }
  if (!there) return;
  const float* const lse = a.ws + a.splits * total * DN + at;
  float M = -INFINITY;
  for (int s = 0; s < a.splits; ++s) M = fmaxf(M, lse[s * total]);
  float den = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const float l = lse[s * total];
    if (l == -INFINITY) continue;
    const float w = __builtin_amdgcn_exp2f(l - M);
    const f32x4 v = *reinterpret_cast<const f32x4*>(a.ws + (s * total + at) * DN + 4 * c);
    den += w;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = fmaf(w, v[i], o[i]);
  }
  const float inv = den == 0.f ? 0.f : 1.f / den;
  if (a.lse && c == 0) {
    const float* const ul = lse + a.splits * total;
    float sum = 0.f;
    for (int s = 0; s < a.splits; ++s)
      if (ul[s * total] != -INFINITY) sum += __builtin_amdgcn_exp2f(ul[s * total] - M);
    a.lse[at] = sum == 0.f ? -INFINITY : (M + __log2f(sum)) * kLn2;
  }
  *reinterpret_cast<u32x2*>(a.out + (int64_t)t * a.o_st + (int64_t)h * a.o_sh + 4 * c) =
      u32x2{pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv)};
}

struct XPlan {
  int64_t blocks;  // row blocks of the batch at most
  int splits;
};
template <int DN, int RG>
XPlan expanded_plan(int64_t T, int64_t N, int B, int H, int max_q_len, int num_cus) {
  using G = XGeo<DN, RG>;
  XPlan p;
  p.blocks = std::min<int64_t>((int64_t)B * ((max_q_len + G::ROWS - 1) / G::ROWS), T / G::ROWS + B);
  // parts of the keys: what gives each CU a block, of four tiles at least in the mean
  const int64_t by_cus = num_cus / std::max<int64_t>(p.blocks * H, 1), by_keys = N / ((int64_t)B * 4 * G::KT);
  p.splits = (int)std::max<int64_t>(1, std::min(by_cus, by_keys));
  return p;
}

template <int DN, int RG, bool LSE>
hipError_t launch_expanded(ExpandedArgs a, int num_cus, hipStream_t stream) {
  using G = XGeo<DN, RG>;
  const XPlan p = expanded_plan<DN, RG>(a.T, a.N, a.B, a.H, a.max_q_len, num_cus);
  a.splits = p.splits;
  const int lds = G::NBUF * G::TILE;
  hipError_t e = hipFuncSetAttribute((const void*)expanded_kernel<DN, RG, LSE>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((expanded_kernel<DN, RG, LSE>), dim3((unsigned)(p.blocks * a.H * a.splits)), dim3(256), lds, stream, a);
  e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  const int64_t rows = (int64_t)a.T * a.H, per = 256 / (DN / 4);
  hipLaunchKernelGGL((expanded_merge_kernel<DN>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace rolaq

int64_t rolaq_expanded_ws_bytes(int64_t T, int64_t N, int B, int H, int DN, int max_q_len, int num_cus) {
  using namespace rolaq;
  const int s = DN == 128 ? expanded_plan<128, 1>(T, N, B, H, max_q_len, num_cus).splits
                          : expanded_plan<64, 1>(T, N, B, H, max_q_len, num_cus).splits;
  return s > 1 ? (int64_t)s * T * H * (DN + 2) * 4 : 0;
}

hipError_t rolaq_launch_expanded(const rolaq::ExpandedArgs& a, int DN, int num_cus, hipStream_t stream) {
  using namespace rolaq;
  if (DN == 128)
    return a.lse ? launch_expanded<128, 1, true>(a, num_cus, stream) : launch_expanded<128, 1, false>(a, num_cus, stream);
  if (DN == 64)
    return a.lse ? launch_expanded<64, 1, true>(a, num_cus, stream) : launch_expanded<64, 1, false>(a, num_cus, stream);
  return hipErrorInvalidValue;
}
