// Attention over expanded latent keys and values (gfx950): per head h
//   s_t = sm_scale (q_nope . k_nope_t,h + q_pe . k_pe_t),  o = sum_t softmax(s)_t v_t,h,
// k_nope and v side by side as kv_b_proj gives them, one k_pe for all heads; causal at the
// end of the keys, or all keys for all queries.
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
  static constexpr int W = 4;                  // waves
  static constexpr int ROWS = 32 * W;          // query rows of a block
  static constexpr int KT = DN == 128 ? 32 : 64;  // keys of a step
  static constexpr int U = KT / 32;            // units of 32 keys
  static constexpr int NB = 2 * DN, PB = 2 * DR;  // bytes of a nope or value row, and of a rope row
  static constexpr int NTILE = KT * NB, PTILE = KT * PB, KTILE = NTILE + PTILE;
  static constexpr int RING = 4;               // steps whose keys, and values, lie in LDS
  static constexpr int V0 = RING * KTILE;      // where the values start
  static constexpr int LDS = V0 + RING * NTILE;
  static constexpr int KS = DK / 16, KN = DN / 16;  // K-steps of the scores, those of the nope part
  static constexpr int ND = DN / 32;           // output column blocks
  static constexpr int SM = KS * U, OM = 2 * ND * U, SLOTS = SM + OM;  // MFMAs of a step
  static_assert(NTILE == 8192 && PTILE == 4096 && 2 * LDS <= 160 * 1024, "5 copies of 1 KB a wave, two blocks a CU");
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

// LSE: for calls that ask for it, the sum of the weights before their rounding as well.
template <int DN, bool LSE>
__global__ __launch_bounds__(256, 2) void expanded_kernel(ExpandedArgs a) {
  using G = XGeo<DN>;
  constexpr int NB = G::NB, PB = G::PB, KT = G::KT, KS = G::KS, KN = G::KN, ND = G::ND, U = G::U, RING = G::RING;
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
  const int steps_all = (sees(min(row0 + G::ROWS, nq) - 1) + KT - 1) / KT;
  const int t0 = (int)((int64_t)steps_all * part / a.splits), t1 = (int)((int64_t)steps_all * (part + 1) / a.splits);
  const int n = t1 - t0;
  const int first_key = KT * t0;  // steps are counted from here

  // ---- tile copies ------------------------------------------------------------------
  // This wave's pieces of a step: two of nope, one of rope, two of values, 64 chunks each.
  const uint8_t* const kv =
      reinterpret_cast<const uint8_t*>(a.kv + (int64_t)(k0 + first_key) * a.kv_st + (int64_t)h * a.kv_sh);
  const uint8_t* const pe = reinterpret_cast<const uint8_t*>(a.pe + (int64_t)(k0 + first_key) * a.pe_st);
  constexpr int NC = NB / 16, PC = PB / 16;  // chunks of a row
  const auto n_row = [&](int j) { return (64 * (2 * wave + j) + lane) / NC; };
  const auto n_off = [&](int j, int row) { return (uint32_t)(row * 2 * (int)a.kv_st); };
  uint32_t noff[2], voff[2], poff;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = n_row(j), c = lane % NC;
    noff[j] = n_off(j, r) + 16 * (c ^ k_swz<NB>(r));
    voff[j] = n_off(j, r) + NB + 16 * (c ^ v_swz<NB>(r));
  }
  const int p_row = (64 * wave + lane) / PC;
  poff = (uint32_t)(p_row * 2 * (int)a.pe_st) + 16 * ((lane % PC) ^ k_swz<PB>(p_row));
  // rows past the last key read that one again
  const auto copy_keys = [&](int t, int slot) {
    const uint8_t* const ks = kv + (int64_t)(KT * t) * (2 * a.kv_st);
    const uint8_t* const ps = pe + (int64_t)(KT * t) * (2 * a.pe_st);
    const uint32_t at = lds0 + slot * G::KTILE;
    const int last = nk - 1 - first_key - KT * t;
    uint32_t o0 = noff[0], o1 = noff[1], o2 = poff;
    if (__builtin_expect(last < KT - 1, 0)) {
      asm volatile("");
      o0 -= n_off(0, max(n_row(0) - last, 0));
      o1 -= n_off(1, max(n_row(1) - last, 0));
      o2 -= (uint32_t)(max(p_row - last, 0) * 2 * (int)a.pe_st);
    }
    copy16(ks, o0, at + 1024 * (2 * wave));
    copy16(ks, o1, at + 1024 * (2 * wave + 1));
    copy16(ps, o2, at + G::NTILE + 1024 * wave);
  };
  const auto copy_values = [&](int t, int slot) {
    const uint8_t* const ks = kv + (int64_t)(KT * t) * (2 * a.kv_st);
    const uint32_t at = lds0 + G::V0 + slot * G::NTILE;
    const int last = nk - 1 - first_key - KT * t;
    uint32_t o0 = voff[0], o1 = voff[1];
    if (__builtin_expect(last < KT - 1, 0)) {
      asm volatile("");
      o0 -= n_off(0, max(n_row(0) - last, 0));
      o1 -= n_off(1, max(n_row(1) - last, 0));
    }
    copy16(ks, o0, at + 1024 * (2 * wave));
    copy16(ks, o1, at + 1024 * (2 * wave + 1));
  };

  // ---- query rows -------------------------------------------------------------------
  const int row = min(row0 + 32 * wave + la32, nq - 1);  // (rows past the last: that one again)
  u32x4 qf[KS];
  {
    const uint16_t* const p = a.q + (int64_t)(q0 + row) * a.q_st + (int64_t)h * a.q_sh + 8 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = gload<u32x4>(p + 16 * s);
  }
  // The first steps' copies go out behind the query's loads, which are waited for here, so that
  // no wait for them is left behind the copies: K 0, K 1, then K j + 2 and V j together.
#pragma unroll
  for (int t = 0; t < RING; ++t)
    if (t < n) copy_keys(t, t);
  if (n > 0) copy_values(0, 0);
  if (n > 1) copy_values(1, 1);
#pragma unroll
  for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qf[s]));
  const int vis = sees(row) - first_key;        // counted from first_key
  const int vis_min = sees(row0) - first_key;   // seen by every row of the block

  f32x16 O[ND];  // O^T: columns 32 d + 8 (j / 4) + 4 g + j % 4 of the lane's row
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int j = 0; j < 16; ++j) O[d][j] = 0.f;
  float ref = kXNoRef, sum = 0.f, usum = 0.f;  // usum (LSE): of the weights as they were
  float most = kXMost;                         // the largest sum of a unit that needs no look at the reference
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
  const auto kread = [&](int slot, int u, int s) {
    return *reinterpret_cast<const u32x4*>(smem + kbase[s] + slot * G::KTILE + u * 32 * (s < KN ? NB : PB));
  };
  // columns 32 d .. of 16 keys m of the values in `slot`, transposed
  const auto vread = [&](int slot, int m, int d) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const uint8_t* const p = smem + vbase[d] + slot * G::NTILE + 16 * m * NB;
    const u32x2 v0 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p)));
    const u32x2 v1 = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * NB)));
    return u32x4{v0.x, v0.y, v1.x, v1.y};
  };

  // ---- the parts of a step ------------------------------------------------------------
  f32x16 zero;
#pragma unroll
  for (int j = 0; j < 16; ++j) zero[j] = 0.f;
  // MFMA i of a step's scores: units in turns, so that chains of one unit are apart
  const auto score = [&](f32x16 (&S)[U], int i, u32x4 k) __attribute__((always_inline)) {
    const int u = i % U, s = i / U;
    S[u] = mfma32x32x16_bf16(k, qf[s], s == 0 ? zero : S[u]);
  };
  const auto output = [&](const u32x4 (&P)[2 * U], int i, u32x4 v) __attribute__((always_inline)) { O[i % ND] = mfma32x32x16_bf16(v, P[i / ND], O[i % ND]); };
  // positions that a row does not see
  const auto mask = [&](f32x16 (&S)[U], int t) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (KT * t + 32 * u + 8 * (j / 4) + 4 * g + j % 4 >= vis) S[u][j] = -INFINITY;
  };
  // Weights of a step in 6 (LSE 8) operations for each of 8 U pairs of keys
  float e0, e1, us[2], uu;
  constexpr int OPS = LSE ? 8 : 6;
  const auto weigh = [&](const f32x16 (&S)[U], u32x4 (&P)[2 * U], int o) __attribute__((always_inline)) {
    const int e = o / OPS, m = e / 4, d = e % 4, j = 8 * (m % 2) + 2 * d;
    switch (o % OPS) {
      case 0: e0 = fmaf(S[m / 2][j], c2, -ref); break;
      case 1: e1 = fmaf(S[m / 2][j + 1], c2, -ref); break;
      case 2: e0 = __builtin_amdgcn_exp2f(e0); break;
      case 3: e1 = __builtin_amdgcn_exp2f(e1); break;
      case 4: {
        uint32_t w = pack_bf16(e0, e1);
        asm volatile("" : "+v"(w));  // formed here, not where a later step uses it
        P[m][d] = w;
        break;
      }
      case 5:
        us[e % 2] = x_sum2(P[m][d], us[e % 2]);
        asm volatile("" : "+v"(us[e % 2]));
        break;
      case 6: uu += e0; break;
      default:
        uu += e1;
        asm volatile("" : "+v"(uu));
        break;
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
      const float to = over ? fmaxf(mx, ref) : ref, f = __builtin_amdgcn_exp2f(ref - to);
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
          s0 = x_sum2(w, s0);
          s1 += p0 + p1;
        }
      got = over ? s0 : got;
      if (LSE) uu = over ? s1 : uu;
    }
    sum += got;
    if (LSE) usum += uu;
  };
  // Values of a step of which a row may not see all may be anything where it does not see them, and 0
  // times what is not finite would be NaN. So before such a step's output every wave looks for
  // one; where there is one, all agree, each clears those of its own pieces,
  // and what they add to the rows that see them comes behind, from memory.
  const auto clean = [&](int slot) __attribute__((always_inline)) {
    u16x2_t big = {0, 0};
    uint8_t* const v = smem + G::V0 + slot * G::NTILE + 16 * lane;
#pragma unroll
    for (int k = 0; k < G::NTILE / 1024; ++k) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(v + 1024 * k);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        big = __builtin_elementwise_max(big, __builtin_bit_cast(u16x2_t, w[e] & 0x7fff7fffu));
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(big[0] >= 0x7f80 || big[1] >= 0x7f80) == 0, 1)) return false;
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
    return true;
  };
  const auto add_cleared = [&](int t) __attribute__((always_inline)) {
#pragma unroll 1
    for (int k = KT * t; k < min(KT * (t + 1), nk - first_key); ++k) {
      const uint8_t* const vr = kv + (int64_t)k * (2 * a.kv_st) + NB + 8 * g;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const u32x2 w = gload<u32x2>(vr + 64 * d + 16 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = e % 2 ? bf16_hi(w[e / 2]) : bf16_lo(w[e / 2]);
            if (k < vis && !(fabsf(x) < INFINITY)) O[d][4 * q + e] += x;
          }
        }
    }
  };

  // Step t, in ring slot I of t: the matrix cores form the scores of step t + 1 and the output of
  // step t - 1 while the vector units turn the scores S of step t into weights.
  // (The first step has zero weights for its output, and zero values: slot RING - 1 is cleared.)
  bool edge_before = false;
  const auto step = [&](auto I, int t, f32x16 (&S)[U], f32x16 (&Sn)[U], u32x4 (&P)[2 * U], const u32x4 (&Pb)[2 * U])
                        __attribute__((always_inline)) {
    constexpr int i = decltype(I)::value, kslot = (i + 1) % RING, vslot = (i + RING - 1) % RING;
    if (t + 3 < n)
      wait_loads<10>();  // K t + 1 and V t - 1 are there; two steps' copies may be under way
    else
      wait_loads<0>();
    __builtin_amdgcn_s_barrier();  // every wave's; and K t and V t - 2 are no longer read
    asm volatile("" ::: "memory");
    if (t + 4 < n) copy_keys(t + 4, i);
    if (t + 2 < n) copy_values(t + 2, (i + 2) % RING);
    const bool edge = KT * (t + 1) > vis_min;
    if (__builtin_expect(edge, 0)) mask(S, t);
    const bool cleared = edge_before && clean(vslot);
    us[0] = us[1] = uu = 0.f;
    // MFMA x of the step: of 5 in a row the second and the fourth are the output's
    constexpr int AHEAD = 4, SL = G::SLOTS, ALL = 8 * U * OPS;
    static_assert(G::SM * 2 == G::OM * 3, "three of the scores to two of the output");
    const auto fetch = [&](int x) __attribute__((always_inline)) {
      const int q = x / 5, r = x % 5;
      if (r % 2 == 0) {
        const int k = 3 * q + r / 2;
        return kread(kslot, k % U, k / U);
      }
      const int k = 2 * q + r / 2;
      return vread(vslot, k / ND, k % ND);
    };
    u32x4 f[AHEAD + 1];
#pragma unroll
    for (int x = 0; x < AHEAD; ++x) f[x] = fetch(x);
#pragma unroll
    for (int x = 0; x < SL; ++x) {
      if (x + AHEAD < SL) f[(x + AHEAD) % (AHEAD + 1)] = fetch(x + AHEAD);
      const int q = x / 5, r = x % 5;
      if (r % 2 == 0)
        score(Sn, 3 * q + r / 2, f[x % (AHEAD + 1)]);
      else
        output(Pb, 2 * q + r / 2, f[x % (AHEAD + 1)]);
#pragma unroll
      for (int o = x * ALL / SL; o < (x + 1) * ALL / SL; ++o) weigh(S, P, o);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (__builtin_expect(cleared, 0)) add_cleared(t - 1);
    settle(S, P);
    edge_before = edge;
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
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int x = 0; x < G::SM; ++x) {
      score(SA, x, kread(0, x % U, x / U));
      __builtin_amdgcn_sched_barrier(0);
    }
    int t = 0;
    for (;;) {
      step(std::integral_constant<int, 0>{}, t, SA, SB, PA, PB_);
      if (++t >= n) break;
      step(std::integral_constant<int, 1>{}, t, SB, SA, PB_, PA);
      if (++t >= n) break;
      step(std::integral_constant<int, 2>{}, t, SA, SB, PA, PB_);
      if (++t >= n) break;
      step(std::integral_constant<int, 3>{}, t, SB, SA, PB_, PA);
      if (++t >= n) break;
    }
    // the last step's output
    wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if ((n & 1) == 0) {
#pragma unroll
      for (int m = 0; m < 2 * U; ++m) PA[m] = PB_[m];
    }
    const int slot = (n - 1) % RING;
    const bool cleared = edge_before && clean(slot);
#pragma unroll
    for (int x = 0; x < G::OM; ++x) {
      output(PA, x, vread(slot, x / ND, x % ND));
      if (x % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
    if (__builtin_expect(cleared, 0)) add_cleared(n - 1);
  }

  // ---- normalise and store -----------------------------------------------------------------
  const bool ok = row0 + 32 * wave + la32 < nq;
  const float l = x_add_halves(sum);
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
  const float ul = LSE ? x_add_halves(usum) : 0.f;
  const int64_t at = (int64_t)(q0 + row) * a.H + h;
  if (a.splits > 1) {
    const int64_t total = (int64_t)a.T * a.H;
    float* const po = a.ws + (part * total + at) * DN + 4 * g;
    if (ok) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<f32x4*>(po + 32 * d + 8 * q) =
              f32x4{O[d][4 * q] * inv, O[d][4 * q + 1] * inv, O[d][4 * q + 2] * inv, O[d][4 * q + 3] * inv};
      float* const pl = a.ws + a.splits * total * DN + part * total + at;
      if (g == 0) *pl = l == 0.f ? -INFINITY : ref + __log2f(l);
      if (LSE && g == 0) pl[a.splits * total] = ul == 0.f ? -INFINITY : ref + __log2f(ul);
    }
    return;
  }
  if (LSE && ok && g == 0) a.lse[at] = ul == 0.f ? -INFINITY : (ref + __log2f(ul)) * kLn2;
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
      const auto x = __builtin_amdgcn_permlane32_swap(w[2 * p][0], w[2 * p + 1][0], false, false);
      const auto y = __builtin_amdgcn_permlane32_swap(w[2 * p][1], w[2 * p + 1][1], false, false);
      if (ok) *reinterpret_cast<u32x4*>(dst + 32 * d + 16 * p + 8 * g) = u32x4{x[0], y[0], x[1], y[1]};
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
template <int DN>
XPlan expanded_plan(int64_t T, int64_t N, int B, int H, int max_q_len, int num_cus) {
  using G = XGeo<DN>;
  XPlan p;
  p.blocks = std::min<int64_t>((int64_t)B * ((max_q_len + G::ROWS - 1) / G::ROWS), T / G::ROWS + B);
  // parts of the keys: what gives each CU a block, of four tiles at least in the mean
  const int64_t by_cus = num_cus / std::max<int64_t>(p.blocks * H, 1), by_keys = N / ((int64_t)B * 256);
  p.splits = (int)std::max<int64_t>(1, std::min(by_cus, by_keys));
  return p;
}

template <int DN, bool LSE>
hipError_t launch_expanded(ExpandedArgs a, int num_cus, hipStream_t stream) {
  using G = XGeo<DN>;
  const XPlan p = expanded_plan<DN>(a.T, a.N, a.B, a.H, a.max_q_len, num_cus);
  a.splits = p.splits;
  const int lds = G::LDS;
  hipError_t e = hipFuncSetAttribute((const void*)expanded_kernel<DN, LSE>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((expanded_kernel<DN, LSE>), dim3((unsigned)(p.blocks * a.H * a.splits)), dim3(256), lds, stream, a);
  e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  const int64_t rows = (int64_t)a.T * a.H, per = 256 / (DN / 4);
  hipLaunchKernelGGL((expanded_merge_kernel<DN>), dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace rolaq

int64_t rolaq_expanded_ws_bytes(int64_t T, int64_t N, int B, int H, int DN, int max_q_len, int num_cus) {
  using namespace rolaq;
  const int s = DN == 128 ? expanded_plan<128>(T, N, B, H, max_q_len, num_cus).splits
                          : expanded_plan<64>(T, N, B, H, max_q_len, num_cus).splits;
  return s > 1 ? (int64_t)s * T * H * (DN + 2) * 4 : 0;
}

hipError_t rolaq_launch_expanded(const rolaq::ExpandedArgs& a, int DN, int num_cus, hipStream_t stream) {
  using namespace rolaq;
  if (DN == 128)
    return a.lse ? launch_expanded<128, true>(a, num_cus, stream) : launch_expanded<128, false>(a, num_cus, stream);
  if (DN == 64)
    return a.lse ? launch_expanded<64, true>(a, num_cus, stream) : launch_expanded<64, false>(a, num_cus, stream);
  return hipErrorInvalidValue;
}
