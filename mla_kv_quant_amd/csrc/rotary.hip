// Rotary positions (gfx950): the rope parts of queries and keys, turned by their tokens'
// positions in one launch.
//
// A pair (a, b) of a head -- neighbours, or half a width apart -- at position p becomes
//   (s (a cos w - b sin w), s (b cos w + a sin w)),  w = 2 pi p f,
// f the pair's turns for a step of one position. f is held as a 64-bit fraction of a turn, so
// that p f modulo one turn is a 64-bit product without its upper half: exact to |p| 2^-65
// of a turn for positions of any size and sign. (FP32 angles, as frameworks
// form them, are off by up to 2^-8 at position 10^5.) What is left is an eighth of a
// turn at most to either side, where sine and cosine are their Taylor series.
//
// Bound: HBM for many tokens, a launch for few. A thread holds the sines and cosines of a few pairs of one
// token and goes through some of its heads with them, four heads' loads under way at once; 16-byte loads and
// stores where the tensors allow them, else a pair at a time. 33 us for 32768 tokens of 16 heads and one key of
// 64 bf16 values out of wider rows, 143 MB at 4.3 TB/s (a plain copy of the same rows: 32); 3.2 us for 8 tokens.
// Threads go on to later tokens, as the frequencies, strides and divisions of their start are worth
// half of a token's work (49 us with a thread for each token, and addresses formed head by head).
#include "rolaq_common.h"
#include "serve_args.h"

#include <algorithm>
#include <type_traits>

namespace rolaq {

// Sine and cosine of t / 2^64 of a turn, to 2^-24 of the largest.
__device__ __forceinline__ void sincos_turn(uint64_t t, float& sn, float& cs) {
  const uint32_t u = (uint32_t)(t >> 32) + (uint32_t)((t >> 31) & 1);
  const uint32_t quarter = (u + 0x20000000u) >> 30;
  // the rest, -2^29 .. 2^29 of 2^32, as an angle
  const float w = (float)(int32_t)(u - (quarter << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  const float z = w * w;
  // sum of (-1)^k w^(2 k + 1) / (2 k + 1)! and (-1)^k w^(2 k) / (2 k)!; the next terms are below 2e-9
  float s = fmaf(z, 2.7557319e-6f, -1.9841270e-4f);
  s = fmaf(z, s, 8.3333333e-3f);
  s = fmaf(z, s, -1.6666667e-1f);
  s = fmaf(z * s, w, w);
  float c = fmaf(z, -2.7557319e-7f, 2.4801587e-5f);
  c = fmaf(z, c, -1.3888889e-3f);
  c = fmaf(z, c, 4.1666667e-2f);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.0f);
  const float s1 = quarter & 1 ? c : s, c1 = quarter & 1 ? s : c;
  sn = quarter & 2 ? -s1 : s1;
  cs = (quarter + 1) & 2 ? -c1 : c1;
}

__device__ __forceinline__ float to_float(uint16_t v, std::integral_constant<int, ROLAQ_BF16>) { return bf16_to_float(v); }
__device__ __forceinline__ float to_float(uint16_t v, std::integral_constant<int, ROLAQ_FP16>) {
  return (float)__builtin_bit_cast(_Float16, v);
}
__device__ __forceinline__ float to_float(float v, std::integral_constant<int, ROLAQ_FP32>) { return v; }
__device__ __forceinline__ void from_float(uint16_t& d, float v, std::integral_constant<int, ROLAQ_BF16>) { d = float_to_bf16(v); }
__device__ __forceinline__ void from_float(uint16_t& d, float v, std::integral_constant<int, ROLAQ_FP16>) {
  d = __builtin_bit_cast(uint16_t, (_Float16)v);
}
__device__ __forceinline__ void from_float(float& d, float v, std::integral_constant<int, ROLAQ_FP32>) { d = v; }

// V pairs a thread: V = 1, or as many as fill 16 bytes (neighbours: half as many as
// there are values in them; halves: two pieces, one of each half).
template <int TYPE, bool TWO, int V>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  using T = typename std::conditional<TYPE == ROLAQ_FP32, float, uint16_t>::type;
  constexpr std::integral_constant<int, TYPE> type{};
  constexpr int N = TWO ? 2 * V : V;  // values of a piece
  constexpr int PIECES = TWO ? 1 : 2;
  struct alignas(V == 1 ? sizeof(T) : 16) Vec {
    T v[N];
  };
  const int per = a.groups * a.slots;
  const int tok = threadIdx.x / per, rest = threadIdx.x - tok * per;
  const int slot = rest / a.groups, g = rest - slot * a.groups;
  if (tok >= a.tokens) return;
  uint64_t f[V];
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = a.turns[V * g + i];
  // (those of the second tensor go on where the first one's end)
  const int behind = slot >= a.H % a.slots ? slot - a.H % a.slots : slot + a.slots - a.H % a.slots;
  for (int64_t t = (int64_t)blockIdx.x * a.tokens + tok; t < a.T; t += (int64_t)gridDim.x * a.tokens) {
    const uint64_t p = (uint64_t)a.positions[t];
    float sn[V], cs[V];
    constexpr int AHEAD = 4;  // heads whose loads are under way together
    // heads from, from + slots .. of n (from < slots)
    const auto turn = [&](int which, int from, int n, bool first) __attribute__((always_inline)) {
      const T* const x = static_cast<const T*>(a.x[which]) + t * a.x_st[which] + N * g;
      T* const y = static_cast<T*>(a.y[which]) + t * a.y_st[which] + N * g;
      for (int h0 = 0; h0 < n; h0 += AHEAD * a.slots) {
        Vec in[AHEAD][PIECES];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          if (h0 + j * a.slots >= n) break;
          const T* const head = x + min(h0 + j * a.slots + from, n - 1) * a.x_sh[which];
#pragma unroll
          for (int i = 0; i < PIECES; ++i) in[j][i] = *reinterpret_cast<const Vec*>(head + i * a.pairs);
        }
        if (first) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            sincos_turn(p * f[i], sn[i], cs[i]);
            sn[i] *= a.scale;
            cs[i] *= a.scale;
          }
          first = false;
        }
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
          const int h = h0 + j * a.slots + from;
          if (h >= n) break;
          T* const to = y + h * a.y_sh[which];
          Vec out[PIECES];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float u = to_float(TWO ? in[j][0].v[2 * i] : in[j][0].v[i], type);
            const float v = to_float(TWO ? in[j][0].v[2 * i + 1] : in[j][PIECES - 1].v[i], type);
            from_float(TWO ? out[0].v[2 * i] : out[0].v[i], u * cs[i] - v * sn[i], type);
            from_float(TWO ? out[0].v[2 * i + 1] : out[PIECES - 1].v[i], v * cs[i] + u * sn[i], type);
          }
#pragma unroll
          for (int i = 0; i < PIECES; ++i) *reinterpret_cast<Vec*>(to + i * a.pairs) = out[i];
        }
      }
    };
    // (slots is at most H: every thread has a head of the first tensor)
    turn(0, slot, a.H, true);
    turn(1, behind, a.Hk, false);
  }
}

template <int TYPE, bool TWO, int V>
hipError_t launch_rotary(RotaryArgs a, int num_cus, hipStream_t stream) {
  a.groups = a.pairs / V;
  // Heads side by side: as many as a block has room for while the card is not full; where tokens alone
  // fill it a quarter of them, so that sines and cosines serve four (32768 tokens of 16: 33 us, each its
  // own 64).
  const int room = std::max(1, 256 / a.groups);
  const int64_t threads = (int64_t)num_cus * 1024;
  const int64_t wanted = (threads + a.T * a.groups - 1) / (a.T * a.groups);
  a.slots = (int)std::min<int64_t>({(int64_t)room, (int64_t)a.H, std::max<int64_t>(wanted, (a.H + 3) / 4)});
  a.tokens = std::max(1, 256 / (a.groups * a.slots));
  // (eight blocks a CU: two turns of the four of the 16-byte bf16 kernels that are resident, by their 103 and 124 registers)
  const int64_t blocks = std::min<int64_t>((a.T + a.tokens - 1) / a.tokens, 8 * num_cus);
  hipLaunchKernelGGL((rotary_kernel<TYPE, TWO, V>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return hipGetLastError();
}

template <int TYPE, bool TWO>
hipError_t launch_rotary_vec(const RotaryArgs& a, int num_cus, hipStream_t stream) {
  constexpr int size = TYPE == ROLAQ_FP32 ? 4 : 2, V = TWO ? 8 / size : 16 / size;
  bool vec = a.pairs % V == 0;
  for (int i = 0; i < (a.Hk ? 2 : 1); ++i) {
    vec = vec && (reinterpret_cast<uintptr_t>(a.x[i]) | reinterpret_cast<uintptr_t>(a.y[i])) % 16 == 0;
    for (int64_t s : {a.x_st[i], a.x_sh[i], a.y_st[i], a.y_sh[i]}) vec = vec && s * size % 16 == 0;
  }
  if (vec) return launch_rotary<TYPE, TWO, V>(a, num_cus, stream);
  return launch_rotary<TYPE, TWO, 1>(a, num_cus, stream);
}

}  // namespace rolaq

hipError_t rolaq_launch_rotary(const rolaq::RotaryArgs& a, int type, bool interleaved, int num_cus, hipStream_t stream) {
  using namespace rolaq;
#define ROLAQ_ROTARY(TYPE)                                                      \
  if (type == TYPE)                                                             \
    return interleaved ? launch_rotary_vec<TYPE, true>(a, num_cus, stream)      \
                       : launch_rotary_vec<TYPE, false>(a, num_cus, stream);
  ROLAQ_ROTARY(ROLAQ_BF16)
  ROLAQ_ROTARY(ROLAQ_FP16)
  ROLAQ_ROTARY(ROLAQ_FP32)
#undef ROLAQ_ROTARY
  return hipErrorInvalidValue;
}
