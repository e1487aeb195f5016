// Eviction by accumulated attention weight (gfx950): which positions of each request stay.
//
// Of a request's n cached positions stay the first `sink`, the last `recent` and, of
// the others, the `need` = budget - sink - recent of largest weight; of equal ones the earlier. A NaN
// counts as the largest, -0 as 0. All stay where n <= budget. Written are their slots and weights in
// order of position, their number, and the slots of the others.
//
// The need-th largest weight is found digit by digit from a histogram of the weights' bits as
// ordered integers (11, 11 and 10 bits): the digit of the bin in which the count from the top
// passes what is needed, then the next digit among that bin's weights. What stays is then known
// position by position, and a running count gives each its place:
// above the threshold, or equal to it while fewer than the rest have been seen.
//
// Bound: latency. A request of up to 16384 positions is one block, which holds the weights in
// registers and goes through all steps with barriers alone. Longer ones are cut into chunks of
// that size, a block each, and the steps into four launches; every chunk leaves its
// histogram, from which the next launch's blocks find the bin, and the places of what
// stays in the chunks before them, for themselves: no atomics on memory, nothing to clear.
#include "rolaq_common.h"
#include "serve_args.h"

#include <algorithm>

namespace rolaq {

constexpr int kEvictThreads = 1024, kEvictPer = 16;
constexpr int kEvictChunk = kEvictThreads * kEvictPer;  // positions of a block
constexpr int kEvictBins = 2048;
constexpr int kEvictWaves = kEvictThreads / 64;

// Weights as integers of the same order; two zeros are equal, a NaN is the largest.
__device__ __forceinline__ uint32_t evict_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w + 0.f);  // -0 + 0 = 0
  return (int32_t)b < 0 ? ~b : b | 0x80000000u;
}
// Digit d (0: the highest) and the bits above it.
__device__ __forceinline__ uint32_t evict_digit(uint32_t key, int d) {
  return d == 0 ? key >> 21 : d == 1 ? (key >> 10) & 2047u : key & 1023u;
}
__device__ __forceinline__ bool evict_same(uint32_t key, uint32_t top, int d) {
  return d == 0 || (d == 1 ? (key ^ top) >> 21 == 0 : (key ^ top) >> 10 == 0);
}

struct EvictRequest {
  int64_t list;   // first entry of its page list
  int64_t n;      // positions
  const float* row;  // its accumulated weights (null: all 0)
  float* out;
};

__device__ __forceinline__ int64_t evict_len(const EvictArgs& a, int b, int64_t* list) {
  const int64_t first = max(a.kv_indptr[b], 0), end = min((int64_t)max(a.kv_indptr[b + 1], 0), a.n_indices);
  *list = first;
  const int64_t reach = max(end - first, (int64_t)0) << a.page_shift;
  return max(min(min(a.kv_lens[b], reach), a.most), (int64_t)0);
}

__device__ __forceinline__ EvictRequest evict_request(const EvictArgs& a, int b) {
  EvictRequest r;
  r.n = evict_len(a, b, &r.list);
  const int64_t req = a.req_idx ? a.req_idx[b] : b;
  const bool there = req >= 0 && req < a.acc_rows;
  r.row = there ? a.acc + req * a.acc_st : nullptr;
  r.out = there ? a.acc_out + req * a.acc_out_st : nullptr;
  return r;
}

// The block's shared memory.
struct EvictShared {
  uint32_t hist[kEvictBins];
  uint32_t wave[kEvictWaves];
  uint32_t bin, above;
  uint32_t count[kEvictPer * kEvictWaves];  // of a wave's turn: above the threshold, equal << 16
  uint64_t sum;
};

// Sum of v over the threads of all lower numbers; *all: over all threads.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* waves, uint32_t* all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t s = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = (uint32_t)__shfl_up((int)s, o);
    if (lane >= o) s += u;
  }
  __syncthreads();  // (waves may still be read from the last call)
  if (lane == 63) waves[wave] = s;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kEvictWaves; ++w) {
    before += w < wave ? waves[w] : 0;
    total += waves[w];
  }
  *all = total;
  return before + s - v;
}

// The bin in which the count from the top passes `need` (of sh.hist), and the count above it.
__device__ void evict_find(EvictShared& sh, uint32_t need) {
  const int t = threadIdx.x;
  // thread t has the bins 2047 - 2 t and 2046 - 2 t
  const uint32_t h0 = sh.hist[kEvictBins - 1 - 2 * t], h1 = sh.hist[kEvictBins - 2 - 2 * t];
  uint32_t all;
  const uint32_t before = block_scan(h0 + h1, sh.wave, &all);
  if (before < need && need <= before + h0) sh.bin = kEvictBins - 1 - 2 * t, sh.above = before;
  if (before + h0 < need && need <= before + h0 + h1) sh.bin = kEvictBins - 2 - 2 * t, sh.above = before + h0;
  __syncthreads();
}

// Where several blocks share a request: a request's part of the workspace. Per
// chunk the weights and the three histograms.
struct EvictWs {
  uint32_t* hist;  // [chunks][3][kEvictBins]
  float* w;        // [chunks * kEvictChunk]
};
__device__ __forceinline__ EvictWs evict_ws(const EvictArgs& a, int b) {
  EvictWs ws;
  ws.hist = reinterpret_cast<uint32_t*>(a.ws) + (int64_t)b * a.chunks * 3 * kEvictBins;
  ws.w = reinterpret_cast<float*>(reinterpret_cast<uint32_t*>(a.ws) + (int64_t)a.B * a.chunks * 3 * kEvictBins) +
         (int64_t)b * a.chunks * kEvictChunk;
  return ws;
}

// STEP -1: everything, one block a request. 0, 1, 2: the histogram of that digit; 3: what stays.
template <int STEP>
__global__ __launch_bounds__(kEvictThreads) void evict_kernel(EvictArgs a) {
  __shared__ EvictShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int chunk = STEP < 0 ? 0 : (int)(blockIdx.x % (unsigned)a.chunks);
  const int b = STEP < 0 ? (int)blockIdx.x : (int)(blockIdx.x / (unsigned)a.chunks);
  const EvictRequest r = evict_request(a, b);
  const int64_t base = (int64_t)chunk * kEvictChunk;
  const bool all_stay = r.n <= a.budget;
  if (STEP >= 0 && STEP < 3 && (base >= r.n || (all_stay && STEP > 0))) return;
  if (STEP == 3 && chunk > 0 && base >= r.n) return;
  const int64_t mid0 = a.sink, mid1 = r.n - a.recent;  // the positions that have to compete
  const uint32_t need = (uint32_t)(a.budget - a.sink - a.recent);

  float w[kEvictPer];
  const auto at = [&](int i) { return base + (int64_t)i * kEvictThreads + tid; };
  const auto competes = [&](int64_t p) { return !all_stay && p >= mid0 && p < mid1; };
  EvictWs ws{};
  if (STEP >= 0) ws = evict_ws(a, b);
#pragma unroll
  for (int i = 0; i < kEvictPer; ++i) {
    const int64_t p = at(i);
    w[i] = 0.f;
    if (STEP <= 0) {
      if (r.row && p < r.n) w[i] = r.row[p];
    } else {
      if (p < r.n) w[i] = ws.w[p];
    }
  }
  if (STEP == 0) {
#pragma unroll
    for (int i = 0; i < kEvictPer; ++i)
      if (at(i) < r.n) ws.w[at(i)] = w[i];
    if (all_stay) return;
  }

  // ---- the threshold ------------------------------------------------------------
  uint32_t top = 0, left = need;  // its bits so far; how many of its bin are needed
  if (!all_stay && need > 0) {
#pragma unroll
    for (int d = 0; d < 3; ++d) {
      if (STEP >= 0 && d > STEP) break;
      __syncthreads();
      if (STEP < 0 || d == STEP) {
        // this block's histogram
        for (int i = tid; i < kEvictBins; i += kEvictThreads) sh.hist[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEvictPer; ++i) {
          const uint32_t k = evict_key(w[i]);
          if (competes(at(i)) && evict_same(k, top, d)) atomicAdd(&sh.hist[evict_digit(k, d)], 1u);
        }
        __syncthreads();
        if (STEP >= 0) {
          uint32_t* const to = ws.hist + ((int64_t)chunk * 3 + d) * kEvictBins;
          for (int i = tid; i < kEvictBins; i += kEvictThreads) to[i] = sh.hist[i];
          return;
        }
      } else {
        // an earlier launch's, of all chunks
        const int used = (int)((r.n + kEvictChunk - 1) / kEvictChunk);
        for (int i = tid; i < kEvictBins; i += kEvictThreads) {
          uint32_t s = 0;
          for (int c = 0; c < used; ++c) s += ws.hist[((int64_t)c * 3 + d) * kEvictBins + i];
          sh.hist[i] = s;
        }
        __syncthreads();
      }
      evict_find(sh, left);
      left -= sh.above;
      top |= sh.bin << (d == 0 ? 21 : d == 1 ? 10 : 0);
    }
  }
  if (STEP >= 0 && STEP < 3) return;

  // ---- what stays, and its places --------------------------------------------------
  // Before this chunk: kept ones that competed above the threshold, and equal ones.
  uint32_t more = 0, equal = 0;
  if (STEP == 3 && chunk > 0 && !all_stay && need > 0) {
    uint32_t m = 0, e = 0;
    for (int c = 0; c < chunk; ++c) {
      const uint32_t* const h = ws.hist + (int64_t)c * 3 * kEvictBins;
      for (int i = tid; i < kEvictBins; i += kEvictThreads) {
        m += (uint32_t)i > top >> 21 ? h[i] : 0;
        m += (uint32_t)i > ((top >> 10) & 2047u) ? h[kEvictBins + i] : 0;
        m += (uint32_t)i > (top & 1023u) ? h[2 * kEvictBins + i] : 0;
        e += (uint32_t)i == (top & 1023u) ? h[2 * kEvictBins + i] : 0;
      }
    }
    block_scan(m, sh.wave, &more);
    block_scan(e, sh.wave, &equal);
  }
  if (!all_stay && chunk > 0) more += (uint32_t)min((int64_t)a.sink, base);  // (the first ones, all before it)
  if (all_stay) more = (uint32_t)base;
  // (the last ones of chunks before this one stay as well)
  if (!all_stay && base > mid1) more += (uint32_t)(base - mid1);

  uint32_t flags[kEvictPer];  // bit 0: stays for certain; bit 1: equal to the threshold
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEvictPer; ++i) {
    const int64_t p = at(i);
    bool sure = false, same = false;
    if (p < r.n) {
      if (!competes(p)) {
        sure = true;
      } else if (need > 0) {
        const uint32_t k = evict_key(w[i]);
        sure = k > top;
        same = k == top;
      }
    }
    const uint64_t s = __ballot(sure), e = __ballot(same);
    // lanes below this one, of either kind
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    flags[i] = (uint32_t)sure | (uint32_t)same << 1 | (uint32_t)__popcll(s & below) << 8 | (uint32_t)__popcll(e & below) << 16;
    if (lane == 0) sh.count[i * kEvictWaves + wave] = (uint32_t)__popcll(s) | (uint32_t)__popcll(e) << 16;
  }
  __syncthreads();
  // running counts over turns and waves (each at most kEvictChunk: 16 bits hold all but the last's sum)
  static_assert(kEvictPer * kEvictWaves <= kEvictThreads, "one thread a count");
  {
    const uint32_t c = tid < kEvictPer * kEvictWaves ? sh.count[tid] : 0;
    uint32_t all;
    const uint32_t s = block_scan(c & 0xffffu, sh.wave, &all);
    const uint32_t e = block_scan(c >> 16, sh.wave, &all);
    __syncthreads();
    if (tid < kEvictPer * kEvictWaves) sh.count[tid] = s | e << 16;
    __syncthreads();
  }
  // slots freed by the requests before this one, and by this one before the chunk
  {
    uint64_t mine = 0;
    for (int i = tid; i < b; i += kEvictThreads) {
      int64_t list;
      mine += (uint64_t)max(evict_len(a, i, &list) - a.budget, (int64_t)0);
    }
    if (tid == 0) sh.sum = 0;
    __syncthreads();
    if (mine) atomicAdd((unsigned long long*)&sh.sum, (unsigned long long)mine);
    __syncthreads();
  }
  const int64_t freed0 = (int64_t)sh.sum;
  const int64_t stay = min(r.n, (int64_t)a.budget);
  if (chunk == 0 && tid == 0) a.kept_lens[b] = stay;
  const uint32_t mask = (1u << a.page_shift) - 1;
#pragma unroll
  for (int i = 0; i < kEvictPer; ++i) {
    const int64_t p = at(i);
    if (p >= r.n) break;
    const uint32_t c = sh.count[i * kEvictWaves + wave];
    const uint32_t s = more + (c & 0xffffu) + ((flags[i] >> 8) & 0xffu);
    const uint32_t e = equal + (c >> 16) + (flags[i] >> 16);
    const bool keeps = (flags[i] & 1) || ((flags[i] & 2) && e < left);
    const int64_t place = (int64_t)s + min(e, left);  // kept ones before this position
    const int32_t slot =
        (int32_t)(((uint32_t)a.kv_indices[r.list + (p >> a.page_shift)] << a.page_shift) + ((uint32_t)p & mask));
    if (keeps) {
      a.kept[(int64_t)b * a.budget + place] = slot;
      if (r.out) r.out[place] = w[i];
    } else {
      const int64_t to = freed0 + (p - place);
      if (to < a.freed_size) a.freed[to] = slot;
    }
    if (r.out && p >= stay) r.out[p] = 0.f;
  }
}

}  // namespace rolaq

int64_t rolaq_evict_ws_bytes(int64_t B, int64_t most) {
  using namespace rolaq;
  const int64_t chunks = (most + kEvictChunk - 1) / kEvictChunk;
  return chunks <= 1 ? 0 : B * chunks * (3 * kEvictBins + kEvictChunk) * 4;
}

hipError_t rolaq_launch_evict(const rolaq::EvictArgs& args, hipStream_t stream) {
  using namespace rolaq;
  EvictArgs a = args;
  a.chunks = (int)((a.most + kEvictChunk - 1) / kEvictChunk);
  if (a.chunks <= 1) {
    hipLaunchKernelGGL((evict_kernel<-1>), dim3(a.B), dim3(kEvictThreads), 0, stream, a);
    return hipGetLastError();
  }
  const dim3 grid((unsigned)((int64_t)a.B * a.chunks));
  hipLaunchKernelGGL((evict_kernel<0>), grid, dim3(kEvictThreads), 0, stream, a);
  hipLaunchKernelGGL((evict_kernel<1>), grid, dim3(kEvictThreads), 0, stream, a);
  hipLaunchKernelGGL((evict_kernel<2>), grid, dim3(kEvictThreads), 0, stream, a);
  hipLaunchKernelGGL((evict_kernel<3>), grid, dim3(kEvictThreads), 0, stream, a);
  return hipGetLastError();
}
