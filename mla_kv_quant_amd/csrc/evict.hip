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
// registers and goes through all steps with barriers alone: 17 us for 32 requests of 16384, of
// which 5 go until the weights and page numbers are there, 2 to 3 into each digit, 6 into what is written; a
// block's own instructions, on one CU. (Weights may share their leading bits: two copies of a histogram, for even
// and odd lanes, halve what equal bins cost and no more, at no loss otherwise; eight, 64 KB to clear and
// add up, were 3 us slower.)
// Longer requests are cut into chunks, a block each, and the steps into four launches. Every chunk leaves its
// histogram as counts from the top down to each bin, from which the next launch's blocks find the bin for
// themselves, and the last one's the number of what stays in the chunks before theirs with one look into each:
// no atomics on memory, nothing to clear. 30 us for one request of 131072: launches of 5, 8, 8 and 10 us.
#include "rolaq_common.h"
#include "mx4_request.h"
#include "serve_args.h"

#include <algorithm>

namespace rolaq {

constexpr int kEvictThreads = 1024;
constexpr int kEvictOne = 16 * kEvictThreads;  // the most positions of a request that is one block
constexpr int kEvictBins = 2048, kEvictCopies = 2;
constexpr int64_t kEvictSmall = 48 * 4096;
constexpr int kEvictWaves = kEvictThreads / 64;

// Weights as integers of the same order; two zeros are equal, a NaN is the largest. No weight is below 2^21.
__device__ __forceinline__ uint32_t evict_key(float w) {
  const uint32_t b = __float_as_uint(w + 0.f);  // -0 + 0 = 0
  return w != w ? 0xffffffffu : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
constexpr uint32_t kEvictNone = 0, kEvictStays = 1;  // in a key's place: no position; one that stays by itself
// Digit d (0: the highest) and the bits above it.
__device__ __forceinline__ uint32_t evict_digit(uint32_t key, int d) {
  return d == 0 ? key >> 21 : d == 1 ? (key >> 10) & 2047u : key & 1023u;
}
__device__ __forceinline__ bool evict_same(uint32_t key, uint32_t top, int d) {
  return d == 0 || (d == 1 ? (key ^ top) >> 21 == 0 : (key ^ top) >> 10 == 0);
}

struct EvictRequest {
  int64_t list;      // first entry of its page list
  int n;             // positions
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
  r.n = (int)evict_len(a, b, &r.list);
  const int64_t req = a.req_idx ? a.req_idx[b] : b;
  const bool there = req >= 0 && req < a.acc_rows;
  r.row = there ? a.acc + req * a.acc_st : nullptr;
  r.out = there ? a.acc_out + req * a.acc_out_st : nullptr;
  return r;
}

// The block's shared memory besides the histogram.
struct EvictShared {
  uint32_t wave[2][kEvictWaves];
  uint32_t bin, above;
  uint64_t sum;
};

// Sum of v over the threads of all lower numbers. `turn`: 0 and 1 in turn, so that one
// barrier is enough.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, EvictShared& sh, int turn, uint32_t* all) {
  const int wave = threadIdx.x >> 6;
  const uint32_t s = wave_scan(v);
  if ((threadIdx.x & 63) == 63) sh.wave[turn][wave] = s;
  __syncthreads();
  uint32_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kEvictWaves; ++w) {
    const uint32_t x = sh.wave[turn][w];
    before += w < wave ? x : 0;
    total += x;
  }
  *all = total;
  return before + s - v;
}

// Where several blocks share a request: a request's part of the workspace.
struct EvictWs {
  uint32_t* counts;  // [chunks][3][kEvictBins]: weights of a chunk in this bin of the digit and those above it
  uint32_t* found;   // [2][2]: after the first and second digit: the threshold's bits, and how many of its bin are needed
  float* w;          // [chunks * chunk]
};
__device__ __forceinline__ EvictWs evict_ws(const EvictArgs& a, int b, int64_t chunk) {
  EvictWs ws;
  uint32_t* const at = reinterpret_cast<uint32_t*>(a.ws);
  const int64_t counts = (int64_t)a.chunks * 3 * kEvictBins;
  ws.counts = at + b * counts;
  ws.found = at + a.B * counts + 4 * b;
  ws.w = reinterpret_cast<float*>(at + a.B * (counts + 4) + b * a.chunks * chunk);
  return ws;
}

// STEP -1: everything, one block a request. 0, 1, 2: the counts of that digit; 3: what stays.
template <int STEP, int PER>
__global__ __launch_bounds__(kEvictThreads) void evict_kernel(EvictArgs a) {
  constexpr int kChunk = PER * kEvictThreads;  // positions of a block
  __shared__ __attribute__((aligned(16))) uint32_t hist[kEvictBins * kEvictCopies];
  __shared__ EvictShared sh;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int chunk = STEP < 0 ? 0 : (int)(blockIdx.x % (unsigned)a.chunks);
  const int b = STEP < 0 ? (int)blockIdx.x : (int)(blockIdx.x / (unsigned)a.chunks);
  const EvictRequest r = evict_request(a, b);
  const int base = chunk * kChunk;
  const bool all_stay = r.n <= a.budget;
  if (STEP >= 0 && STEP < 3 && (base >= r.n || (all_stay && STEP > 0))) return;
  if (STEP == 3 && chunk > 0 && base >= r.n) return;
  const int mid0 = a.sink, mid1 = r.n - a.recent;  // between them they have to compete
  const uint32_t need = (uint32_t)(a.budget - a.sink - a.recent);

  float w[PER];
  const auto at = [&](int i) { return base + i * kEvictThreads + tid; };
  EvictWs ws{};
  if (STEP >= 0) ws = evict_ws(a, b, kChunk);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int p = at(i);
    w[i] = 0.f;
    if (STEP <= 0) {
      if (r.row && p < r.n) w[i] = r.row[p];
    } else {
      if (p < r.n) w[i] = ws.w[p];
    }
  }
  // slots, and those freed by the requests before this one
  constexpr bool kLast = STEP < 0 || STEP == 3;
  int32_t page[kLast ? PER : 1];
  if constexpr (kLast) {
#pragma unroll
    for (int i = 0; i < PER; ++i) page[i] = at(i) < r.n ? a.kv_indices[r.list + (at(i) >> a.page_shift)] : 0;
    if (tid == 0) sh.sum = 0;
    uint64_t mine = 0;
    for (int i = tid; i < b; i += kEvictThreads) {
      int64_t list;
      mine += (uint64_t)max(evict_len(a, i, &list) - a.budget, (int64_t)0);
    }
    __syncthreads();
    if (mine) atomicAdd((unsigned long long*)&sh.sum, (unsigned long long)mine);
  }
  if (STEP == 0) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (at(i) < r.n) ws.w[at(i)] = w[i];
    if (all_stay) return;
  }

  uint32_t key[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int p = at(i);
    key[i] = evict_key(w[i]);
    if (all_stay || p < mid0 || p >= mid1) key[i] = kEvictStays;
    if (p >= r.n) key[i] = kEvictNone;
  }

  // ---- the threshold ------------------------------------------------------------
  uint32_t top = 0, left = need;  // its bits so far; how many of its bin are needed
  if (all_stay || need == 0) top = 0xffffffffu, left = 0;
  if (!all_stay && need > 0) {
    if (STEP >= 2) top = ws.found[2 * (STEP - 2)], left = ws.found[2 * (STEP - 2) + 1];
    const int hi = kEvictBins - 1 - 2 * tid;  // this thread's bins are hi and hi - 1
    u32x4* const mine = reinterpret_cast<u32x4*>(hist + (hi - 1) * kEvictCopies);  // their copies
    if (STEP < 3) *mine = u32x4{0, 0, 0, 0};
#pragma unroll
    for (int d = 0; d < 3; ++d) {
      if (STEP >= 0 && (d > STEP || d + 1 < STEP)) continue;
      uint32_t c1, c0;  // weights in bin hi and above, and those of hi - 1 as well
      if (STEP < 0 || d == STEP) {
        // this block's counts
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const uint32_t k = key[i];
          if (k > kEvictStays && evict_same(k, top, d))
            atomicAdd(&hist[evict_digit(k, d) * kEvictCopies + lane % kEvictCopies], 1u);
        }
        __syncthreads();
        const u32x4 h = *mine;
        const uint32_t h0 = h[0] + h[1], h1 = h[2] + h[3];
        if (STEP < 0) *mine = u32x4{0, 0, 0, 0};
        uint32_t all;
        c1 = block_scan(h0 + h1, sh, d & 1, &all) + h1;
        c0 = c1 + h0;
        if (STEP >= 0) {
          *reinterpret_cast<u32x2*>(ws.counts + ((int64_t)chunk * 3 + d) * kEvictBins + hi - 1) = u32x2{c0, c1};
          return;
        }
        if (c1 - h1 < left && left <= c1) sh.bin = hi, sh.above = c1 - h1;
        if (c1 < left && left <= c0) sh.bin = hi - 1, sh.above = c1;
      } else {
        // the last launch's, of all chunks
        const int used = (r.n + kChunk - 1) / kChunk;
        const uint32_t* const from = ws.counts + d * kEvictBins + hi - 1;
        c1 = c0 = 0;
#pragma unroll 8
        for (int c = 0; c < used; ++c) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(from + (int64_t)c * 3 * kEvictBins);
          c0 += x[0];
          c1 += x[1];
        }
        // (bin hi + 1 is the next lower thread's hi - 1)
        uint32_t above = (uint32_t)__shfl_up((int)c0, 1);
        if (lane == 63) sh.wave[0][wave] = c0;
        __syncthreads();
        if (lane == 0) above = wave ? sh.wave[0][wave - 1] : 0;
        if (above < left && left <= c1) sh.bin = hi, sh.above = above;
        if (c1 < left && left <= c0) sh.bin = hi - 1, sh.above = c1;
      }
      __syncthreads();
      left -= sh.above;
      top |= sh.bin << (d == 0 ? 21 : d == 1 ? 10 : 0);
      if (STEP >= 1 && STEP < 3 && d + 1 == STEP && chunk == 0 && tid == 0) {
        ws.found[2 * d] = top;
        ws.found[2 * d + 1] = left;
      }
    }
  }
  if (STEP >= 0 && STEP < 3) return;

  // ---- what stays, and its places --------------------------------------------------
  // Before this chunk: kept ones that competed above the threshold, and equal ones.
  uint32_t more = 0, equal = 0;
  if (STEP == 3 && chunk > 0 && !all_stay && need > 0) {
    const uint32_t digit[3] = {top >> 21, (top >> 10) & 2047u, top & 1023u};
    uint32_t m = 0, e = 0;
    for (int c = tid; c < chunk; c += kEvictThreads) {
      const uint32_t* const h = ws.counts + (int64_t)c * 3 * kEvictBins;
#pragma unroll
      for (int d = 0; d < 3; ++d) m += digit[d] + 1 < kEvictBins ? h[d * kEvictBins + digit[d] + 1] : 0;
      e += h[2 * kEvictBins + digit[2]] - h[2 * kEvictBins + digit[2] + 1];
    }
    block_scan(m, sh, 1, &more);
    block_scan(e, sh, 0, &equal);
  }
  if (!all_stay && chunk > 0) more += (uint32_t)min(a.sink, base);  // (the first ones, all before it)
  if (all_stay) more = (uint32_t)base;
  // (the last ones of chunks before this one stay as well)
  if (!all_stay && base > mid1) more += (uint32_t)(base - mid1);

  const auto sure = [&](int i) { return key[i] > top || key[i] == kEvictStays; };
  uint32_t* const count = hist;  // of a wave's turn: staying for certain, equal << 16
#pragma unroll
  for (int i = 0; i < PER; ++i) asm volatile("" ::"v"(w[i]));  // read, before another wave writes there in place
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t c = (uint32_t)__popcll(__ballot(sure(i))) | (uint32_t)__popcll(__ballot(key[i] == top)) << 16;
    if (lane == 0) count[i * kEvictWaves + wave] = c;
  }
  __syncthreads();
  // running counts over turns and waves
  static_assert(PER * kEvictWaves <= kEvictThreads && kChunk < 65536, "one thread a count, of 16 bits");
  {
    uint32_t all;
    const uint32_t s = block_scan(tid < PER * kEvictWaves ? count[tid] : 0, sh, 1, &all);
    if (tid < PER * kEvictWaves) count[tid] = s;
    __syncthreads();
  }
  const int64_t freed0 = (int64_t)sh.sum;
  int32_t* const freed = a.freed + freed0;
  const uint32_t room = (uint32_t)min(max(a.freed_size - freed0, (int64_t)0), (int64_t)0x7fffffff);
  int32_t* const kept = a.kept + (int64_t)b * a.budget;
  const int stay = min(r.n, a.budget);
  if (chunk == 0 && tid == 0) a.kept_lens[b] = stay;
  const uint32_t mask = (1u << a.page_shift) - 1;
  // lanes of a mask below this one, and n
  const auto below = [](uint64_t m, uint32_t n) {
    return (uint32_t)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, n));
  };
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t p = (uint32_t)at(i);
    const uint32_t c = (uint32_t)__builtin_amdgcn_readfirstlane((int)count[i * kEvictWaves + wave]);
    const uint32_t s = below(__ballot(sure(i)), more + (c & 0xffffu));
    const uint32_t e = below(__ballot(key[i] == top), equal + (c >> 16));
    const uint32_t place = s + min(e, left);  // kept ones before this position
    const uint32_t slot = ((uint32_t)page[i] << a.page_shift) + (p & mask);
    if (sure(i) || (key[i] == top && e < left)) {
      kept[place] = (int32_t)slot;
      if (r.out) r.out[place] = w[i];
    } else if (key[i] != kEvictNone && p - place < room) {
      freed[p - place] = (int32_t)slot;
    }
    if (r.out && (int)p >= stay && (int)p < r.n) r.out[p] = 0.f;
  }
}

// Positions of a block where several share a request. In chunks of 4096 four times as many blocks count as in
// chunks of 16384, and each reads four times as many histograms (the reads grow with the square): 30.1 against 34.0 us
// for one request of 131072 positions, 35.9 / 37.5 for 196608, 36.6 / 38.2 for 200000, 38.8 / 38.2 for 212992,
// 38.7 / 39.2 for 229376, 41.7 / 37.6 for 262144; four requests 33.5 / 35.0, 37.4 / 39.0, 38.3 / 39.9, 40.6 / 40.0,
// 40.5 / 40.9, 43.8 / 39.4. The limit lies where they first meet, by whole chunks of 16384. (It does not look at the number of
// requests: 16 of 131072 positions take 50.0 / 40.7, 16 of 65536 28.4 / 36.3.)
static int evict_per(int64_t most) { return most <= kEvictSmall ? 4 : 16; }

template <int STEP, int PER>
hipError_t launch_evict(const EvictArgs& a, unsigned blocks, hipStream_t stream) {
  hipLaunchKernelGGL((evict_kernel<STEP, PER>), dim3(blocks), dim3(kEvictThreads), 0, stream, a);
  return hipGetLastError();
}

template <int PER>
hipError_t launch_evict_steps(const EvictArgs& a, hipStream_t stream) {
  const unsigned blocks = (unsigned)((int64_t)a.B * a.chunks);
  hipError_t e = launch_evict<0, PER>(a, blocks, stream);
  if (e == hipSuccess) e = launch_evict<1, PER>(a, blocks, stream);
  if (e == hipSuccess) e = launch_evict<2, PER>(a, blocks, stream);
  if (e == hipSuccess) e = launch_evict<3, PER>(a, blocks, stream);
  return e;
}

}  // namespace rolaq

int64_t rolaq_evict_blocks(int64_t B, int64_t most) {
  using namespace rolaq;
  const int64_t chunk = (int64_t)evict_per(most) * kEvictThreads;
  return most <= kEvictOne ? B : B * ((most + chunk - 1) / chunk);
}

int64_t rolaq_evict_ws_bytes(int64_t B, int64_t most) {
  using namespace rolaq;
  if (most <= kEvictOne) return 0;
  const int64_t chunk = (int64_t)evict_per(most) * kEvictThreads, chunks = (most + chunk - 1) / chunk;
  return B * (chunks * (3 * kEvictBins + chunk) + 4) * 4;
}

hipError_t rolaq_launch_evict(const rolaq::EvictArgs& args, hipStream_t stream) {
  using namespace rolaq;
  EvictArgs a = args;
  a.chunks = 1;
  // (where four turns of the threads reach them all: 60 requests of 80 15.3 us with sixteen, 8.8 so)
  if (a.most <= 4 * kEvictThreads) return launch_evict<-1, 4>(a, (unsigned)a.B, stream);
  if (a.most <= kEvictOne) return launch_evict<-1, 16>(a, (unsigned)a.B, stream);
  const int per = evict_per(a.most);
  a.chunks = (int)((a.most + per * kEvictThreads - 1) / (per * kEvictThreads));
  return per == 4 ? launch_evict_steps<4>(a, stream) : launch_evict_steps<16>(a, stream);
}
