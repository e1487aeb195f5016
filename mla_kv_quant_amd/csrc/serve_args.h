// Kernel argument blocks of the operators around the caches (rotary positions, the
// expanded attention, accumulated weights, eviction), shared by the host launchers and
// the C ABI layer.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rolaq {

struct RotaryArgs {
  const int64_t* positions;  // [T]
  const uint64_t* turns;     // [dim / 2] turns of a step of one position, times 2^64
  float scale;               // of sines and cosines
  int64_t T;
  int dim, pairs;            // rotary width and half of it
  int H, Hk;                 // heads of x[0] and of x[1]
  const void* x[2];          // elements [T, heads, dim], strides (st, sh), innermost 1
  void* y[2];
  int64_t x_st[2], x_sh[2], y_st[2], y_sh[2];
  // set by the launcher
  int groups;  // threads that share a head's pairs
  int slots;   // heads of a token that threads take side by side
  int tokens;  // tokens of a block
};

struct EvictArgs {
  const float* acc;  // [acc_rows, most or more] accumulated weights, row stride acc_st
  float* acc_out;
  int64_t acc_st, acc_out_st;
  int acc_rows;
  const int64_t* req_idx;  // [B] or null
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  int64_t n_indices;
  int page_shift;
  const int64_t* kv_lens;
  int B, budget, sink, recent;
  int32_t* kept;       // [B, budget]
  int64_t* kept_lens;  // [B]
  int32_t* freed;
  int64_t freed_size;
  uint8_t* ws;
  int64_t most;  // the most positions of a request that take part, at most acc's columns
  int chunks;    // set by the launcher: blocks of a request
};

struct ExpandedArgs {
  const uint16_t* q;  // [T, H, DN + DR] bf16, strides (q_st, q_sh)
  int64_t q_st, q_sh;
  const uint16_t* kv;  // [N, H, DN + DN] bf16 (key | value), strides (kv_st, kv_sh)
  int64_t kv_st, kv_sh;
  const uint16_t* pe;  // [N, DR] bf16, row stride pe_st
  int64_t pe_st;
  const int32_t* qo_indptr;  // [B + 1]
  const int32_t* kv_indptr;  // [B + 1]
  int T, N, B, H, max_q_len;
  float sm_scale;
  int causal;
  uint16_t* out;  // [T, H, DN] bf16, strides (o_st, o_sh)
  int64_t o_st, o_sh;
  float* lse;  // [T, H] or null
  float* ws;   // partials of split keys
  // set by the launcher
  int splits;     // parts of the keys at most
  int blocks;     // row blocks at most
  float partial;  // what a part's partials cost
  int cus;
};

}  // namespace rolaq

enum RolaqType { ROLAQ_BF16 = 0, ROLAQ_FP16 = 1, ROLAQ_FP32 = 2 };

hipError_t rolaq_launch_rotary(const rolaq::RotaryArgs& a, int type, bool interleaved, int num_cus, hipStream_t stream);
int64_t rolaq_evict_blocks(int64_t B, int64_t most);  // of a launch
hipError_t rolaq_launch_evict(const rolaq::EvictArgs& a, hipStream_t stream);
// Bytes of workspace that evict asks for where a request has `most` positions at most.
int64_t rolaq_evict_ws_bytes(int64_t B, int64_t most);
hipError_t rolaq_launch_expanded(const rolaq::ExpandedArgs& a, int DN, int num_cus, hipStream_t stream);
// Bytes of workspace that the expanded attention asks for (0: none).
int64_t rolaq_expanded_ws_bytes(int64_t T, int64_t N, int B, int H, int DN, int max_q_len, int num_cus);
