// Kernel argument blocks of the 4-bit (MX4) latent cache, shared by the host
// launchers and the C ABI layer.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rolaq {

// Scale bytes: s stands for 2^(s - 127) in [2^-64, 2^32]; a block that is not
// finite, or too large, has kMx4NaN.
constexpr int kMx4Low = 63, kMx4High = 159, kMx4NaN = 255;
constexpr int kMx4Requests = 1024;  // the most requests whose tiles attend's blocks share out

struct Mx4AttendArgs {
  const uint16_t* q;  // [T, H, D + R] bf16, strides (q_st, q_sh)
  int64_t q_st, q_sh;
  const uint8_t* codes;   // [num_slots, D / 2]
  const uint8_t* scales;  // [num_slots, D / 32]
  const uint16_t* rope;   // [num_slots, R] bf16
  int64_t num_slots;
  const int32_t* qo_indptr;  // [B + 1] query offsets, or null: one query for each request
  const int32_t* kv_indptr;  // [B + 1] page list offsets
  const int32_t* kv_indices;
  int64_t n_indices;
  int page_shift;
  const int64_t* kv_lens;  // [B] cached positions, the queries' own among them
  int T, B, H, max_q_len;
  float sm_scale;
  uint16_t* out;  // [T, H, D] bf16, strides (o_st, o_sh)
  int64_t o_st, o_sh;
  float* lse;   // [T, H] or null
  uint8_t* ws;  // workspace: the merge's jobs and the partials
  // set by the launcher
  int blocks;      // > 0: the batch's tiles shared out over so many blocks; 0: a block for each row block
  int row_blocks;  // row blocks of a request of max_q_len queries
  int h_inv;       // 65536 / H rounded up
  int by_pair;     // the merge's jobs are numbered by (request, row block), not by block
};

struct Mx4WeightsArgs {
  const uint16_t* q;  // as Mx4AttendArgs has them
  int64_t q_st, q_sh;
  const uint8_t* codes;
  const uint8_t* scales;
  const uint16_t* rope;
  int64_t num_slots;
  const int32_t* qo_indptr;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  int64_t n_indices;
  int page_shift;
  const int64_t* kv_lens;
  int T, B, H, max_q_len;
  float sm_scale;
  const float* lse;        // [T, H]
  const int64_t* req_idx;  // [B] or null
  float* acc;              // [acc_rows, acc_cols], row stride acc_st
  int64_t acc_st;
  int acc_rows;
  int64_t acc_cols;
  int add;      // to what acc holds; else in its place
  float* ws;    // room for parts of the rows, or null
  // set by the launcher
  int parts;        // of the rows of every request
  int64_t ws_part;  // entries of ws that a part has
  int cost_shift;   // of the steps over a request's rows, where their sum would pass 32 bits
};

struct Mx4RowsArgs {
  const int64_t* slots;  // [n]
  int64_t n, num_slots;
  const uint16_t* x;  // writer: latent rows [n, D] bf16, row stride xs
  int64_t xs;
  const uint16_t* k_pe;  // writer: rope rows, strides (pe_s0, pe_s1)
  int64_t pe_s0, pe_s1;
  uint8_t* codes;
  uint8_t* scales;
  uint16_t* rope;
  uint16_t* out;  // reader: [n, out_st] bf16, latent (D) then rope (R)
  int64_t out_st;
  const uint16_t* rot;  // reader of rotated rows: R_eff [D, D] row-major, 16-byte aligned
};

}  // namespace rolaq

hipError_t rolaq_launch_mx4_attend(const rolaq::Mx4AttendArgs& a, int D, int num_cus, hipStream_t stream);
hipError_t rolaq_launch_mx4_weights(const rolaq::Mx4WeightsArgs& a, int D, int num_cus, hipStream_t stream);
// Bytes of workspace with which it takes parts of the rows (0: none), `all_rows`, of `rows` a request at most.
int64_t rolaq_mx4_weights_ws_bytes(int64_t n_indices, int page_shift, int B, int64_t all_rows, int64_t rows, int D,
                                   int num_cus);
// Bytes of workspace that attend asks for at width D, whatever the batch.
int64_t rolaq_mx4_attend_ws_bytes(int D, int num_cus);
hipError_t rolaq_launch_mx4_write_plain(const rolaq::Mx4RowsArgs& a, int D, hipStream_t stream);
hipError_t rolaq_launch_mx4_read(const rolaq::Mx4RowsArgs& a, int D, hipStream_t stream);
hipError_t rolaq_launch_mx4_unrotate(const rolaq::Mx4RowsArgs& a, int D, int num_cus, hipStream_t stream);
