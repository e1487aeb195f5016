// A batch over the MX4 cache as its kernels read it on the device.
#pragma once

#include "rolaq_common.h"

namespace rolaq {

// A request's part of the batch.
struct Mx4Request {
  int q0, nq;        // first query, queries (max_q_len at most)
  int past;          // positions before the first query's own (negative: the first ones see nothing)
  int len;           // cached positions
  int list;          // first entry of its page list
};

template <typename Args>
__device__ __forceinline__ Mx4Request mx4_request(const Args& a, int b) {
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

}  // namespace rolaq
