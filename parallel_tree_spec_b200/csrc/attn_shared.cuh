// Tree attention for requests that share leading pages: what its kernels have in
// common (attn_shared.cu: any type and shape; attn_prefix.cu: bf16 tensor cores).
//
// The requests group_indptr[g] .. group_indptr[g+1] form group g; the first
// shared_pages[g] pages of each are the same pages.  A softmax row over the union
// of two column sets is joined from the two sets' parts: with
//   m = max s_j,  l = sum e^(s_j - m),  O = sum e^(s_j - m) v_j
// of each set, M = max(m1, m2), L = l1 e^(m1-M) + l2 e^(m2-M) and likewise O.  So
// the shared columns are one piece of work for all rows of a group, read once,
// and each request's own columns another.
#pragma once

#include "common.cuh"

namespace pts {

// n / d by multiplication: exact for n * d < 2^32 (the launcher checks its n).
struct FastDiv {
  uint32_t d, m;           // m = ceil(2^32 / d)
  __host__ __device__ __forceinline__ FastDiv() {}
  __host__ explicit FastDiv(uint32_t divisor)
      : d(divisor), m(divisor > 1 ? (uint32_t)((0x100000000ull + divisor - 1) / divisor) : 0u) {}
  __device__ __forceinline__ int div(int n) const { return d == 1 ? n : (int)__umulhi((uint32_t)n, m); }
};

struct SharedAttnParams {
  const void* q;
  const void* kv;
  const int32_t* qo_indptr;
  const int32_t* page_indptr;
  const int32_t* page_indices;
  const int32_t* last_page_len;
  const uint64_t* mask_bits;
  int mask_words;
  void* out;
  const int32_t* group_indptr;
  const int32_t* shared_pages;
  int batch, groups;
  int Hq, Hkv, g, D, page_len, max_pages;
  float scale;             // of the scores
};

// Tokens of request b's cache and, of those, the ones before its query rows.
__device__ __forceinline__ int kv_tokens(const SharedAttnParams& p, int b) {
  const int n = p.page_indptr[b + 1] - p.page_indptr[b];
  return n > 0 ? (n - 1) * p.page_len + min(max(p.last_page_len[b], 0), p.page_len) : 0;
}

// The requests of group gi, within the batch whatever group_indptr holds.
__device__ __forceinline__ int2 group_requests(const SharedAttnParams& p, int gi) {
  const int b0 = min(max(p.group_indptr[gi], 0), p.batch);
  return make_int2(b0, min(max(p.group_indptr[gi + 1], b0), p.batch));
}

// The pages of group gi that its rows attend together: shared_pages[gi], but none
// that holds a query row's own token or lies past a member's table.  A whole warp
// calls it; every lane returns the result.  `lead` (nullable) receives the group's first
// request with rows, or the one past its last.
__device__ __forceinline__ int group_shared_pages(const SharedAttnParams& p, int gi, int* lead = nullptr) {
  const int lane = threadIdx.x & 31;
  const int2 range = group_requests(p, gi);
  const int b0 = range.x, b1 = range.y;
  int s = p.shared_pages[gi], first = b1;
#pragma unroll 4
  for (int b = b0 + lane; b < b1; b += 32) {
    const int n = p.qo_indptr[b + 1] - p.qo_indptr[b], before = kv_tokens(p, b) - n;
    if (n > 0) {                                        // no rows: nothing to attend
      s = min(s, before > 0 ? before / p.page_len : 0);
      first = min(first, b);
    }
  }
  if (lead) *lead = __reduce_min_sync(0xffffffffu, first);
  return max(0, __reduce_min_sync(0xffffffffu, s));
}

// The group that holds request b.
__device__ __forceinline__ int group_of(const SharedAttnParams& p, int b) {
  int lo = 0, hi = p.groups;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.group_indptr[mid] <= b) lo = mid;
    else hi = mid;
  }
  return lo;
}

// attn_prefix.cu: bf16, head_dim 64 or 128, pages of whole 16-token runs.
bool prefix_attn_supports(int head_dim, int page_len, int elem_bytes);
size_t prefix_attn_workspace(int batch, int groups, int total_q, int max_qo_len, int max_kv_len, int max_own_len,
                             int Hq, int Hkv, int D);
int prefix_attn_launch(const SharedAttnParams& a, int total_q, int max_qo_len, int max_kv_len, int max_own_len,
                       void* workspace, int32_t* error, cudaStream_t stream);

}  // namespace pts
