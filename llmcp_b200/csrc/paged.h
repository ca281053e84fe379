// The paged key/value cache: what its kernels share (paged_store.cu: append and read; paged_attn.cu: attention).
//
// Pages   [num_pages][2: keys, values][kv_heads][page_size][head_dim]; bf16, or 4 bits: two codes to a byte (even
//         dimension in the low half, code + 8, codes -7 .. 7) beside f16 scales [...][page_size][head_dim / 32].
// Batch   rows q_start[b] .. q_start[b + 1] - 1 of a call are the last tokens of sequence b's kv_len[b]; token j of
//         sequence b lies in page page_table[b][j / page_size].
// A page index or a length that does not fit is never followed: the rows concerned are left out and status bit
// kStatusBadBatch is raised.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace llmcp_b200 {

constexpr int kStatusWaitRanOut = 1; // as in the other kernels with bounded waits
constexpr int kStatusBadBatch = 4;

struct PagedKv {
  uint8_t *pages;
  uint16_t *scales; // null: bf16 pages
  int64_t num_pages;
  int page_shift; // page_size = 1 << page_shift
  int kv_heads, head_dim;
};

struct PagedBatch {
  const int32_t *q_start, *kv_len, *page_table;
  int64_t table_stride;
  int sequences, table_width;
  int tokens, max_q, max_kv;
};

struct PagedAppend {
  const uint16_t *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head; // strides in elements
  const uint16_t *q_norm, *k_norm;                     // null: no normalisation
  float eps;
  const float *cos, *sin; // [cos_rows][rot]
  int64_t cos_rows;
  int heads, rot;
  uint16_t *q_out; // [tokens][heads][head_dim]
};

struct PagedAttention {
  const uint16_t *q; // [tokens][heads][head_dim] with strides
  int64_t q_row, q_head;
  int heads;
  float scale, softcap; // softcap 0: none
  const float *slopes;  // [heads] or null
  const int32_t *prefix; // [sequences] or null
  const uint16_t *gate; // or null
  int64_t gate_row, gate_head;
  uint16_t *out; // [tokens][heads][head_dim]
  void *workspace;
};

cudaError_t launch_paged_append(const PagedKv &kv, const PagedBatch &batch, const PagedAppend &call, int *status, int sms, cudaStream_t stream);
cudaError_t launch_paged_read(const PagedKv &kv, const PagedBatch &batch, void *k_out, void *v_out, int out_dtype, int *status, int sms,
                              cudaStream_t stream);
cudaError_t launch_paged_attention(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, int *status, int sms,
                                   cudaStream_t stream, int *launches);
size_t paged_attention_workspace(const PagedKv &kv, const PagedBatch &batch, int heads, int sms);

// ---- device side -----------------------------------------------------------------------------------------------------

#ifdef __CUDACC__
// Two f32 values in one register pair.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// One sequence of a batch as a kernel uses it: its rows and its length, or count = 0 where they do not fit together.
struct PagedSequence {
  int first, count; // rows of the call
  int length;       // keys, those rows' among them
};

__device__ __forceinline__ PagedSequence paged_sequence(const PagedBatch &batch, int page_shift, int b, int *status) {
  PagedSequence s;
  s.first = batch.q_start[b];
  const int end = batch.q_start[b + 1];
  s.count = end - s.first;
  s.length = batch.kv_len[b];
  const int64_t room = static_cast<int64_t>(batch.table_width) << page_shift;
  if (s.first < 0 || end < s.first || end > batch.tokens || s.count > batch.max_q || s.length < 0 || s.length > batch.max_kv ||
      s.length > room) {
    if (status)
      atomicOr(status, kStatusBadBatch);
    s.count = 0;
    s.length = 0;
  }
  return s;
}

// The sequence that owns row t, or -1.  One token of every sequence is the common case and needs no search.
__device__ __forceinline__ int paged_owner(const PagedBatch &batch, int t) {
  if (t < batch.sequences && batch.q_start[t] == t && batch.q_start[t + 1] == t + 1)
    return t;
  int low = 0, high = batch.sequences; // the last b with q_start[b] <= t
  while (high - low > 1) {
    const int middle = (low + high) >> 1;
    if (batch.q_start[middle] <= t)
      low = middle;
    else
      high = middle;
  }
  return batch.q_start[low] <= t && t < batch.q_start[low + 1] ? low : -1;
}

// Row (in units of one head's row of head_dim values) of token `position` of sequence b, for keys (0) or values (1) of
// kv head g; -1 where the page does not exist.
__device__ __forceinline__ int64_t paged_row(const PagedKv &kv, const PagedBatch &batch, int b, int position, int which, int g) {
  const int page = batch.page_table[b * batch.table_stride + (position >> kv.page_shift)];
  if (page < 0 || page >= kv.num_pages)
    return -1;
  return (((static_cast<int64_t>(page) * 2 + which) * kv.kv_heads + g) << kv.page_shift) + (position & ((1 << kv.page_shift) - 1));
}
#endif

} // namespace llmcp_b200
