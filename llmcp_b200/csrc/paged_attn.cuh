// What the attention kernels over the paged cache share: how a sequence's keys are split, the score's functions, the
// rows of out and of the workspace, the tensor maps.
#pragma once

#include "paged.h"
#include "tc_common.cuh"

namespace llmcp_b200 {

// Sequences are cut into `chunks` pieces of `chunk` keys (the last ones of a short sequence empty); 1: nothing to join.
struct PagedSplit {
  int chunk, chunks;
};
constexpr int kMaxChunks = 512;

PagedSplit paged_rows_split(const PagedKv &kv, const PagedBatch &batch, int rows, int sms);
int paged_rows_tile(const PagedKv &kv, int rows); // keys that a CTA of the few-rows kernel takes at a time
cudaError_t launch_paged_rows(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, const PagedSplit &split, int *status,
                              cudaStream_t stream);

// The kernel for many rows; its workspace holds the parts and, for a 4-bit cache, its rows of 16 bits.
PagedSplit paged_tile_split(const PagedKv &kv, const PagedBatch &batch, int heads, int sms);
size_t paged_tile_workspace(const PagedKv &kv, const PagedBatch &batch, int heads, const PagedSplit &split);
cudaError_t launch_paged_tile(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, const PagedSplit &split, int *status,
                              cudaStream_t stream);

// Joins the chunks of every row.  Workspace of a call: [row][chunk][head_dim] f32 sums, then [row][chunk] (maximum in
// units of log 2, sum of weights), row = token * heads + head.
cudaError_t launch_paged_merge(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, const PagedSplit &split, cudaStream_t stream);

inline size_t paged_parts_bytes(const PagedKv &kv, const PagedBatch &batch, int heads, const PagedSplit &split) {
  return split.chunks == 1 ? 0 : static_cast<size_t>(batch.tokens) * heads * split.chunks * (kv.head_dim + 2) * sizeof(float);
}

// Rows of values (or codes) in boxes of box_rows rows x 64 bf16 dimensions, or a whole row of codes, swizzled.
inline bool paged_value_map(CUtensorMap *map, const PagedKv &kv, int64_t rows, int box_rows) {
  tc::EncodeTiled encode = tc::encode_tiled();
  if (!encode)
    return false;
  const bool q4 = kv.scales != nullptr;
  const cuuint64_t cols = q4 ? kv.head_dim / 2 : kv.head_dim;
  const cuuint64_t dims[2] = {cols, static_cast<cuuint64_t>(rows)}, strides[1] = {q4 ? cols : 2 * cols};
  const cuuint32_t box[2] = {q4 ? static_cast<cuuint32_t>(cols) : 64u, static_cast<cuuint32_t>(box_rows)}, elem[2] = {1, 1};
  const int span = q4 ? kv.head_dim / 2 : 128;
  return encode(map, q4 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, kv.pages, dims, strides, box, elem,
                CU_TENSOR_MAP_INTERLEAVE_NONE,
                span == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : span == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The scales of 16 rows (head_dim bytes) as one row of the map.
inline bool paged_scale_map(CUtensorMap *map, const PagedKv &kv, int64_t rows, int box_rows) {
  tc::EncodeTiled encode = tc::encode_tiled();
  if (!encode)
    return false;
  const cuuint64_t cols = kv.head_dim / 2, dims[2] = {cols, static_cast<cuuint64_t>(rows / 16)}, strides[1] = {2 * cols};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(cols), static_cast<cuuint32_t>(box_rows / 16)}, elem[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, kv.scales, dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// [token][head][dim] rows with strides, in boxes of 64 dimensions x `group` heads x `box_tokens` tokens, swizzled.
inline bool paged_rows_map(CUtensorMap *map, const uint16_t *base, int dim, int heads, int tokens, int64_t head_stride, int64_t token_stride, int group, int box_tokens) {
  tc::EncodeTiled encode = tc::encode_tiled();
  if (!encode)
    return false;
  // the stride of a dimension with one entry is never used, but has to be one
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(2 * (heads > 1 ? head_stride : dim)), static_cast<cuuint64_t>(2 * (tokens > 1 ? token_stride : dim))};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(box_tokens)}, elem[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<uint16_t *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

#ifdef __CUDACC__
// 2^x by the hardware's instruction (relative error about 2^-22; 0 for -infinity).
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// scale * tanh of two values by an odd polynomial, fitted for the smallest largest error: of at most 1 by degree 13 (absolute
// error 4.4e-8), of at most 1/2 by degree 9 (6.3e-9).
template <bool HALF> __device__ __forceinline__ uint64_t tanh_by_fma(uint64_t y, float scale) {
  const uint64_t u = mul2(y, y);
  uint64_t r;
  if constexpr (HALF) {
    r = fma2(u, pair(0.017151297808556672f, 0.017151297808556672f), pair(-0.05299423135979913f, -0.05299423135979913f));
    r = fma2(r, u, pair(0.13324906986917054f, 0.13324906986917054f));
    r = fma2(r, u, pair(-0.333330757952904f, -0.333330757952904f));
    r = fma2(r, u, pair(0.9999999873746263f, 0.9999999873746263f));
  } else {
    r = fma2(u, pair(0.0010531353245070575f, 0.0010531353245070575f), pair(-0.006239815943848765f, -0.006239815943848765f));
    r = fma2(r, u, pair(0.020331109759454728f, 0.020331109759454728f));
    r = fma2(r, u, pair(-0.05347844709285361f, -0.05347844709285361f));
    r = fma2(r, u, pair(0.1332570887576237f, 0.1332570887576237f));
    r = fma2(r, u, pair(-0.33332882758746407f, -0.33332882758746407f));
    r = fma2(r, u, pair(0.9999999563685537f, 0.9999999563685537f));
  }
  return mul2(mul2(y, pair(scale, scale)), r);
}

// cap tanh(x / cap) of two scores in units of log 2.  tanh(y) = 1 - 2 / (1 + e^2y) loses its relative precision next to 0,
// and a cap far above the scores must not show: up to 1/2 the polynomial takes over.
__device__ __forceinline__ float2 capped_log2(uint64_t x, float cap, float over_cap) {
  constexpr float kLog2e = 1.4426950408889634f;
  const uint64_t ratio = mul2(x, pair(over_cap, over_cap));
  const float2 y = halves(ratio), near = halves(tanh_by_fma<true>(ratio, cap * kLog2e));
  auto far = [&](float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + exp2_approx(v * (2.0f * kLog2e))));
    return cap * kLog2e * __fmaf_rn(-2.0f, r, 1.0f);
  };
  return make_float2(fabsf(y.x) <= 0.5f ? near.x : far(y.x), fabsf(y.y) <= 0.5f ? near.y : far(y.y));
}

// x sigmoid(gate) = x h^2 / (1 + h^2), h = 2^(gate log2 e / 2): h^2 leaves f32 at gates below -87, where x times it may still be
// an ordinary number, so x is multiplied twice.  At h = 2^12 and above the quotient is x to 2^-24.  A NaN stays one.
__device__ __forceinline__ float times_sigmoid(float x, float gate) {
  float exponent;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(exponent) : "f"(gate * 0.7213475204444817f), "f"(12.0f));
  const float h = exp2_approx(exponent);
  return __fdividef(x * h * h, __fmaf_rn(h, h, 1.0f));
}

// Eight dimensions of a finished row: times their gate, where there is one, as bf16.
__device__ __forceinline__ void paged_store_row(uint16_t *to, float4 x, float4 y, uint4 gate8, bool gated) {
  float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  if (gated) {
    const uint32_t w[4] = {gate8.x, gate8.y, gate8.z, gate8.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = times_sigmoid(v[i], __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16));
  }
  uint32_t words[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(words[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
  *reinterpret_cast<uint4 *>(to) = make_uint4(words[0], words[1], words[2], words[3]);
}
// Where a row's eight dimensions from d lie in out, and its gate.
template <int D> __device__ __forceinline__ int64_t paged_out_at(const PagedAttention &call, int token, int head, int d) {
  return (static_cast<int64_t>(token) * call.heads + head) * D + d;
}
__device__ __forceinline__ uint4 paged_gate(const PagedAttention &call, int token, int head, int d) {
  return call.gate ? *reinterpret_cast<const uint4 *>(call.gate + token * call.gate_row + head * call.gate_head + d) : make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ float2 *paged_part_sums(const PagedAttention &call, int tokens, int chunks, int head_dim) {
  return reinterpret_cast<float2 *>(static_cast<float *>(call.workspace) + static_cast<int64_t>(tokens) * call.heads * chunks * head_dim);
}

// A chunk's part of a row: eight dimensions of its sum, and (once) its reference and the sum of its weights.
__device__ __forceinline__ void paged_store_part(float *to, float4 x, float4 y) {
  reinterpret_cast<float4 *>(to)[0] = x;
  reinterpret_cast<float4 *>(to)[1] = y;
}
template <int D>
__device__ __forceinline__ void paged_store_sums(const PagedAttention &call, int tokens, int chunks, int chunk, int token, int head, float top, float total) {
  paged_part_sums(call, tokens, chunks, D)[(static_cast<int64_t>(token) * call.heads + head) * chunks + chunk] = make_float2(top, total);
}
#endif

} // namespace llmcp_b200
