// Attention of a ragged batch over the paged key/value cache: which kernel takes a call, and the joining of a row's
// chunks.  score = softcap tanh(q k scale / softcap) - slope |p - j| for the key
// j of a row at position p; keys j <= p and j < prefix are seen; a row that sees none gets zeros.

#include "common.cuh"
#include "paged.h"
#include "paged_attn.cuh"

namespace llmcp_b200 {

namespace {

// One CTA per (row, head): groups of head_dim / 8 threads take the chunks in turn.
template <int D>
__global__ void __launch_bounds__(256)
paged_merge_kernel(PagedKv kv, PagedBatch batch, PagedAttention call, PagedSplit split) {
  constexpr int kLanes = D / 8, kGroups = 256 / kLanes;
  __shared__ float weights[kMaxChunks];
  __shared__ float tops[8], totals[8];
  __shared__ float4 parts[kGroups][kLanes][2];
  const int token = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dependency_sync();
  const int b = paged_owner(batch, token);
  if (b < 0)
    return;
  const PagedSequence s = paged_sequence(batch, kv.page_shift, b, nullptr);
  if (s.count == 0)
    return;
  const int position = s.length - s.count + (token - s.first);
  const int sees = max(0, min(s.length, max(position + 1, call.prefix ? call.prefix[b] : 0))); // chunks from there on are not written
  const int used = max(1, (sees + split.chunk - 1) / split.chunk);
  const int64_t row = (static_cast<int64_t>(token) * call.heads + head) * split.chunks;
  const float2 *sums = paged_part_sums(call, batch.tokens, split.chunks, D) + row;
  float2 mine[kMaxChunks / 256];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMaxChunks / 256; ++i) {
    mine[i] = tid + 256 * i < used ? sums[tid + 256 * i] : make_float2(-INFINITY, 0.0f);
    top = fmaxf(top, mine[i].x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0)
    tops[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w)
    top = fmaxf(top, tops[w]);
  float total = 0.0f;
#pragma unroll
  for (int i = 0; i < kMaxChunks / 256; ++i) {
    const float weight = mine[i].x == -INFINITY ? 0.0f : exp2_approx(mine[i].x - top);
    weights[tid + 256 * i] = weight;
    total += weight * mine[i].y;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0)
    totals[warp] = total;
  __syncthreads();
  const int d = tid % kLanes * 8;
  const float *src = static_cast<const float *>(call.workspace) + row * D + d;
  float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y = x;
  auto add = [](float4 &to, const float4 &v, float w) {
    to.x = __fmaf_rn(v.x, w, to.x), to.y = __fmaf_rn(v.y, w, to.y), to.z = __fmaf_rn(v.z, w, to.z), to.w = __fmaf_rn(v.w, w, to.w);
  };
#pragma unroll 4
  for (int c = tid / kLanes; c < used; c += kGroups) {
    const float4 *part = reinterpret_cast<const float4 *>(src + static_cast<int64_t>(c) * D);
    add(x, part[0], weights[c]);
    add(y, part[1], weights[c]);
  }
  parts[tid / kLanes][tid % kLanes][0] = x;
  parts[tid / kLanes][tid % kLanes][1] = y;
  __syncthreads();
  if (tid < kLanes) {
    for (int i = 1; i < kGroups; ++i) {
      add(x, parts[i][tid][0], 1.0f);
      add(y, parts[i][tid][1], 1.0f);
    }
    total = 0.0f;
    for (int w = 0; w < 8; ++w)
      total += totals[w];
    const float inv = total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
    paged_store_row(call.out + paged_out_at<D>(call, token, head, d), make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv),
                    make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv), paged_gate(call, token, head, d), call.gate != nullptr);
  }
}

} // namespace

cudaError_t launch_paged_merge(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, const PagedSplit &split, cudaStream_t stream) {
  const dim3 grid(batch.tokens, call.heads);
  switch (kv.head_dim) {
  case 64:
    return launch_chained(paged_merge_kernel<64>, grid, dim3(256), 0, stream, kv, batch, call, split);
  case 128:
    return launch_chained(paged_merge_kernel<128>, grid, dim3(256), 0, stream, kv, batch, call, split);
  default:
    return launch_chained(paged_merge_kernel<256>, grid, dim3(256), 0, stream, kv, batch, call, split);
  }
}

// Chunks of whole CTA tiles.  One sequence: as many as the SMs hold at a time (131001 keys in 4 bits: 53 us with two or
// three per SM, 62 with six).  Several: more and shorter ones, which even out their lengths (64 sequences of 2000 to
// 8000 keys, bf16: 242 us with two per SM, 222 with six, 212 with eight).
PagedSplit paged_rows_split(const PagedKv &kv, const PagedBatch &batch, int rows, int sms) {
  const int64_t tile = paged_rows_tile(kv, rows), tiles = (batch.max_kv + tile - 1) / tile;
  const int64_t wanted = static_cast<int64_t>(sms) * (batch.sequences == 1 ? 3 : 8);
  const int64_t each = (tiles * batch.sequences * kv.kv_heads + wanted - 1) / wanted;
  const int64_t most = (tiles + kMaxChunks - 1) / kMaxChunks;
  const int64_t chunk = each > most ? each : most;
  if (chunk >= tiles)
    return PagedSplit{batch.max_kv > 0 ? static_cast<int>(tiles * tile) : 1, 1};
  return PagedSplit{static_cast<int>(chunk * tile), static_cast<int>((tiles + chunk - 1) / chunk)};
}

namespace {
// Rows that share a key head, if they are few enough for the kernel that is made for them; else 0.
int few_rows(const PagedKv &kv, const PagedBatch &batch, int heads) {
  const int64_t rows = static_cast<int64_t>(batch.max_q) * (heads / kv.kv_heads);
  return rows <= 16 ? static_cast<int>(rows) : 0;
}
} // namespace

size_t paged_attention_workspace(const PagedKv &kv, const PagedBatch &batch, int heads, int sms) {
  if (const int rows = few_rows(kv, batch, heads))
    return paged_parts_bytes(kv, batch, heads, paged_rows_split(kv, batch, rows, sms));
  return paged_tile_workspace(kv, batch, heads, paged_tile_split(kv, batch, heads, sms));
}

cudaError_t launch_paged_attention(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, int *status, int sms,
                                   cudaStream_t stream, int *launches) {
  const int rows = few_rows(kv, batch, call.heads);
  const PagedSplit split = rows ? paged_rows_split(kv, batch, rows, sms) : paged_tile_split(kv, batch, call.heads, sms);
  const cudaError_t e = rows ? launch_paged_rows(kv, batch, call, split, status, stream) : launch_paged_tile(kv, batch, call, split, status, stream);
  *launches = rows || !kv.scales ? 1 : 2;
  if (e != cudaSuccess || split.chunks == 1)
    return e;
  *launches += 1;
  return launch_paged_merge(kv, batch, call, split, stream);
}

} // namespace llmcp_b200
