// Attention of a ragged batch over the paged key/value cache: which kernel takes a call, and the joining of a row's
// chunks.  score = softcap tanh(q k scale / softcap) - slope |p - j| for the key
// j of a row at position p; keys j <= p and j < prefix are seen; a row that sees none gets zeros.

#include "common.cuh"
#include "paged.h"
#include "paged_attn.cuh"

namespace llmcp_b200 {

namespace {

// One CTA per (row, head) and 64 dimensions: 32 groups of 8 threads take the chunks in turn, so that a row of many chunks
// is not longer on its way than a few of their loads.
template <int D>
__global__ void __launch_bounds__(256)
paged_merge_kernel(PagedKv kv, PagedBatch batch, PagedAttention call, PagedSplit split) {
  __shared__ float weights[kMaxChunks];
  __shared__ float tops[8], totals[8];
  __shared__ float4 parts[8][8][2];
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
  // the first parts are on their way before their weights are known
  const int d = blockIdx.z * 64 + tid % 8 * 8, group = tid / 8;
  const float4 *src = reinterpret_cast<const float4 *>(static_cast<const float *>(call.workspace) + row * D + d);
  constexpr int kAhead = 4;
  float4 first[kAhead][2];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int c = group + 32 * i;
    first[i][0] = first[i][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (c < used) {
      first[i][0] = src[static_cast<int64_t>(c) * (D / 4)];
      first[i][1] = src[static_cast<int64_t>(c) * (D / 4) + 1];
    }
  }
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
  float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](float4 x, float4 y, float w) {
    const float p[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] = __fmaf_rn(p[i], w, v[i]);
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (group + 32 * i < used)
      add(first[i][0], first[i][1], weights[group + 32 * i]);
#pragma unroll 4
  for (int c = group + 32 * kAhead; c < used; c += 32)
    add(src[static_cast<int64_t>(c) * (D / 4)], src[static_cast<int64_t>(c) * (D / 4) + 1], weights[c]);
#pragma unroll
  for (int o = 8; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (lane < 8) {
    parts[warp][lane][0] = make_float4(v[0], v[1], v[2], v[3]);
    parts[warp][lane][1] = make_float4(v[4], v[5], v[6], v[7]);
  }
  __syncthreads();
  if (tid < 8) {
    total = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      total += totals[w];
      if (w > 0)
        add(parts[w][tid][0], parts[w][tid][1], 1.0f);
    }
    const float inv = total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
    paged_store_row(call.out + paged_out_at<D>(call, token, head, d), make_float4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                    make_float4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv), paged_gate(call, token, head, d), call.gate != nullptr);
  }
}

// A warp per (row, head): for rows of at most 32 chunks, of which there are many.
template <int D>
__global__ void __launch_bounds__(256)
paged_merge_few_kernel(PagedKv kv, PagedBatch batch, PagedAttention call, PagedSplit split) {
  constexpr int E = D / 32; // dimensions of a lane
  const int token = blockIdx.x, head = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  grid_dependency_sync();
  if (head >= call.heads)
    return;
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
  const float2 mine = lane < used ? paged_part_sums(call, batch.tokens, split.chunks, D)[row + lane] : make_float2(-INFINITY, 0.0f);
  const float *src = static_cast<const float *>(call.workspace) + row * D + lane * E;
  float top = mine.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float weight = mine.x == -INFINITY ? 0.0f : exp2_approx(mine.x - top);
  float total = weight * mine.y, v[E];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    total += __shfl_xor_sync(0xffffffffu, total, o);
#pragma unroll
  for (int i = 0; i < E; ++i)
    v[i] = 0.0f;
#pragma unroll 4
  for (int c = 0; c < used; ++c) {
    const float w = __shfl_sync(0xffffffffu, weight, c);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 part = *reinterpret_cast<const float2 *>(src + static_cast<int64_t>(c) * D + i);
      v[i] = __fmaf_rn(part.x, w, v[i]);
      v[i + 1] = __fmaf_rn(part.y, w, v[i + 1]);
    }
  }
  const float inv = total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
  const int64_t to = paged_out_at<D>(call, token, head, lane * E);
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    float x = v[i] * inv, y = v[i + 1] * inv;
    if (call.gate) {
      const uint32_t gate = *reinterpret_cast<const uint32_t *>(call.gate + token * call.gate_row + head * call.gate_head + lane * E + i);
      x = times_sigmoid(x, __uint_as_float(gate << 16));
      y = times_sigmoid(y, __uint_as_float(gate & 0xffff0000u));
    }
    *reinterpret_cast<uint32_t *>(call.out + to + i) = f32x2_to_bf16x2_hw(x, y);
  }
}

template <int D>
cudaError_t merge(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, const PagedSplit &split, cudaStream_t stream) {
  // one sequence of 131001 tokens, 103 chunks of 16 rows: 4.0 us less by chunk groups; 96 x 3 rows of 20 heads, 4 chunks: 20 us less by warps
  if (split.chunks <= 32 && static_cast<int64_t>(batch.tokens) * call.heads >= 256)
    return launch_chained(paged_merge_few_kernel<D>, dim3(batch.tokens, (call.heads + 7) / 8), dim3(256), 0, stream, kv, batch, call, split);
  return launch_chained(paged_merge_kernel<D>, dim3(batch.tokens, call.heads, D / 64), dim3(256), 0, stream, kv, batch, call, split);
}

} // namespace

cudaError_t launch_paged_merge(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, const PagedSplit &split, cudaStream_t stream) {
  return kv.head_dim == 64 ? merge<64>(kv, batch, call, split, stream) : kv.head_dim == 128 ? merge<128>(kv, batch, call, split, stream)
                                                                                             : merge<256>(kv, batch, call, split, stream);
}

// Chunks of whole CTA tiles, so many for every SM.  One sequence: as many as an SM holds at a time, 2 over bf16 pages and 3
// over 4 bits (30001 keys in bf16: 27 us with 2, 30 with 4, 38 with 8; 131001 in 4 bits: 44 us with 3, 52 with 4).  A few
// sequences: 2, or 4 over 4 bits (16 of 1000 to 4000 keys in 4 bits: 27 us with 3, 24 with 4, 30 with 6).  So many that
// their key heads alone fill the SMs: 8, which evens out their lengths (64 of 2000 to 8000 keys in bf16: 231 us with 4,
// 217 with 6, 212 with 8, 211 with 12; 96 x 3 rows of 1250 to 5000 in 4 bits: 104, 103, 90, 92).
PagedSplit paged_rows_split(const PagedKv &kv, const PagedBatch &batch, int rows, int sms) {
  const int64_t tile = paged_rows_tile(kv, rows), tiles = (batch.max_kv + tile - 1) / tile;
  const bool q4 = kv.scales != nullptr;
  const int64_t per_sm = batch.sequences == 1 ? (q4 ? 3 : 2) : static_cast<int64_t>(batch.sequences) * kv.kv_heads < sms ? (q4 ? 4 : 2) : 8;
  const int64_t wanted = sms * per_sm;
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
  *launches = rows || !kv.scales || batch.max_kv == 0 ? 1 : 3;
  if (e != cudaSuccess || split.chunks == 1)
    return e;
  *launches += 1;
  return launch_paged_merge(kv, batch, call, split, stream);
}

} // namespace llmcp_b200
