// Attention of a ragged batch over the paged key/value cache, the plain form: a warp per (row, query head) walks the
// keys in order with a running maximum and sum.  score = softcap tanh(q k scale / softcap) - slope |p - j| for the key
// j of a row at position p; keys j <= p and j < prefix are seen; a row that sees none gets zeros.

#include "common.cuh"
#include "paged.h"
#include "paged_attn.cuh"

namespace llmcp_b200 {

namespace {

constexpr int kWarps = 4;

template <int E>
__global__ void __launch_bounds__(32 * kWarps)
paged_attention_plain_kernel(PagedKv kv, PagedBatch batch, PagedAttention call, int *__restrict__ status) {
  constexpr int D = 32 * E;
  const int lane = threadIdx.x & 31;
  const int64_t unit = blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5);
  const int t = static_cast<int>(unit / call.heads), h = static_cast<int>(unit % call.heads);
  grid_dependency_sync();
  if (t >= batch.tokens)
    return;
  const int b = paged_owner(batch, t);
  if (b < 0)
    return;
  const PagedSequence s = paged_sequence(batch, kv.page_shift, b, status);
  if (s.count == 0)
    return;
  const int position = s.length - s.count + (t - s.first), g = h / (call.heads / kv.kv_heads);
  float q[E], acc[E];
  for (int i = 0; i < E; ++i) {
    q[i] = bf16_to_f32(call.q[t * call.q_row + h * call.q_head + lane * E + i]);
    acc[i] = 0.0f;
  }
  const int last = min(s.length, max(position + 1, call.prefix ? call.prefix[b] : 0));
  const float slope = call.slopes ? call.slopes[h] : 0.0f;
  float m = -INFINITY, l = 0.0f;
  for (int j = 0; j < last; ++j) {
    float k[2][E];
    for (int which = 0; which < 2; ++which) {
      const int64_t row = paged_row(kv, batch, b, j, which, g);
      if (row < 0 && lane == 0 && status)
        atomicOr(status, kStatusBadBatch);
      for (int i = 0; i < E; ++i) {
        const int d = lane * E + i;
        k[which][i] = row < 0 ? 0.0f
                      : kv.scales ? (static_cast<int>(kv.pages[row * (D / 2) + d / 2] >> (4 * (d & 1)) & 15) - 8) * f16_bits_to_f32(kv.scales[row * (D / 32) + d / 32])
                                  : bf16_to_f32(reinterpret_cast<const uint16_t *>(kv.pages)[row * D + d]);
      }
    }
    float x = 0.0f;
    for (int i = 0; i < E; ++i)
      x = __fmaf_rn(q[i], k[0][i], x);
    for (int o = 16; o > 0; o >>= 1)
      x += __shfl_xor_sync(0xffffffffu, x, o);
    x *= call.scale;
    if (call.softcap > 0.0f)
      x = call.softcap * tanhf(x / call.softcap);
    x -= slope * fabsf(static_cast<float>(position - j));
    const float top = fmaxf(m, x);
    const float keep = expf(m - top), p = expf(x - top);
    l = l * keep + p;
    for (int i = 0; i < E; ++i)
      acc[i] = acc[i] * keep + p * k[1][i];
    m = top;
  }
  for (int i = 0; i < E; ++i) {
    float y = last > 0 ? acc[i] / l : 0.0f;
    if (call.gate)
      y = y / (1.0f + expf(-bf16_to_f32(call.gate[t * call.gate_row + h * call.gate_head + lane * E + i])));
    call.out[(static_cast<int64_t>(t) * call.heads + h) * D + lane * E + i] = f32_to_bf16(y);
  }
}

} // namespace

namespace {

// One CTA per (row, head): groups of head_dim / 4 threads take the chunks in turn.
template <int D>
__global__ void __launch_bounds__(256)
paged_merge_kernel(PagedKv kv, PagedBatch batch, PagedAttention call, PagedSplit split) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ float weights[kMaxChunks];
  __shared__ float tops[8], totals[8];
  __shared__ float4 parts[kGroups][kLanes];
  const int token = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  grid_dependency_sync();
  const int b = paged_owner(batch, token);
  if (b < 0)
    return;
  const PagedSequence s = paged_sequence(batch, kv.page_shift, b, nullptr);
  if (s.count == 0)
    return;
  const int used = max(1, (s.length + split.chunk - 1) / split.chunk);
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
  const int d = tid % kLanes * 4;
  const float *src = static_cast<const float *>(call.workspace) + row * D + d;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int c = tid / kLanes; c < used; c += kGroups) {
    const float4 v = *reinterpret_cast<const float4 *>(src + static_cast<int64_t>(c) * D);
    const float w = weights[c];
    acc.x = __fmaf_rn(v.x, w, acc.x), acc.y = __fmaf_rn(v.y, w, acc.y);
    acc.z = __fmaf_rn(v.z, w, acc.z), acc.w = __fmaf_rn(v.w, w, acc.w);
  }
  parts[tid / kLanes][tid % kLanes] = acc;
  __syncthreads();
  if (tid < kLanes) {
    for (int i = 1; i < kGroups; ++i) {
      const float4 v = parts[i][tid];
      acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
    }
    total = 0.0f;
    for (int w = 0; w < 8; ++w)
      total += totals[w];
    paged_store_out<D>(call, token, head, d, acc, total);
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

// Chunks of whole CTA tiles, so many that every SM gets a few CTAs (sequences shorter than max_kv leave theirs empty).
PagedSplit paged_rows_split(const PagedKv &kv, const PagedBatch &batch, int sms) {
  const int64_t tile = paged_rows_tile(kv), tiles = (batch.max_kv + tile - 1) / tile;
  const int64_t wanted = static_cast<int64_t>(sms) * 6;
  const int64_t each = (tiles * batch.sequences * kv.kv_heads + wanted - 1) / wanted;
  const int64_t most = (tiles + kMaxChunks - 1) / kMaxChunks;
  const int64_t chunk = each > most ? each : most;
  if (chunk >= tiles)
    return PagedSplit{batch.max_kv > 0 ? static_cast<int>(tiles * tile) : 1, 1};
  return PagedSplit{static_cast<int>(chunk * tile), static_cast<int>((tiles + chunk - 1) / chunk)};
}

namespace {
bool few_rows(const PagedKv &kv, const PagedBatch &batch, int heads) {
  return static_cast<int64_t>(batch.max_q) * (heads / kv.kv_heads) <= 16;
}
} // namespace

size_t paged_attention_workspace(const PagedKv &kv, const PagedBatch &batch, int heads, int sms) {
  return few_rows(kv, batch, heads) ? paged_parts_bytes(kv, batch, heads, paged_rows_split(kv, batch, sms)) : 0;
}

cudaError_t launch_paged_attention(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, int *status, int sms,
                                   cudaStream_t stream, int *launches) {
  *launches = 1;
  if (few_rows(kv, batch, call.heads)) {
    const PagedSplit split = paged_rows_split(kv, batch, sms);
    if (cudaError_t e = launch_paged_rows(kv, batch, call, split, status, stream); e != cudaSuccess || split.chunks == 1)
      return e;
    *launches = 2;
    return launch_paged_merge(kv, batch, call, split, stream);
  }
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(batch.tokens) * call.heads + kWarps - 1) / kWarps);
  switch (kv.head_dim) {
  case 64:
    return launch_chained(paged_attention_plain_kernel<2>, dim3(grid), dim3(32 * kWarps), 0, stream, kv, batch, call, status);
  case 128:
    return launch_chained(paged_attention_plain_kernel<4>, dim3(grid), dim3(32 * kWarps), 0, stream, kv, batch, call, status);
  case 256:
    return launch_chained(paged_attention_plain_kernel<8>, dim3(grid), dim3(32 * kWarps), 0, stream, kv, batch, call, status);
  default:
    return cudaErrorInvalidValue;
  }
}

} // namespace llmcp_b200
