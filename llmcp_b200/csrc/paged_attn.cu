// Attention of a ragged batch over the paged key/value cache, the plain form: a warp per (row, query head) walks the
// keys in order with a running maximum and sum.  score = softcap tanh(q k scale / softcap) - slope |p - j| for the key
// j of a row at position p; keys j <= p and j < prefix are seen; a row that sees none gets zeros.

#include "common.cuh"
#include "paged.h"

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

size_t paged_attention_workspace(const PagedKv &, const PagedBatch &, int, int) { return 0; }

cudaError_t launch_paged_attention(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, int *status,
                                   cudaStream_t stream, int *launches) {
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(batch.tokens) * call.heads + kWarps - 1) / kWarps);
  *launches = 1;
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
