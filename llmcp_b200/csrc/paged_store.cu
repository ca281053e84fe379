// Append to and read from the paged key/value cache.
//
// Append, per new token and head:  x = q or k row;  n = x / sqrt(mean(x^2) + eps) * (1 + w) where there is a norm weight;
// rotated pairs (d, d + rot / 2): (a c - b s, b c + a s);  y = n rounded once to bf16.  Queries go to q_out, keys and
// values (as they are) to their page row, in 4 bits as blocks of 32: d = f16(min(max |y| / 7, 65504)),
// code = round(y / d) held to -7 .. 7, 0 where d is 0.
//
// The arithmetic up to y is in f64, so that y is the correctly rounded value: a last-bit difference in f32 would now
// and then move y to its neighbour and, in 4 bits, a code with it.  (bf16 x f32 products are exact in f64.)  The step
// from y to the code needs no more than f32: y has 8 significant bits, d 11 and code + 1/2 at most 4, so y / d is either
// exactly half way between two codes or at least 2^-15 away from it.
//
// Bound by HBM for many tokens and by latency for few.  A warp takes one token's rows of kItems heads, a lane head_dim /
// 32 neighbouring dimensions; the rows of all its heads are requested before the first is worked on.  Partners of a
// rotation lie in the same place of another lane (rot / 2 is a multiple of head_dim / 32) and come by shuffle.

#include "common.cuh"
#include "paged.h"

namespace llmcp_b200 {

namespace {

constexpr int kWarps = 8;

template <int E> struct Row { // E neighbouring bf16 values of a lane, two to a word
  uint32_t w[E / 2];
};

template <int E> __device__ __forceinline__ Row<E> load_row(const uint16_t *p, bool vectors) {
  Row<E> r;
  if (vectors) {
    if constexpr (E == 8) {
      const uint4 x = *reinterpret_cast<const uint4 *>(p);
      r.w[0] = x.x, r.w[1] = x.y, r.w[2] = x.z, r.w[3] = x.w;
    } else if constexpr (E == 4) {
      const uint2 x = *reinterpret_cast<const uint2 *>(p);
      r.w[0] = x.x, r.w[1] = x.y;
    } else {
      r.w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
  } else {
#pragma unroll
    for (int i = 0; i < E / 2; ++i)
      r.w[i] = p[2 * i] | static_cast<uint32_t>(p[2 * i + 1]) << 16;
  }
  return r;
}

template <int E> __device__ __forceinline__ void store_row(uint16_t *p, const Row<E> &r) {
  if constexpr (E == 8)
    *reinterpret_cast<uint4 *>(p) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
  else if constexpr (E == 4)
    *reinterpret_cast<uint2 *>(p) = make_uint2(r.w[0], r.w[1]);
  else
    *reinterpret_cast<uint32_t *>(p) = r.w[0];
}

// f64 -> bf16 in one rounding: truncate to f32, keep "something was cut off" in the last bit, round that to bf16.
__device__ __forceinline__ uint32_t f64_to_bf16(double x) {
  float f = __double2float_rz(x);
  if (static_cast<double>(f) != x)
    f = __uint_as_float(__float_as_uint(f) | 1u);
  return f32_to_bf16(f);
}

// Eight (four, two) values of this lane to codes and their block's scale; 32 / E lanes share a block.
template <int E> __device__ __forceinline__ uint32_t quantise(const Row<E> &r, int lane, uint16_t *scale) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < E / 2; ++i)
    top = max(top, max(r.w[i] & 0x7fffu, r.w[i] >> 16 & 0x7fffu));
#pragma unroll
  for (int o = 1; o < 32 / E; o <<= 1)
    top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  uint16_t d16;
  float d = fminf(__fdiv_rn(__uint_as_float(top << 16), 7.0f), 65504.0f);
  if (top > 0x7f80u)
    d = __uint_as_float(0x7fffffffu); // a NaN among the values makes the block NaN
  asm("cvt.rn.f16.f32 %0, %1;" : "=h"(d16) : "f"(d));
  *scale = d16;
  d = f16_bits_to_f32(d16);
  const float inv = __fdiv_rn(1.0f, d);
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float y = __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
    float z = __fmul_rn(y, inv);
    // the product is within 2^-22 of the quotient: only next to a middle does the quotient itself decide
    if (fabsf(fabsf(z - rintf(z)) - 0.5f) < 1e-4f)
      z = __fdiv_rn(y, d);
    const int code = d > 0.0f ? max(-7, min(7, __float2int_rn(z))) : 0;
    codes |= static_cast<uint32_t>(code + 8) << (4 * i);
  }
  return codes;
}

template <int E> __device__ __forceinline__ void store_cached(const PagedKv &kv, int64_t row, const Row<E> &r, int lane) {
  if (!kv.scales) {
    store_row<E>(reinterpret_cast<uint16_t *>(kv.pages) + row * (32 * E) + lane * E, r);
    return;
  }
  uint16_t scale;
  const uint32_t codes = quantise<E>(r, lane, &scale);
  uint8_t *dst = kv.pages + row * (16 * E) + lane * (E / 2);
  if constexpr (E == 8)
    *reinterpret_cast<uint32_t *>(dst) = codes;
  else if constexpr (E == 4)
    *reinterpret_cast<uint16_t *>(dst) = static_cast<uint16_t>(codes);
  else
    *dst = static_cast<uint8_t>(codes);
  if (lane % (32 / E) == 0)
    kv.scales[row * E + lane / (32 / E)] = scale;
}

template <int E, int ITEMS>
__global__ void __launch_bounds__(32 * kWarps)
paged_append_kernel(PagedKv kv, PagedBatch batch, PagedAppend call, int vectors, int *__restrict__ status) {
  constexpr int D = 32 * E;
  const int lane = threadIdx.x & 31;
  const int items = call.heads + 2 * kv.kv_heads, groups = (items + ITEMS - 1) / ITEMS;
  const int64_t unit = blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5);
  const int t = static_cast<int>(unit / groups), item0 = static_cast<int>(unit % groups) * ITEMS;
  grid_dependency_sync();
  if (t >= batch.tokens)
    return;

  // requested first: these do not depend on whose token it is
  Row<E> rows[ITEMS];
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const int item = item0 + u;
    if (item < call.heads)
      rows[u] = load_row<E>(call.q + t * call.q_row + item * call.q_head + lane * E, vectors & 1);
    else if (item < call.heads + kv.kv_heads)
      rows[u] = load_row<E>(call.k + t * call.k_row + (item - call.heads) * call.k_head + lane * E, vectors & 2);
    else if (item < items)
      rows[u] = load_row<E>(call.v + t * call.v_row + (item - call.heads - kv.kv_heads) * call.v_head + lane * E, vectors & 4);
  }
  const int b = paged_owner(batch, t);
  if (b < 0)
    return; // behind the last sequence
  const PagedSequence s = paged_sequence(batch, kv.page_shift, b, status);
  const int position = s.length - s.count + (t - s.first);
  if (s.count == 0)
    return;
  if (position < 0 || (call.rot > 0 && position >= call.cos_rows)) {
    if (lane == 0 && status)
      atomicOr(status, kStatusBadBatch);
    return;
  }
  const int lanes_apart = call.rot / 2 / E;
  float c[E], n[E];
  if (lane < 2 * lanes_apart) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      c[i] = call.cos[static_cast<int64_t>(position) * call.rot + lane * E + i];
      n[i] = call.sin[static_cast<int64_t>(position) * call.rot + lane * E + i];
    }
  }
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    const int item = item0 + u;
    if (item >= items)
      break;
    const bool is_q = item < call.heads, is_v = item >= call.heads + kv.kv_heads;
    if (!is_v) {
      const uint16_t *weight = is_q ? call.q_norm : call.k_norm;
      double x[E];
#pragma unroll
      for (int i = 0; i < E; ++i)
        x[i] = __uint_as_float(i & 1 ? rows[u].w[i / 2] & 0xffff0000u : rows[u].w[i / 2] << 16);
      if (weight) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < E; ++i)
          sum += x[i] * x[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
          sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const double inv = 1.0 / sqrt(sum * (1.0 / D) + static_cast<double>(call.eps));
#pragma unroll
        for (int i = 0; i < E; ++i)
          x[i] = x[i] * inv * (1.0 + static_cast<double>(bf16_to_f32(weight[lane * E + i])));
      }
      if (lanes_apart > 0) {
        const int partner = lane < lanes_apart ? lane + lanes_apart : lane - lanes_apart;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const double other = __shfl_sync(0xffffffffu, x[i], partner & 31);
          if (lane < lanes_apart)
            x[i] = x[i] * static_cast<double>(c[i]) - other * static_cast<double>(n[i]);
          else if (lane < 2 * lanes_apart)
            x[i] = x[i] * static_cast<double>(c[i]) + other * static_cast<double>(n[i]);
        }
      }
      if (weight || lane < 2 * lanes_apart) { // else the row is what it was
#pragma unroll
        for (int i = 0; i < E / 2; ++i)
          rows[u].w[i] = f64_to_bf16(x[2 * i]) | f64_to_bf16(x[2 * i + 1]) << 16;
      }
    }
    if (is_q) {
      store_row<E>(call.q_out + (static_cast<int64_t>(t) * call.heads + item) * D + lane * E, rows[u]);
    } else {
      const int g = is_v ? item - call.heads - kv.kv_heads : item - call.heads;
      const int64_t row = paged_row(kv, batch, b, position, is_v, g);
      if (row >= 0)
        store_cached<E>(kv, row, rows[u], lane);
      else if (lane == 0 && status)
        atomicOr(status, kStatusBadBatch);
    }
  }
}

// A warp takes one token's keys and values of ITEMS / 2 heads.
template <int E, int ITEMS, bool F32>
__global__ void __launch_bounds__(32 * kWarps)
paged_read_kernel(PagedKv kv, PagedBatch batch, void *__restrict__ k_out, void *__restrict__ v_out, int *__restrict__ status) {
  constexpr int D = 32 * E;
  const int lane = threadIdx.x & 31;
  const int items = 2 * kv.kv_heads, groups = (items + ITEMS - 1) / ITEMS;
  const int64_t unit = blockIdx.x * static_cast<int64_t>(kWarps) + (threadIdx.x >> 5);
  const int t = static_cast<int>(unit / groups), item0 = static_cast<int>(unit % groups) * ITEMS;
  grid_dependency_sync();
  if (t >= batch.tokens)
    return;
  const int b = paged_owner(batch, t);
  if (b < 0)
    return;
  const PagedSequence s = paged_sequence(batch, kv.page_shift, b, status);
  if (s.count == 0)
    return;
  const int position = s.length - s.count + (t - s.first);
  const int64_t first = position < 0 ? -1 : paged_row(kv, batch, b, position, 0, 0);
  if (first < 0) {
    if (lane == 0 && status)
      atomicOr(status, kStatusBadBatch);
    return;
  }
  Row<E> rows[ITEMS];
  uint32_t codes[ITEMS];
  uint16_t scales[ITEMS];
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    if (item0 + u >= items)
      break;
    const int64_t row = first + (static_cast<int64_t>(item0 + u) << kv.page_shift);
    if (!kv.scales) {
      rows[u] = load_row<E>(reinterpret_cast<const uint16_t *>(kv.pages) + row * D + lane * E, true);
    } else {
      const uint8_t *src = kv.pages + row * (D / 2) + lane * (E / 2);
      codes[u] = E == 8 ? *reinterpret_cast<const uint32_t *>(src) : E == 4 ? *reinterpret_cast<const uint16_t *>(src) : *src;
      scales[u] = kv.scales[row * E + lane / (32 / E)];
    }
  }
#pragma unroll
  for (int u = 0; u < ITEMS; ++u) {
    if (item0 + u >= items)
      break;
    const bool is_v = item0 + u >= kv.kv_heads;
    const int g = item0 + u - (is_v ? kv.kv_heads : 0);
    const int64_t at = (static_cast<int64_t>(t) * kv.kv_heads + g) * D + lane * E;
    float f[E];
#pragma unroll
    for (int i = 0; i < E; ++i)
      f[i] = kv.scales ? __fmul_rn(static_cast<float>(static_cast<int>(codes[u] >> (4 * i) & 15) - 8), f16_bits_to_f32(scales[u]))
                       : __uint_as_float(i & 1 ? rows[u].w[i / 2] & 0xffff0000u : rows[u].w[i / 2] << 16);
    if (F32) {
      float *dst = static_cast<float *>(is_v ? v_out : k_out) + at;
      if constexpr (E == 2) {
        *reinterpret_cast<float2 *>(dst) = make_float2(f[0], f[1]);
      } else {
#pragma unroll
        for (int i = 0; i < E; i += 4)
          *reinterpret_cast<float4 *>(dst + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
      }
    } else {
      if (kv.scales) {
#pragma unroll
        for (int i = 0; i < E / 2; ++i)
          rows[u].w[i] = f32x2_to_bf16x2_hw(f[2 * i], f[2 * i + 1]);
      }
      store_row<E>(static_cast<uint16_t *>(is_v ? v_out : k_out) + at, rows[u]);
    }
  }
}

bool aligned(const void *p, int64_t stride0, int64_t stride1, int elements) {
  return reinterpret_cast<uintptr_t>(p) % (2 * elements) == 0 && stride0 % elements == 0 && stride1 % elements == 0;
}

// Rows of several heads per warp once there are warps enough to fill the GPU four times over (148 x 64 at a time).
bool many(int64_t rows) { return rows >= 4 * 148 * 64; }

unsigned blocks(int64_t tokens, int items, int per_warp) {
  return static_cast<unsigned>((tokens * ((items + per_warp - 1) / per_warp) + kWarps - 1) / kWarps);
}

template <int E>
cudaError_t append(const PagedKv &kv, const PagedBatch &batch, const PagedAppend &call, int *status, cudaStream_t stream) {
  const int vectors = (aligned(call.q, call.q_row, call.q_head, E) ? 1 : 0) | (aligned(call.k, call.k_row, call.k_head, E) ? 2 : 0) |
                      (aligned(call.v, call.v_row, call.v_head, E) ? 4 : 0);
  const int items = call.heads + 2 * kv.kv_heads;
  if (many(static_cast<int64_t>(batch.tokens) * items))
    return launch_chained(paged_append_kernel<E, 4>, dim3(blocks(batch.tokens, items, 4)), dim3(32 * kWarps), 0, stream, kv, batch, call,
                          vectors, status);
  return launch_chained(paged_append_kernel<E, 1>, dim3(blocks(batch.tokens, items, 1)), dim3(32 * kWarps), 0, stream, kv, batch, call,
                        vectors, status);
}

template <int E, bool F32>
cudaError_t read(const PagedKv &kv, const PagedBatch &batch, void *k_out, void *v_out, int *status, cudaStream_t stream) {
  const int items = 2 * kv.kv_heads;
  if (many(static_cast<int64_t>(batch.tokens) * items))
    return launch_chained(paged_read_kernel<E, 4, F32>, dim3(blocks(batch.tokens, items, 4)), dim3(32 * kWarps), 0, stream, kv, batch, k_out,
                          v_out, status);
  return launch_chained(paged_read_kernel<E, 1, F32>, dim3(blocks(batch.tokens, items, 1)), dim3(32 * kWarps), 0, stream, kv, batch, k_out,
                        v_out, status);
}

} // namespace

cudaError_t launch_paged_append(const PagedKv &kv, const PagedBatch &batch, const PagedAppend &call, int *status, cudaStream_t stream) {
  switch (kv.head_dim) {
  case 64:
    return append<2>(kv, batch, call, status, stream);
  case 128:
    return append<4>(kv, batch, call, status, stream);
  case 256:
    return append<8>(kv, batch, call, status, stream);
  default:
    return cudaErrorInvalidValue;
  }
}

cudaError_t launch_paged_read(const PagedKv &kv, const PagedBatch &batch, void *k_out, void *v_out, int out_dtype, int *status,
                              cudaStream_t stream) {
  const bool f32 = out_dtype == kF32;
  switch (kv.head_dim) {
  case 64:
    return f32 ? read<2, true>(kv, batch, k_out, v_out, status, stream) : read<2, false>(kv, batch, k_out, v_out, status, stream);
  case 128:
    return f32 ? read<4, true>(kv, batch, k_out, v_out, status, stream) : read<4, false>(kv, batch, k_out, v_out, status, stream);
  case 256:
    return f32 ? read<8, true>(kv, batch, k_out, v_out, status, stream) : read<8, false>(kv, batch, k_out, v_out, status, stream);
  default:
    return cudaErrorInvalidValue;
  }
}

} // namespace llmcp_b200
