// Append to and read from the paged key/value cache.
//
// Append, per new token and head:  x = q or k row;  n = x / sqrt(mean(x^2) + eps) * (1 + w) where there is a norm weight;
// rotated pairs (d, d + rot / 2): (a c - b s, b c + a s);  y = n rounded once to bf16.  Queries go to q_out, keys and
// values (as they are) to their page row, in 4 bits as blocks of 32: d = f16(min(max |y| / 7, 65504)),
// code = round(y / d) held to -7 .. 7, 0 where d is 0.
//
// y is the correctly rounded value: a last-bit difference would now and then move it to its neighbour and, in 4 bits, a
// code with it.  The f32 result is taken where its error bound cannot reach the middle between two bf16 values (the
// rounded ends of its error interval are equal); a row with a value nearer than that is computed again in f64 (bf16 x f32
// products are exact there), one row in ten or so with norms, one in a hundred without.  The step from y to the code needs no more
// than f32: y has 8 significant bits, d 11 and code + 1/2 at most 4, so y / d is either exactly half way between two
// codes or at least 2^-15 away from it, and only next to a middle is the quotient itself formed.
//
// Bound by HBM for many tokens (by instructions with norms in 4 bits) and by latency for few.  A lane takes eight
// neighbouring dimensions (rows of 64 to 256: 8 to 32 lanes).  Partners of a rotation lie in the same place of another lane and come by
// shuffle; where rot / 2 is not a multiple of 8 a lane takes head_dim / 32 dimensions.

#include "common.cuh"
#include "paged.h"

namespace llmcp_b200 {

namespace {

constexpr int kWarps = 4;

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

// Row of kv head 0's key of row t of the call; the other heads' keys, then the values, follow page_size rows apart.  -1 where
// there is none.
__device__ __forceinline__ int64_t cached_row(const PagedKv &kv, const PagedBatch &batch, int t, int *status) {
  const int b = paged_owner(batch, t);
  if (b < 0)
    return -1;
  const PagedSequence s = paged_sequence(batch, kv.page_shift, b, status);
  if (s.count == 0)
    return -1;
  const int position = s.length - s.count + (t - s.first);
  const int64_t row = position < 0 ? -1 : paged_row(kv, batch, b, position, 0, 0);
  if (row < 0 && status)
    atomicOr(status, kStatusBadBatch);
  return row;
}

// This lane's values as f32.
template <int E> __device__ __forceinline__ float value_at(const Row<E> &r, int i) {
  return __uint_as_float(i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
}

// A lane's values to codes and their block's scale; 32 / E lanes share a block.
template <int E> __device__ __forceinline__ uint32_t quantise(const Row<E> &r, uint16_t *scale) {
  uint32_t pair = 0;
#pragma unroll
  for (int i = 0; i < E / 2; ++i)
    pair = __vmaxu2(pair, r.w[i] & 0x7fff7fffu);
#pragma unroll
  for (int o = 1; o < 32 / E; o <<= 1)
    pair = __vmaxu2(pair, __shfl_xor_sync(0xffffffffu, pair, o));
  const uint32_t top = max(pair & 0xffffu, pair >> 16);
  uint16_t d16;
  float d = fminf(__fdiv_rn(__uint_as_float(top << 16), 7.0f), 65504.0f);
  if (top > 0x7f80u)
    d = __uint_as_float(0x7fffffffu); // a NaN among the values makes the block NaN
  asm("cvt.rn.f16.f32 %0, %1;" : "=h"(d16) : "f"(d));
  *scale = d16;
  d = f16_bits_to_f32(d16);
  // products with 1 / d are within 2^-22 of the quotients; blocks of zeros, or of NaN, get the code 0
  const bool some = d > 0.0f;
  const float inv = some ? __fdiv_rn(1.0f, d) : 0.0f;
  constexpr float kRound = 12582912.0f + 8.0f; // added to z: the low bits are z rounded to an even integer, + 8
  uint32_t codes = 0;
  bool near = false;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const float z = some ? fminf(fmaxf(__fmul_rn(value_at(r, i), inv), -7.25f), 7.25f) : 0.0f;
    const float t = z + kRound;
    near |= fabsf(z - (t - kRound)) > 0.4999f;
    codes |= (__float_as_uint(t) & 15u) << (4 * i);
  }
  if (near) {
    codes = 0;
#pragma unroll 1
    for (int i = 0; i < E; ++i) {
      const float z = fminf(fmaxf(__fdiv_rn(__uint_as_float((r.w[i / 2] >> (16 * (i & 1))) << 16), d), -7.0f), 7.0f);
      codes |= (__float_as_uint(z + kRound) & 15u) << (4 * i);
    }
  }
  return codes;
}

template <int D, int E> __device__ __forceinline__ void store_cached(const PagedKv &kv, int64_t row, const Row<E> &r, uint32_t codes, uint16_t scale, int l) {
  if (!kv.scales) {
    store_row<E>(reinterpret_cast<uint16_t *>(kv.pages) + row * D + l * E, r);
    return;
  }
  uint8_t *dst = kv.pages + row * (D / 2) + l * (E / 2);
  if constexpr (E == 8)
    *reinterpret_cast<uint32_t *>(dst) = codes;
  else if constexpr (E == 4)
    *reinterpret_cast<uint16_t *>(dst) = static_cast<uint16_t>(codes);
  else
    *dst = static_cast<uint8_t>(codes);
  if (l % (32 / E) == 0)
    kv.scales[row * (D / 32) + l / (32 / E)] = scale;
}

// A lane's part of one row, normalised (weight) and rotated (cos, sin, sign -1 or +1 for the first or second of a pair, 0:
// not) in f64.  Reads everything again: it is called seldom, and the registers of the f32 path stay few.
template <int D, int E>
__device__ __noinline__ Row<E> rotated_in_f64(const uint16_t *src, const uint16_t *weight, float eps, const float *cos, const float *sin, float sign,
                                              int partner) {
  constexpr int kLanes = D / E;
  double x[E], sum = 0.0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    x[i] = bf16_to_f32(src[i]);
    sum += x[i] * x[i];
  }
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1)
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const double inv = 1.0 / sqrt(sum * (1.0 / D) + static_cast<double>(eps));
  Row<E> r;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (weight)
      x[i] = x[i] * inv * (1.0 + static_cast<double>(bf16_to_f32(weight[i])));
    const double other = __shfl_sync(0xffffffffu, x[i], partner);
    const double y = sign != 0.0f ? x[i] * static_cast<double>(cos[i]) + static_cast<double>(sign) * other * static_cast<double>(sin[i]) : x[i];
    const uint32_t bits = f64_to_bf16(y);
    r.w[i / 2] = i & 1 ? r.w[i / 2] | bits << 16 : bits;
  }
  return r;
}

// A block takes one token (or, for few tokens, some of its heads: blockIdx.y); a warp its heads kRows at a time, the next
// ones requested while these are worked on.
template <int D, int E>
__global__ void __launch_bounds__(32 * kWarps, 6)
paged_append_kernel(PagedKv kv, PagedBatch batch, PagedAppend call, int vectors, int *__restrict__ status) {
  constexpr int kLanes = D / E, kRows = 32 / kLanes; // lanes of a row, rows side by side in a warp
  const int lane = threadIdx.x & 31, l = lane % kLanes, side = lane / kLanes, t = blockIdx.x;
  const int items = call.heads + 2 * kv.kv_heads, step = gridDim.y * kWarps * kRows;
  int front = (blockIdx.y * kWarps + (threadIdx.x >> 5)) * kRows; // of the warp's items
  grid_dependency_sync();
  if (front >= items)
    return;
  const uint16_t *q = call.q + t * call.q_row + l * E, *k = call.k + t * call.k_row + l * E, *v = call.v + t * call.v_row + l * E;
  auto source = [&](int item) { // past the last item the first key, which nobody uses
    const int key = item - call.heads, value = key - kv.kv_heads;
    return key < 0 ? q + item * call.q_head : value < 0 ? k + key * call.k_head : value < kv.kv_heads ? v + value * call.v_head : k;
  };
  const bool dense = (vectors & 7) == 7;
  // requested first: these do not depend on whose token it is
  Row<E> row = load_row<E>(source(front + side), dense);
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
  const int64_t first = paged_row(kv, batch, b, position, 0, 0); // row of kv head 0's key; heads, then values, follow page by page
  if (first < 0 && lane == 0 && status)
    atomicOr(status, kStatusBadBatch);
  const int lanes_apart = call.rot / 2 / E;
  const bool turned = l < 2 * lanes_apart;
  const float sign = turned ? (l < lanes_apart ? -1.0f : 1.0f) : 0.0f;
  const int partner = side * kLanes + (turned ? (l < lanes_apart ? l + lanes_apart : l - lanes_apart) : l);
  // y = x c + other n, with c = 1 and n = 0 where nothing turns
  const float *cs = call.cos + static_cast<int64_t>(position) * call.rot + l * E, *sn = call.sin + static_cast<int64_t>(position) * call.rot + l * E;
  float c[E], n[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    c[i] = 1.0f;
    n[i] = 0.0f;
  }
  if (turned) {
    if (E >= 4 && (vectors & 8)) {
#pragma unroll
      for (int i = 0; i < E / 4; ++i) {
        const float4 v = reinterpret_cast<const float4 *>(cs)[i], w = reinterpret_cast<const float4 *>(sn)[i];
        c[4 * i] = v.x, c[4 * i + 1] = v.y, c[4 * i + 2] = v.z, c[4 * i + 3] = v.w;
        n[4 * i] = w.x, n[4 * i + 1] = w.y, n[4 * i + 2] = w.z, n[4 * i + 3] = w.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        c[i] = cs[i];
        n[i] = sn[i];
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i)
      n[i] *= sign;
  }
  const bool norms = call.q_norm || call.k_norm;
#pragma unroll 1
  for (; front < items; front += step) {
    const int item = front + side;
    Row<E> next = row;
    if (front + step < items)
      next = load_row<E>(source(item + step), dense);
    const bool is_q = item < call.heads, is_v = item >= call.heads + kv.kv_heads;
    const uint16_t *weight = is_v ? nullptr : is_q ? call.q_norm : call.k_norm;
    if (weight)
      weight += l * E;
    if ((norms || call.rot > 0) && front < call.heads + kv.kv_heads) { // the same for the whole warp
      float x[E];
#pragma unroll
      for (int i = 0; i < E; ++i)
        x[i] = value_at(row, i);
      // Error bounds in units of 2^-24.  y = x c + p with p = other n rounded: |p| + |y|, and |y| for the interval's ends.
      // With a norm x and other are off by up to 13 of themselves (sum of squares of exact terms, mean and eps: E + 7, at
      // most 15, half of which is left by the root; rsqrt 2.2; its product, 1 + w and theirs 3), which is
      // 13 (|x c| + |p|) <= 13 (|y| + 2 |p|) more.  The last percent is for the bound's own rounding.
      const float of_p = (weight ? 27.0f : 1.0f) * 1.01f / 16777216.0f, of_y = (weight ? 15.0f : 2.0f) * 1.01f / 16777216.0f;
      if (norms) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i)
          sum = __fmaf_rn(x[i], x[i], sum);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1)
          sum += __shfl_xor_sync(0xffffffffu, sum, o);
        float inv;
        asm("rsqrt.approx.f32 %0, %1;" : "=f"(inv) : "f"(sum * (1.0f / D) + call.eps));
        if (weight) {
          const Row<E> w = load_row<E>(weight, vectors & 16);
#pragma unroll
          for (int i = 0; i < E; ++i)
            x[i] = x[i] * inv * (1.0f + value_at(w, i));
        }
      }
      bool sure = true;
      Row<E> done;
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        float y[2], off[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int e = 2 * i + h;
          const float p = __shfl_sync(0xffffffffu, x[e], partner) * n[e];
          y[h] = __fmaf_rn(x[e], c[e], p);
          off[h] = __fmaf_rn(fabsf(p), of_p, fabsf(y[h]) * of_y);
        }
        done.w[i] = f32x2_to_bf16x2_hw(y[0] + off[0], y[1] + off[1]);
        sure &= done.w[i] == f32x2_to_bf16x2_hw(y[0] - off[0], y[1] - off[1]);
      }
      const bool changed = !is_v && (weight || turned);
      if (__any_sync(0xffffffffu, changed && !sure))
        done = rotated_in_f64<D, E>(source(item), weight, call.eps, cs, sn, is_v ? 0.0f : sign, partner);
      if (changed)
        row = done;
    }
    uint32_t codes = 0;
    uint16_t scale = 0;
    if (kv.scales && front + kRows > call.heads) // some row of the warp is a key or value
      codes = quantise<E>(row, &scale);
    if (is_q)
      store_row<E>(call.q_out + (static_cast<int64_t>(t) * call.heads + item) * D + l * E, row);
    else if (item < items && first >= 0)
      store_cached<D, E>(kv, first + (static_cast<int64_t>(item - call.heads) << kv.page_shift), row, codes, scale, l);
    row = next;
  }
}

// Blocks and warps as above; bf16 pages are copied, head_dim / 32 dimensions per lane.
template <int E, bool F32>
__global__ void __launch_bounds__(32 * kWarps)
paged_read_kernel(PagedKv kv, PagedBatch batch, void *__restrict__ k_out, void *__restrict__ v_out, int *__restrict__ status) {
  constexpr int D = 32 * E, kAhead = 4;
  const int lane = threadIdx.x & 31, t = blockIdx.x, step = gridDim.y * kWarps;
  grid_dependency_sync();
  const int64_t first = cached_row(kv, batch, t, status);
  if (first < 0)
    return;
  const uint16_t *src = reinterpret_cast<const uint16_t *>(kv.pages) + first * D + lane * E;
  const int64_t at = static_cast<int64_t>(t) * kv.kv_heads * D + lane * E;
  for (int item = blockIdx.y * kWarps + (threadIdx.x >> 5); item < 2 * kv.kv_heads; item += kAhead * step) {
    Row<E> rows[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (item + u * step < 2 * kv.kv_heads)
        rows[u] = load_row<E>(src + (static_cast<int64_t>(item + u * step) << kv.page_shift) * D, true);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int head = (item + u * step) % kv.kv_heads;
      if (item + u * step >= 2 * kv.kv_heads)
        break;
      void *out = item + u * step >= kv.kv_heads ? v_out : k_out;
      if constexpr (F32) {
        float *dst = static_cast<float *>(out) + at + head * D;
#pragma unroll
        for (int i = 0; i < E; i += 2)
          *reinterpret_cast<float2 *>(dst + i) = make_float2(value_at(rows[u], i), value_at(rows[u], i + 1));
      } else {
        store_row<E>(static_cast<uint16_t *>(out) + at + head * D, rows[u]);
      }
    }
  }
}

// The same from 4 bits: a lane takes 16 dimensions (8 bytes of codes, 32 or 64 bytes out), rows of several heads lie side
// by side in the warp.
template <int D, bool F32>
__global__ void __launch_bounds__(32 * kWarps)
paged_read_q4_kernel(PagedKv kv, PagedBatch batch, void *__restrict__ k_out, void *__restrict__ v_out, int *__restrict__ status) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes;
  const int lane = threadIdx.x & 31, l = lane % kLanes, t = blockIdx.x;
  grid_dependency_sync();
  const int64_t first = cached_row(kv, batch, t, status);
  if (first < 0)
    return;
  const uint8_t *src = kv.pages + first * (D / 2) + l * 8;
  const uint16_t *scales = kv.scales + first * (D / 32) + l / 2;
  const int64_t at = static_cast<int64_t>(t) * kv.kv_heads * D + l * 16;
  for (int item = (blockIdx.y * kWarps + (threadIdx.x >> 5)) * kRows + lane / kLanes; item < 2 * kv.kv_heads; item += gridDim.y * kWarps * kRows) {
    const int64_t row = static_cast<int64_t>(item) << kv.page_shift;
    const uint2 codes = *reinterpret_cast<const uint2 *>(src + row * (D / 2));
    const float d = f16_bits_to_f32(scales[row * (D / 32)]);
    const bool is_v = item >= kv.kv_heads;
    void *out = is_v ? v_out : k_out;
    const int64_t to = at + (item - (is_v ? kv.kv_heads : 0)) * D;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t w = h ? codes.y : codes.x;
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) { // nibbles i and i + 4 as 1024 + code + 8 in f16, 1032 off again: exact
        uint32_t pair = (w >> (4 * i) & 0x000f000fu) | 0x64006400u;
        asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(pair) : "r"(0x64086408u));
        asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, h; }" : "=f"(f[i]), "=f"(f[i + 4]) : "r"(pair));
        f[i] *= d;
        f[i + 4] *= d;
      }
      if constexpr (F32) {
        float *dst = static_cast<float *>(out) + to + 8 * h;
        *reinterpret_cast<float4 *>(dst) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4 *>(dst + 4) = make_float4(f[4], f[5], f[6], f[7]);
      } else {
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(out) + to + 8 * h) =
            make_uint4(f32x2_to_bf16x2_hw(f[0], f[1]), f32x2_to_bf16x2_hw(f[2], f[3]), f32x2_to_bf16x2_hw(f[4], f[5]), f32x2_to_bf16x2_hw(f[6], f[7]));
      }
    }
  }
}

bool aligned(const void *p, int64_t stride0, int64_t stride1, int elements) {
  return reinterpret_cast<uintptr_t>(p) % (2 * elements) == 0 && stride0 % elements == 0 && stride1 % elements == 0;
}

// A token's heads go to several blocks as long as there are fewer blocks than the SMs take at a time.
dim3 grid(int tokens, int items, int rows) {
  const int all = (items + kWarps * rows - 1) / (kWarps * rows), room = 148 * 8 / tokens;
  return dim3(tokens, room < 1 ? 1 : room < all ? room : all);
}

template <int D, int E>
cudaError_t append(const PagedKv &kv, const PagedBatch &batch, const PagedAppend &call, int *status, cudaStream_t stream) {
  constexpr int kRows = 32 * E / D;
  const bool tables = reinterpret_cast<uintptr_t>(call.cos) % 16 == 0 && reinterpret_cast<uintptr_t>(call.sin) % 16 == 0 && call.rot % 4 == 0;
  const int vectors = (call.heads == 0 || aligned(call.q, call.q_row, call.q_head, E) ? 1 : 0) | (aligned(call.k, call.k_row, call.k_head, E) ? 2 : 0) |
                      (aligned(call.v, call.v_row, call.v_head, E) ? 4 : 0) | (tables ? 8 : 0) |
                      (aligned(call.q_norm, 0, 0, E) && aligned(call.k_norm, 0, 0, E) ? 16 : 0);
  return launch_chained(paged_append_kernel<D, E>, grid(batch.tokens, call.heads + 2 * kv.kv_heads, kRows), dim3(32 * kWarps), 0, stream, kv, batch,
                        call, vectors, status);
}

template <int E, bool F32>
cudaError_t read(const PagedKv &kv, const PagedBatch &batch, void *k_out, void *v_out, int *status, cudaStream_t stream) {
  constexpr int D = 32 * E;
  if (kv.scales)
    return launch_chained(paged_read_q4_kernel<D, F32>, grid(batch.tokens, 2 * kv.kv_heads, 512 / D), dim3(32 * kWarps), 0, stream, kv, batch, k_out,
                          v_out, status);
  return launch_chained(paged_read_kernel<E, F32>, grid(batch.tokens, 2 * kv.kv_heads, 1), dim3(32 * kWarps), 0, stream, kv, batch, k_out, v_out, status);
}

} // namespace

cudaError_t launch_paged_append(const PagedKv &kv, const PagedBatch &batch, const PagedAppend &call, int *status, cudaStream_t stream) {
  const bool eights = call.rot % 16 == 0;
  switch (kv.head_dim) {
  case 64:
    return eights ? append<64, 8>(kv, batch, call, status, stream) : append<64, 2>(kv, batch, call, status, stream);
  case 128:
    return eights ? append<128, 8>(kv, batch, call, status, stream) : append<128, 4>(kv, batch, call, status, stream);
  case 256:
    return append<256, 8>(kv, batch, call, status, stream);
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
