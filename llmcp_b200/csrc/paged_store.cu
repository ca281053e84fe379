// Append to and read from the paged key/value cache.
//
// Append, per new token and head:  x = q or k row;  n = x / sqrt(mean(x^2) + eps) * (1 + w) where there is a norm weight;
// rotated pairs (d, d + rot / 2): (a c - b s, b c + a s);  y = n rounded once to bf16.  Queries go to q_out, keys and
// values (as they are) to their page row, in 4 bits as blocks of 32: d = f16(min(max |y| / 7, 65504)),
// code = round(y / d) held to -7 .. 7, 0 where d is 0.
//
// y is the correctly rounded value: a last-bit difference would now and then move it to its neighbour and, in 4 bits, a
// code with it.  The f32 result is taken where its error bound cannot reach the middle between two bf16 values (the
// rounded ends of its error interval are equal) and nothing leaves f32's normal range; a row with a value for which that
// fails is computed again in f64 (bf16 x f32 products are exact there), one row of 256 in ten or so with norms, one in fifty
// without.  The step from y to the code needs no more than f32: y has 8 significant bits, d 11 and code + 1/2 at most 4, so
// y / d is either exactly half way between two codes or at least 2^-15 away from it, and a quotient with its remainder's
// share added tells the two apart.
//
// Append is bound by instructions (180 for 256 query values, 120 more for 256 values' codes), read by HBM.  In a captured
// graph, 8192 tokens of 32 + 2 x 8 heads of 128: 62 us over bf16 pages, 64 us over 4 bits, of 26 and 28 us that their bytes
// take.  30001 tokens of 4 heads of 256 read from bf16 pages: 40 us, 6.2 TB/s.  One token: 5.5 us.  A warp takes a whole token
// where there are enough of them (a block for each, with four warps that each found sequence, page and angles: 22 % longer,
// and 12 % to read).
// A lane takes eight neighbouring dimensions (rows of 64 to 256: 8 to 32 lanes).  Partners of a rotation lie in the same
// place of another lane and come by shuffle; where rot / 2 is not a multiple of 8 a lane takes head_dim / 32 dimensions.

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

// The two bf16 values of a word.
__device__ __forceinline__ uint64_t unpacked(uint32_t w) { return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// A lane's values to codes and their block's scale; 32 / E lanes share a block.
template <int E> __device__ __forceinline__ uint32_t quantise(const Row<E> &r, uint16_t *scale) {
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < E / 2; ++i)
    largest = __vmaxu2(largest, r.w[i] & 0x7fff7fffu);
#pragma unroll
  for (int o = 1; o < 32 / E; o <<= 1)
    largest = __vmaxu2(largest, __shfl_xor_sync(0xffffffffu, largest, o));
  const uint32_t top = max(largest & 0xffffu, largest >> 16);
  // Scales between the least normal f16 and 32768: top has 8 significant bits and a middle between two f16 values 12, so
  // top / 7 is at least 2^-15 of itself away from every middle and the product rounds as the quotient does; no |y| / d is
  // above 7.01.  The product with the reciprocal is within 2^-22 of y / d; with its remainder's share added (a step of
  // iterative refinement) it is y / d itself where that is half way between two codes.  (A seventh of all blocks has
  // d = top / 7 exactly, and such quotients.)
  float d = __uint_as_float(top << 16) * (1.0f / 7.0f);
  const bool plain = top == 0 || (d >= 0x1p-14f && d < 32768.0f);
  uint16_t d16;
  asm("cvt.rn.f16.f32 %0, %1;" : "=h"(d16) : "f"(d));
  d = f16_bits_to_f32(d16);
  float inv;
  asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(d));
  if (top == 0)
    inv = 0.0f;
  constexpr float kRound = 12582912.0f + 8.0f; // added to z: the low bits are z rounded to an even integer, + 8
  uint32_t codes = 0, high = 0;
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    const uint64_t y = unpacked(r.w[i]), z = mul2(y, pair(inv, inv));
    const float2 t = halves(add2(fma2(fma2(z, pair(-d, -d), y), pair(inv, inv), z), pair(kRound, kRound)));
    codes += (__float_as_uint(t.x) << (8 * i)) + (__float_as_uint(t.y) << (8 * i + 4));
    high += (__float_as_uint(kRound - 8.0f) << (8 * i)) + (__float_as_uint(kRound - 8.0f) << (8 * i + 4)); // a constant
  }
  codes -= high;
  if (!plain) {
    // any other scale; a NaN among the values makes the block NaN, and its codes 0
    d = top > 0x7f80u ? __uint_as_float(0x7fffffffu) : fminf(__fdiv_rn(__uint_as_float(top << 16), 7.0f), 65504.0f);
    asm("cvt.rn.f16.f32 %0, %1;" : "=h"(d16) : "f"(d));
    d = f16_bits_to_f32(d16);
    codes = 0;
    Row<E> left = r;
#pragma unroll 1
    for (int i = 0; i < E; ++i) {
      const float y = __uint_as_float(left.w[0] << 16);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) // moved along, not indexed: that would put every row into local memory
        left.w[j] = __funnelshift_r(left.w[j], j + 1 < E / 2 ? left.w[j + 1] : 0u, 16);
      const float z = d > 0.0f ? fminf(fmaxf(__fdiv_rn(y, d), -7.0f), 7.0f) : 0.0f;
      codes |= (__float_as_uint(z + kRound) & 15u) << (4 * i);
    }
  }
  *scale = d16;
  return codes;
}

// A lane's part of one row, normalised (weight) and rotated (cos, sin, sign -1 or +1 for the first or second of a pair, 0:
// not) in f64.  Reads everything again: it is called seldom, and the registers of the f32 path stay few.
template <int D, int E>
__device__ __noinline__ Row<E> rotated_in_f64(const uint16_t *src, const uint16_t *weight, float eps, const float *cos, const float *sin, float sign,
                                              int partner) {
  constexpr int kLanes = D / E;
  // x / root as the product with the reciprocal and its remainder's share: a quotient that puts y half way between two bf16
  // values has to come out as it is.  (An infinite root has no remainder.)
  double inv = 0.0, back = 0.0;
  if (weight) {
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const double x = bf16_to_f32(src[i]);
      sum += x * x;
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1)
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const double root = sqrt(sum * (1.0 / D) + static_cast<double>(eps));
    inv = 1.0 / root;
    back = root <= 1e300 ? root : 0.0;
  }
  Row<E> r;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    double x = bf16_to_f32(src[i]);
    if (weight) {
      const double quotient = x * inv;
      x = __fma_rn(__fma_rn(-quotient, back, x), inv, quotient) * (1.0 + static_cast<double>(bf16_to_f32(weight[i])));
    }
    const double other = __shfl_sync(0xffffffffu, x, partner);
    const double y = sign != 0.0f ? x * static_cast<double>(cos[i]) + static_cast<double>(sign) * other * static_cast<double>(sin[i]) : x;
    const uint32_t bits = f64_to_bf16(y);
    r.w[i / 2] = i & 1 ? r.w[i / 2] | bits << 16 : bits;
  }
  return r;
}

// A lane's part of a row of the cache, or of a bf16 row.
template <int E, bool kCodes> __device__ __forceinline__ void store_part(const Row<E> &row, bool here, int l, uint8_t *dst, uint16_t *scales) {
  if constexpr (kCodes) {
    uint16_t scale;
    const uint32_t codes = quantise<E>(row, &scale);
    if (!here)
      return;
    if constexpr (E == 8)
      *reinterpret_cast<uint32_t *>(dst) = codes;
    else if constexpr (E == 4)
      *reinterpret_cast<uint16_t *>(dst) = static_cast<uint16_t>(codes);
    else
      *dst = static_cast<uint8_t>(codes);
    if (l % (32 / E) == 0)
      *scales = scale;
  } else {
    if (here)
      store_row<E>(reinterpret_cast<uint16_t *>(dst), row);
  }
}

struct Place { // of a warp's token and of a lane in it
  int l, side;       // the lane's place in its row, the row's in the warp
  int group, step;   // the warp's next kRows heads of the kind at hand; as many such groups further are its next
  float sign;        // -1, +1: first or second of a rotated pair, 0: not rotated
  int to_partner;    // lanes
  bool dense;        // rows by vectors
};

template <int E> struct Turn { // y = (x c + other n) inv: c and n hold cos, +-sin and the weights, 1 and 0 where nothing turns
  uint64_t c[E / 2], n[E / 2];
};

// Coefficients of a lane.
template <int E>
__device__ __forceinline__ Turn<E> turn_of(const Place &place, const float *cs, const float *sn, const uint16_t *weight, int vectors) {
  float c[E], n[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    c[i] = 1.0f;
    n[i] = 0.0f;
  }
  if (place.sign != 0.0f) {
    if (E >= 4 && (vectors & 8)) {
#pragma unroll
      for (int i = 0; i < E / 4; ++i) {
        const float4 f = reinterpret_cast<const float4 *>(cs)[i], g = reinterpret_cast<const float4 *>(sn)[i];
        c[4 * i] = f.x, c[4 * i + 1] = f.y, c[4 * i + 2] = f.z, c[4 * i + 3] = f.w;
        n[4 * i] = g.x, n[4 * i + 1] = g.y, n[4 * i + 2] = g.z, n[4 * i + 3] = g.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        c[i] = cs[i];
        n[i] = sn[i];
      }
    }
  }
  if (weight) {
    const Row<E> w = load_row<E>(weight, vectors & 16), u = load_row<E>(weight + place.to_partner * E, vectors & 16);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      c[i] *= 1.0f + value_at(w, i);
      n[i] *= 1.0f + value_at(u, i);
    }
  }
  Turn<E> r;
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    r.c[i] = pair(c[2 * i], c[2 * i + 1]);
    r.n[i] = pair(place.sign * n[2 * i], place.sign * n[2 * i + 1]);
  }
  return r;
}

__device__ __forceinline__ float least_of(float a, float b, float c) {
  float r;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Whether a lane has a value below 2^-50 or a coefficient below 2^-30 that is not 0.
template <int E> __device__ __forceinline__ bool has_small(const Row<E> &row, const Turn<E> &turn) {
  bool small = false;
#pragma unroll
  for (int i = 0; i < E / 2; ++i) {
    const float2 x = halves(unpacked(row.w[i])), c = halves(turn.c[i]), n = halves(turn.n[i]);
    small |= (x.x != 0.0f && fabsf(x.x) < 0x1p-50f) || (x.y != 0.0f && fabsf(x.y) < 0x1p-50f);
    small |= (c.x != 0.0f && fabsf(c.x) < 0x1p-30f) || (c.y != 0.0f && fabsf(c.y) < 0x1p-30f);
    small |= (n.x != 0.0f && fabsf(n.x) < 0x1p-30f) || (n.y != 0.0f && fabsf(n.y) < 0x1p-30f);
  }
  return small;
}

// A warp's part of the heads of one kind of its token.  row: the first of them, requested before.  kTurns: normalised and
// rotated; kCodes: stored as codes and scales.  Rows that need f64 are left for the end of up to 32 turns: a call inside the
// loop would take its registers from it.
template <int D, int E, bool kTurns, bool kCodes>
__device__ __forceinline__ void store_heads(Place &place, Row<E> row, int heads, const uint16_t *src, int64_t head_stride, uint8_t *dst, int64_t dst_stride,
                                            uint16_t *scales, int64_t scale_stride, bool stored, const uint16_t *weight, float eps,
                                            const float *cs, const float *sn, bool rotates, int vectors) {
  constexpr int kLanes = D / E, kRows = 32 / kLanes;
  const int lane = threadIdx.x & 31, step = place.step * kRows;
  int item = place.group * kRows + place.side;
  src += item * head_stride;
  dst += item * dst_stride;
  if constexpr (kCodes)
    scales += item * scale_stride;
  const int64_t src_step = step * head_stride, dst_step = step * dst_stride, scale_step = step * scale_stride;
  const bool turns = kTurns && (rotates || weight); // the same for the whole warp
  const bool changed = weight || place.sign != 0.0f;
  Turn<E> turn;
  if (turns)
    turn = turn_of<E>(place, cs, sn, weight, vectors);
  while (item - place.side < heads) {
    uint32_t again = 0;
    int turn_no = 0;
#pragma unroll 1
    for (; turn_no < 32 && item - place.side < heads; ++turn_no) {
      bool here = item < heads;
      Row<E> next = {};
      src += src_step;
      item += step;
      if (item < heads)
        next = load_row<E>(src, place.dense);
      if (turns) {
        // Error bounds in units of 2^-24, with p = other n rounded and y = x c + p.  Without a norm |p| + |y|.  With one c
        // and n are off by 2 of themselves, which makes y's 2 |x c| + 3 |p| + |y| <= 5 |p| + 3 |y|; inv is off by 9.7 (sum
        // of squares of exact terms, mean and eps: E + 7, at most 15, half of which is left by the root; rsqrt 2.2) and its
        // product by 1 more.  And |y| for the interval's ends; the last percents are for the bound's own rounding.
        // That holds where nothing leaves f32's normal range: where |p| + |y| is below 2^-100, before or after its product
        // with inv, it has to be because it is 0.
        bool sure = true;
        float inv = 1.0f, of_y = 2.03f / 16777216.0f, p_to_y = 0.51f;
        if (weight) {
          uint64_t squares = mul2(unpacked(row.w[0]), unpacked(row.w[0]));
#pragma unroll
          for (int i = 1; i < E / 2; ++i)
            squares = fma2(unpacked(row.w[i]), unpacked(row.w[i]), squares);
          float sum = halves(squares).x + halves(squares).y;
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1)
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
          asm("rsqrt.approx.f32 %0, %1;" : "=f"(inv) : "f"(sum * (1.0f / D) + eps));
          of_y = inv * (15.0f / 16777216.0f);
          p_to_y = 0.35f;
          // squares that overflow, or vanish beside an eps of 0, are f64's
          sure = sum >= 0x1p-80f && sum <= 0x1p120f;
        }
        Row<E> done;
        float least = INFINITY;
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
          const uint64_t p = mul2(unpacked(__shfl_sync(0xffffffffu, row.w[i], lane + place.to_partner)), turn.n[i]);
          const uint64_t y = fma2(unpacked(row.w[i]), turn.c[i], p), scaled = mul2(y, pair(inv, inv));
          const float2 a = halves(p), z = halves(y);
          const float off_x = __fmaf_rn(fabsf(a.x), p_to_y, fabsf(z.x)), off_y = __fmaf_rn(fabsf(a.y), p_to_y, fabsf(z.y));
          const uint64_t off = pair(off_x, off_y);
          least = least_of(least, off_x, off_y);
          const float2 up = halves(fma2(off, pair(of_y, of_y), scaled)), down = halves(fma2(off, pair(-of_y, -of_y), scaled));
          done.w[i] = f32x2_to_bf16x2_hw(up.x, up.y);
          sure &= done.w[i] == f32x2_to_bf16x2_hw(down.x, down.y);
        }
        const bool in_range = least * fminf(inv, 1.0f) >= 0x1p-100f;
        if (__any_sync(0xffffffffu, changed && !(sure && in_range) && here) &&
            (__any_sync(0xffffffffu, changed && !sure && here) || __any_sync(0xffffffffu, (inv < 0x1p-20f || has_small(row, turn)) && here))) {
          again |= 1u << turn_no;
          here = false;
        }
        if (changed)
          row = done;
      }
      store_part<E, kCodes>(row, stored && here, place.l, dst, scales);
      if constexpr (kCodes)
        scales += scale_step;
      dst += dst_step;
      row = next;
    }
    if constexpr (kTurns) {
      for (; again; again &= again - 1) {
        const int back = turn_no - (__ffs(again) - 1);
        const bool here = item - back * step < heads;
        const uint16_t *from = src - back * src_step - (here ? 0 : place.side * head_stride);
        const Row<E> done = rotated_in_f64<D, E>(from, weight, eps, cs, sn, place.sign, lane + place.to_partner);
        store_part<E, kCodes>(done, stored && here, place.l, dst - back * dst_step, kCodes ? scales - back * scale_step : nullptr);
      }
    }
  }
  place.group = (item - place.side) / kRows - (heads + kRows - 1) / kRows;
}

// `share` warps take one token, 32 / kLanes of its query, then key, then value heads at a time each, and request the next
// ones while they work on these.  Registers: rows of 256 gain more from 80 each (8192 tokens with norms: 6 % longer with 64),
// shorter ones from more warps (9066 tokens of 32 + 2 x 8 heads in 4 bits: 8 % longer with 80).  Either way some 30 words a
// thread are kept in local memory, most of them around the loop and not in it.
template <int D, int E, bool kCodes>
__global__ void __launch_bounds__(32 * kWarps, D == 256 ? 6 : 8)
paged_append_kernel(PagedKv kv, PagedBatch batch, PagedAppend call, int vectors, unsigned share, int *__restrict__ status) {
  constexpr int kLanes = D / E, kRows = 32 / kLanes; // lanes of a row, rows side by side in a warp
  const unsigned warp = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int t = static_cast<int>(warp / share), lane = threadIdx.x & 31;
  grid_dependency_sync();
  if (static_cast<unsigned>(t) >= static_cast<unsigned>(batch.tokens))
    return;
  Place place;
  place.l = lane % kLanes;
  place.side = lane / kLanes;
  place.group = static_cast<int>(warp % share);
  place.step = static_cast<int>(share);
  place.dense = (vectors & 7) == 7;
  const int apart = call.rot / 2 / E;
  place.sign = place.l < 2 * apart ? (place.l < apart ? -1.0f : 1.0f) : 0.0f;
  place.to_partner = place.sign < 0.0f ? apart : place.sign > 0.0f ? -apart : 0;
  const uint16_t *q = call.q + t * call.q_row + place.l * E, *k = call.k + t * call.k_row + place.l * E, *v = call.v + t * call.v_row + place.l * E;
  const int of_q = (call.heads + kRows - 1) / kRows;
  auto request = [&](const uint16_t *src, int64_t stride, int heads) {
    const int item = place.group * kRows + place.side;
    Row<E> r = {};
    if (item < heads)
      r = load_row<E>(src + item * stride, place.dense);
    return r;
  };
  Row<E> row = request(q, call.q_head, call.heads); // requested first: this does not depend on whose token it is
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
  const float *cs = call.cos + static_cast<int64_t>(position) * call.rot + place.l * E, *sn = call.sin + static_cast<int64_t>(position) * call.rot + place.l * E;
  const bool rotates = call.rot > 0;
  if (place.group < of_q)
    store_heads<D, E, true, false>(place, row, call.heads, q, call.q_head,
                                   reinterpret_cast<uint8_t *>(call.q_out + static_cast<int64_t>(t) * call.heads * D + place.l * E), 2 * D, nullptr, 0, true,
                                   call.q_norm ? call.q_norm + place.l * E : nullptr, call.eps, cs, sn, rotates, vectors);
  else
    place.group -= of_q;
  constexpr int kBytes = kCodes ? D / 2 : 2 * D; // of a row
  const int64_t page_rows = static_cast<int64_t>(1) << kv.page_shift;
  uint8_t *dst = kv.pages + first * kBytes + place.l * (kBytes / kLanes);
  uint16_t *scales = kCodes ? kv.scales + first * (D / 32) + place.l / (32 / E) : nullptr;
  const int of_k = (kv.kv_heads + kRows - 1) / kRows;
  if (place.group < of_k) {
    row = request(k, call.k_head, kv.kv_heads);
    store_heads<D, E, true, kCodes>(place, row, kv.kv_heads, k, call.k_head, dst, page_rows * kBytes, scales, page_rows * (D / 32), first >= 0,
                                    call.k_norm ? call.k_norm + place.l * E : nullptr, call.eps, cs, sn, rotates, vectors);
  } else {
    place.group -= of_k;
  }
  if (place.group >= of_k)
    return;
  row = request(v, call.v_head, kv.kv_heads);
  dst += kv.kv_heads * page_rows * kBytes;
  if (kCodes)
    scales += kv.kv_heads * page_rows * (D / 32);
  store_heads<D, E, false, kCodes>(place, row, kv.kv_heads, v, call.v_head, dst, page_rows * kBytes, scales, page_rows * (D / 32), first >= 0, nullptr, 0.0f,
                                   nullptr, nullptr, false, vectors);
}

// Warps as above; bf16 pages are copied, head_dim / 32 dimensions per lane.
template <int E, bool F32>
__global__ void __launch_bounds__(32 * kWarps)
paged_read_kernel(PagedKv kv, PagedBatch batch, void *__restrict__ k_out, void *__restrict__ v_out, unsigned share, int *__restrict__ status) {
  constexpr int D = 32 * E, kAhead = 8;
  const unsigned warp = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, t = static_cast<int>(warp / share), step = static_cast<int>(share);
  grid_dependency_sync();
  if (static_cast<unsigned>(t) >= static_cast<unsigned>(batch.tokens))
    return;
  const int64_t first = cached_row(kv, batch, t, status);
  if (first < 0)
    return;
  const uint16_t *src = reinterpret_cast<const uint16_t *>(kv.pages) + first * D + lane * E;
  const int64_t at = static_cast<int64_t>(t) * kv.kv_heads * D + lane * E;
  for (int item = static_cast<int>(warp % share); item < 2 * kv.kv_heads; item += kAhead * step) {
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
paged_read_q4_kernel(PagedKv kv, PagedBatch batch, void *__restrict__ k_out, void *__restrict__ v_out, unsigned share, int *__restrict__ status) {
  constexpr int kLanes = D / 16, kRows = 32 / kLanes, kAhead = 2;
  const unsigned warp = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, l = lane % kLanes, t = static_cast<int>(warp / share);
  grid_dependency_sync();
  if (static_cast<unsigned>(t) >= static_cast<unsigned>(batch.tokens))
    return;
  const int64_t first = cached_row(kv, batch, t, status);
  if (first < 0)
    return;
  const uint8_t *src = kv.pages + first * (D / 2) + l * 8;
  const uint16_t *scales = kv.scales + first * (D / 32) + l / 2;
  const int64_t at = static_cast<int64_t>(t) * kv.kv_heads * D + l * 16;
  const int step = static_cast<int>(share) * kRows;
  for (int front = static_cast<int>(warp % share) * kRows + lane / kLanes; front < 2 * kv.kv_heads; front += kAhead * step) {
    uint2 codes[kAhead];
    uint16_t scale[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t row = static_cast<int64_t>(front + u * step) << kv.page_shift;
      if (front + u * step < 2 * kv.kv_heads) {
        codes[u] = *reinterpret_cast<const uint2 *>(src + row * (D / 2));
        scale[u] = scales[row * (D / 32)];
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int item = front + u * step;
      if (item >= 2 * kv.kv_heads)
        break;
      const float d = f16_bits_to_f32(scale[u]);
      const bool is_v = item >= kv.kv_heads;
      void *out = is_v ? v_out : k_out;
      const int64_t to = at + (item - (is_v ? kv.kv_heads : 0)) * D;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t w = h ? codes[u].y : codes[u].x;
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
}

bool aligned(const void *p, int64_t stride0, int64_t stride1, int elements) {
  return reinterpret_cast<uintptr_t>(p) % (2 * elements) == 0 && stride0 % elements == 0 && stride1 % elements == 0;
}

// Warps per token: as many as the SMs hold at a time, 32 each.  256 tokens of 16 + 2 x 2 heads of 128: 9.2 us with half of
// them, 8.1 with these or more; 4000 of 16 + 2 x 1 heads of 64: 14.8 us with these, 19.9 with four times as many.
int warps_per_token(int tokens, int groups, int sms) {
  const int share = sms * 32 / tokens;
  return share < 1 ? 1 : share < groups ? share : groups;
}

dim3 grid(int tokens, int share) { return dim3(static_cast<unsigned>((static_cast<int64_t>(tokens) * share + kWarps - 1) / kWarps)); }

template <int D, int E>
cudaError_t append(const PagedKv &kv, const PagedBatch &batch, const PagedAppend &call, int *status, int sms, cudaStream_t stream) {
  constexpr int kRows = 32 * E / D;
  const bool tables = reinterpret_cast<uintptr_t>(call.cos) % 16 == 0 && reinterpret_cast<uintptr_t>(call.sin) % 16 == 0 && call.rot % 4 == 0;
  const int vectors = (call.heads == 0 || aligned(call.q, call.q_row, call.q_head, E) ? 1 : 0) | (aligned(call.k, call.k_row, call.k_head, E) ? 2 : 0) |
                      (aligned(call.v, call.v_row, call.v_head, E) ? 4 : 0) | (tables ? 8 : 0) |
                      (aligned(call.q_norm, 0, 0, E) && aligned(call.k_norm, 0, 0, E) ? 16 : 0);
  const int share = warps_per_token(batch.tokens, (call.heads + kRows - 1) / kRows + 2 * ((kv.kv_heads + kRows - 1) / kRows), sms);
  if (kv.scales)
    return launch_chained(paged_append_kernel<D, E, true>, grid(batch.tokens, share), dim3(32 * kWarps), 0, stream, kv, batch, call, vectors, share, status);
  return launch_chained(paged_append_kernel<D, E, false>, grid(batch.tokens, share), dim3(32 * kWarps), 0, stream, kv, batch, call, vectors, share, status);
}

template <int E, bool F32>
cudaError_t read(const PagedKv &kv, const PagedBatch &batch, void *k_out, void *v_out, int *status, int sms, cudaStream_t stream) {
  constexpr int D = 32 * E;
  const int rows = kv.scales ? 512 / D : 1, share = warps_per_token(batch.tokens, (2 * kv.kv_heads + rows - 1) / rows, sms);
  if (kv.scales)
    return launch_chained(paged_read_q4_kernel<D, F32>, grid(batch.tokens, share), dim3(32 * kWarps), 0, stream, kv, batch, k_out, v_out, share, status);
  return launch_chained(paged_read_kernel<E, F32>, grid(batch.tokens, share), dim3(32 * kWarps), 0, stream, kv, batch, k_out, v_out, share, status);
}

} // namespace

cudaError_t launch_paged_append(const PagedKv &kv, const PagedBatch &batch, const PagedAppend &call, int *status, int sms, cudaStream_t stream) {
  const bool eights = call.rot % 16 == 0;
  switch (kv.head_dim) {
  case 64:
    return eights ? append<64, 8>(kv, batch, call, status, sms, stream) : append<64, 2>(kv, batch, call, status, sms, stream);
  case 128:
    return eights ? append<128, 8>(kv, batch, call, status, sms, stream) : append<128, 4>(kv, batch, call, status, sms, stream);
  case 256:
    return append<256, 8>(kv, batch, call, status, sms, stream);
  default:
    return cudaErrorInvalidValue;
  }
}

cudaError_t launch_paged_read(const PagedKv &kv, const PagedBatch &batch, void *k_out, void *v_out, int out_dtype, int *status, int sms,
                              cudaStream_t stream) {
  const bool f32 = out_dtype == kF32;
  switch (kv.head_dim) {
  case 64:
    return f32 ? read<2, true>(kv, batch, k_out, v_out, status, sms, stream) : read<2, false>(kv, batch, k_out, v_out, status, sms, stream);
  case 128:
    return f32 ? read<4, true>(kv, batch, k_out, v_out, status, sms, stream) : read<4, false>(kv, batch, k_out, v_out, status, sms, stream);
  case 256:
    return f32 ? read<8, true>(kv, batch, k_out, v_out, status, sms, stream) : read<8, false>(kv, batch, k_out, v_out, status, sms, stream);
  default:
    return cudaErrorInvalidValue;
  }
}

} // namespace llmcp_b200
