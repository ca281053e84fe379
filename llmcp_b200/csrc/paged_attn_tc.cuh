// What the two attention kernels for prompts share: MMAs and descriptors, tensor-memory stores, a thread's scores on their way
// to weights, and rows of queries and results between global and shared memory.
//
// In both, 128 rows (tokens x the query heads that share a key head) lie in the 128 lanes of tensor memory, a thread of a
// warpgroup each, and scores S = Q K^T, weights P = 2^(S - reference) and O += P V are tcgen05 products.  Keys and values
// are 16-bit tiles: bf16 from the pages, or f16 from an expanded 4-bit cache (an eighth of the values where they are large,
// taken back in the score and at the end); f16 queries are scaled by a power of two per row.
#pragma once

#include "common.cuh"
#include "paged.h"
#include "paged_attn.cuh"
#include "tc_common.cuh"

namespace llmcp_b200 {

namespace tc {

constexpr int kRows = 128;
// A row's weights are 2^(score - reference): the reference is a score that none has outgrown by more than 2^8, so that O is
// hardly ever rescaled.
constexpr float kHeadroom = 8.0f;

struct Tile {
  PagedKv kv;
  PagedBatch batch;
  PagedAttention call;
  int chunk, chunks, box_rows;
  int tokens_per_tile;   // of 128 rows
  unsigned group, one_over_group; // query heads that share a key head; 2^16 / group rounded up
  int64_t expanded_rows; // rows of a sequence's keys in the expanded cache; 0: pages
  const float *divisors; // [sequence][keys, values][kv head]: what the expanded values were divided by; null where there are none
  int out_of_range;      // a row coordinate past the last row: reads as zeros
  uint32_t spin_limit;
};

// D = f32, A and B 16 bits (bf16 or f16), M = 128; B either K-major or MN-major.
template <bool F16, int N, bool MN> static constexpr uint32_t kInstruction =
    (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | (MN ? 1u << 16 : 0u) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(kRows >> 4) << 24);

// A from tensor memory or shared memory, B from shared memory.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t instruction, uint32_t accumulate) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }"
               :
               : "r"(d), "r"(a), "l"(b), "r"(instruction), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t instruction, uint32_t accumulate) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0;\n"
               "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
               :
               : "r"(d), "l"(a), "l"(b), "r"(instruction), "r"(accumulate)
               : "memory");
}

// MN-major operand with 128-byte swizzle: atoms of 64 values (128 bytes) x 8 keys; `slab` bytes to the next 64 values.
__device__ __forceinline__ uint64_t mn_descriptor(uint32_t smem_address, uint32_t slab) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_address & 0x3ffffu) >> 4);
  d |= static_cast<uint64_t>(slab >> 4) << 16;  // leading byte offset: next 64 values
  d |= static_cast<uint64_t>(1024 >> 4) << 32;  // stride byte offset: next 8 keys
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
               "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
               :
               : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
                 "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
               : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               :
               : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <bool F16> __device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if constexpr (F16)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 2^y of two finite values by multiplications: y = n + f with n an integer and |f| <= 1/2 (the range reduction of Cody and
// Waite), 2^f by a polynomial of degree 4 (relative error 2.6e-6, fitted for the smallest largest error), n into the
// exponent.  Below 2^-126 the result is some number about as small.
__device__ __forceinline__ float2 exp2_by_fma(uint64_t y) {
  constexpr float kRound = 12582912.0f; // 1.5 * 2^23: what is added to it is rounded to an integer
  float2 v = halves(y);
  y = pair(fmaxf(v.x, -126.0f), fmaxf(v.y, -126.0f));
  const uint64_t t = add2(y, pair(kRound, kRound)), f = fma2(add2(t, pair(-kRound, -kRound)), pair(-1.0f, -1.0f), y);
  uint64_t r = fma2(f, pair(0.00957010032775151f, 0.00957010032775151f), pair(0.05591786276854936f, 0.05591786276854936f));
  r = fma2(r, f, pair(0.24024744889319694f, 0.24024744889319694f));
  r = fma2(r, f, pair(0.693121814447754f, 0.693121814447754f));
  r = fma2(r, f, pair(0.9999992614202372f, 0.9999992614202372f));
  const float2 n = halves(t), e = halves(r);
  v.x = __int_as_float(__float_as_int(e.x) + (__float_as_int(n.x) << 23));
  v.y = __int_as_float(__float_as_int(e.y) + (__float_as_int(n.y) << 23));
  return v;
}

// Two barriers awaited together: a look at one takes some 150 cycles, and looks at both overlap.
__device__ __forceinline__ bool wait_for_both(uint64_t *a, uint32_t pa, uint64_t *b, uint32_t pb, volatile int *abort_flag, uint32_t limit) {
  const uint32_t aa = smem_u32(a), ab = smem_u32(b);
  for (uint32_t spin = 0; spin < limit; ++spin) {
    const bool ra = mbar_poll<false>(aa, pa), rb = mbar_poll<false>(ab, pb);
    if (ra && rb)
      return true;
    if ((spin & 63) == 63 && *abort_flag)
      return false;
  }
  *abort_flag = 1;
  return false;
}

// The scores of a row in a tile, from tensor memory.
template <int KT> __device__ __forceinline__ void load_scores(uint32_t (&x)[KT / 32][32], uint32_t address) {
#pragma unroll
  for (int c = 0; c < KT / 32; ++c)
    tmem_issue32(address + c * 32, x[c]);
#pragma unroll
  for (int c = 0; c < KT / 32; ++c)
    tmem_wait_loads_into(x[c]);
}

// What makes a row's products scores.
struct RowScores {
  float factor;        // to units of log 2, or (capped) to scores
  float cap, over_cap; // cap 0: none
  float slope;         // bias by distance from position `at`
  int at;
  int sees, sees_least; // keys below: this row, every row of its tile
  bool biased;
};

template <int KT, bool HALF> __device__ __forceinline__ void cap_scores(uint32_t (&x)[KT / 32][32], float into, float scale) {
#pragma unroll
  for (int c = 0; c < KT / 32; ++c)
#pragma unroll
    for (int u = 0; u < 32; u += 2) {
      const float2 v = halves(tanh_by_fma<HALF>(mul2(pair(__uint_as_float(x[c][u]), __uint_as_float(x[c][u + 1])), pair(into, into)), scale));
      x[c][u] = __float_as_uint(v.x);
      x[c][u + 1] = __float_as_uint(v.y);
    }
}

// Products to scores (up to the returned factor), capped, biased and masked.
template <int KT> __device__ __forceinline__ float shape_scores(uint32_t (&x)[KT / 32][32], const RowScores &r, int j0) {
  float scaled = r.factor;
  if (r.cap > 0.0f) {
    float most[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < KT / 32; ++c)
#pragma unroll
      for (int u = 0; u < 32; u += 2)
        most[u >> 1 & 3] = max3(most[u >> 1 & 3], fabsf(__uint_as_float(x[c][u])), fabsf(__uint_as_float(x[c][u + 1])));
    const float into = r.factor * r.over_cap, far = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * into, scale = r.cap * 1.4426950408889634f;
    // the hardware's exp and reciprocal are few; scores within the cap, which is the rule, do without
    if (!__any_sync(0xffffffffu, !(far <= 0.5f))) {
      cap_scores<KT, true>(x, into, scale);
    } else if (!__any_sync(0xffffffffu, !(far <= 1.0f))) {
      cap_scores<KT, false>(x, into, scale);
    } else {
#pragma unroll
      for (int c = 0; c < KT / 32; ++c)
#pragma unroll
        for (int u = 0; u < 32; u += 2) {
          const float2 v = capped_log2(mul2(pair(__uint_as_float(x[c][u]), __uint_as_float(x[c][u + 1])), pair(r.factor, r.factor)), r.cap, r.over_cap);
          x[c][u] = __float_as_uint(v.x);
          x[c][u + 1] = __float_as_uint(v.y);
        }
    }
    scaled = 1.0f;
  }
  if (r.biased) {
    const float from = static_cast<float>(r.at - j0); // a distance: whole numbers are exact to 2^24, positions go past it
#pragma unroll
    for (int c = 0; c < KT / 32; ++c)
#pragma unroll
      for (int u = 0; u < 32; ++u)
        x[c][u] = __float_as_uint(__fmaf_rn(-r.slope, fabsf(from - static_cast<float>(c * 32 + u)), __uint_as_float(x[c][u]) * scaled));
    scaled = 1.0f;
  }
  if (j0 + KT > r.sees_least) {
#pragma unroll
    for (int c = 0; c < KT / 32; ++c)
#pragma unroll
      for (int u = 0; u < 32; ++u)
        if (j0 + c * 32 + u >= r.sees)
          x[c][u] = 0xff800000u;
  }
  return scaled;
}

template <int KT> __device__ __forceinline__ float largest_score(const uint32_t (&x)[KT / 32][32], float scaled) {
  float most[4]; // side by side: one chain of maxima would take as long as everything else
#pragma unroll
  for (int u = 0; u < 4; ++u)
    most[u] = -INFINITY;
#pragma unroll
  for (int c = 0; c < KT / 32; ++c)
#pragma unroll
    for (int u = 0; u < 32; u += 2)
      most[u >> 1 & 3] = max3(most[u >> 1 & 3], __uint_as_float(x[c][u]), __uint_as_float(x[c][u + 1]));
  const float best = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
  return best == -INFINITY ? best : best * scaled;
}

// Weights over the scores in tensor memory; returns their sum.  f16 weights lie between 2^7 (a row's largest, at least)
// and 2^15, and keep their precision down to 2^-14.  The hardware gives 16 exponentials a cycle; where no score is masked
// FMAS of eight pairs come by multiplications instead.
template <int KT, bool F16, int FMAS>
__device__ __forceinline__ float store_weights(const uint32_t (&x)[KT / 32][32], uint32_t address, float scaled, float reference) {
  const float minus = (reference == -INFINITY ? 0.0f : -reference) + (F16 ? 15.0f - kHeadroom : 0.0f);
  uint64_t added[4] = {0, 0, 0, 0}; // pairs of sums
  const uint64_t scaled2 = pair(scaled, scaled), minus2 = pair(minus, minus);
#pragma unroll
  for (int c = 0; c < KT / 32; ++c) {
    uint32_t w[16];
#pragma unroll
    for (int u = 0; u < 32; u += 2) {
      const uint64_t y = fma2(pair(__uint_as_float(x[c][u]), __uint_as_float(x[c][u + 1])), scaled2, minus2);
      float2 e;
      if ((u >> 1) % 8 * FMAS % 8 < FMAS) { // spread evenly
        e = exp2_by_fma(y);
      } else {
        e = halves(y);
        e = make_float2(exp2_approx(e.x), exp2_approx(e.y));
      }
      added[u >> 1 & 3] = add2(added[u >> 1 & 3], pair(e.x, e.y));
      w[u >> 1] = pack16<F16>(e.x, e.y);
    }
    tmem_store16(address + c * 16, w);
  }
  const float2 sum = halves(add2(add2(added[0], added[1]), add2(added[2], added[3])));
  tmem_wait_stores();
  return sum.x + sum.y;
}

// A row of O times `moved` (0: cleared, whatever it holds).
template <int D> __device__ __forceinline__ void rescale_row(uint32_t address, float moved) {
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t o[32];
    tmem_load32(address + c * 32, o);
#pragma unroll
    for (int u = 0; u < 32; ++u)
      o[u] = __float_as_uint(moved == 0.0f ? 0.0f : __uint_as_float(o[u]) * moved);
    tmem_store32(address + c * 32, o);
  }
  tmem_wait_stores();
}

// Rows of queries, gates and results lie in shared memory as K-major slabs of 64 dimensions, 128 rows of 128 bytes each,
// 16-byte pieces where the 128-byte swizzle has them.  Everything below is done once per CTA and written as short loops:
// unrolled, its instructions take longer to fetch than to execute.
// They come in by TMA, a slab a copy: a box of 64 dimensions x group heads x tokens_per_tile tokens of a [token][head][dim]
// tensor (rows of the next sequence among them, zeros past the tensor, and nothing in the rows past a whole number of tokens).
__device__ __forceinline__ void load_slab(uint8_t *to, const CUtensorMap *map, int dim, int head0, int token0, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(to)),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(dim), "r"(head0), "r"(token0), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ uint32_t piece_at(int row, int piece) { return (piece / 8) * (kRows * 128) + row * 128 + ((piece % 8 ^ row & 7) << 4); }

// Which rows of global memory those are: row r is token r / group, head r % group.  (r below 128 and group at most 128: the
// product with the reciprocal is exact enough.)
struct TileRows {
  unsigned rows, group, one_over_group;
  int token0, head0;
  __device__ __forceinline__ int64_t at(unsigned r, int64_t token_stride, int64_t head_stride) const {
    const unsigned token = r * one_over_group >> 16;
    return static_cast<int64_t>(token0 + token) * token_stride + static_cast<int64_t>(head0 + (r - token * group)) * head_stride;
  }
};

template <int DIMS, int WARPS>
__device__ __forceinline__ void copy_rows_out(uint16_t *to, int64_t token_stride, int64_t head_stride, const uint8_t *from, const TileRows &t, int warp, int lane) {
  constexpr int kLanes = DIMS / 8, kSide = 32 / kLanes;
  const int piece = lane % kLanes;
#pragma unroll 2
  for (int r = warp * kSide + lane / kLanes; r < static_cast<int>(t.rows); r += WARPS * kSide)
    *reinterpret_cast<uint4 *>(to + t.at(r, token_stride, head_stride) + piece * 8) = *reinterpret_cast<const uint4 *>(from + piece_at(r, piece));
}

// f16 queries: the power of two that takes a row's largest |q| into [2^14, 2^15) (1 for a row of zeros), with the sign of
// the scale; and what takes it back.
template <int D> __device__ __forceinline__ float query_multiplier(const uint8_t *queries, int row, bool negative, float *unscale) {
  uint32_t top2 = 0;
#pragma unroll 4
  for (int piece = 0; piece < D / 8; ++piece) {
    const uint4 v = *reinterpret_cast<const uint4 *>(queries + piece_at(row, piece));
    top2 = __vmaxu2(__vmaxu2(top2, __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu)), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
  }
  const uint32_t top = max(top2 & 0xffffu, top2 >> 16);
  const int up = top == 0 ? 0 : min(126, 14 - (static_cast<int>(top >> 7) - 127));
  *unscale = __int_as_float((127 - up) << 23);
  return __uint_as_float(static_cast<uint32_t>(up + 127) << 23 | (negative ? 0x80000000u : 0u));
}

// Two bf16 queries as the products take them: f16 times the multiplier, or bf16 with the sign of the scale; zeros where the
// scale is 0.
template <bool F16> __device__ __forceinline__ uint32_t query_pair(uint32_t w, float multiplier, bool negative, bool flat) {
  if constexpr (F16)
    w = pack16<true>(__uint_as_float(w << 16) * multiplier, __uint_as_float(w & 0xffff0000u) * multiplier);
  else
    w ^= negative ? 0x80008000u : 0u;
  return flat ? 0u : w;
}
template <bool F16> __device__ __forceinline__ uint4 query_piece(uint4 v, float multiplier, bool negative, bool flat) {
  return make_uint4(query_pair<F16>(v.x, multiplier, negative, flat), query_pair<F16>(v.y, multiplier, negative, flat),
                    query_pair<F16>(v.z, multiplier, negative, flat), query_pair<F16>(v.w, multiplier, negative, flat));
}

// DIMS dimensions of a thread's row of O, times `scale` and its gate (in shared memory, where there is one), as bf16 into
// the gate's place; zeros where the row has no weights.
template <int DIMS> __device__ __forceinline__ void unload_row(uint8_t *to, int row, uint32_t address, float scale, bool empty, bool gated) {
#pragma unroll 1
  for (int c = 0; c < DIMS / 32; ++c) {
    uint32_t o[32];
    __syncwarp();
    tmem_load32(address + c * 32, o);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint4 *at = reinterpret_cast<uint4 *>(to + piece_at(row, c * 4 + k));
      const uint4 gate = gated ? *at : make_uint4(0, 0, 0, 0);
      const uint32_t g[4] = {gate.x, gate.y, gate.z, gate.w};
      uint32_t words[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x = empty ? 0.0f : __uint_as_float(o[8 * k + 2 * i]) * scale, y = empty ? 0.0f : __uint_as_float(o[8 * k + 2 * i + 1]) * scale;
        if (gated) {
          x = times_sigmoid(x, __uint_as_float(g[i] << 16));
          y = times_sigmoid(y, __uint_as_float(g[i] & 0xffff0000u));
        }
        words[i] = pack16<false>(x, y);
      }
      *at = make_uint4(words[0], words[1], words[2], words[3]);
    }
  }
}

// The same as a part, f32 rows of the workspace.
template <int DIMS> __device__ __forceinline__ void unload_part(float *to, uint32_t address, float scale, bool empty, bool valid) {
#pragma unroll 1
  for (int c = 0; c < DIMS / 32; ++c) {
    uint32_t o[32];
    __syncwarp();
    tmem_load32(address + c * 32, o);
    if (!valid)
      continue;
#pragma unroll
    for (int u = 0; u < 32; u += 4)
      *reinterpret_cast<float4 *>(to + c * 32 + u) = empty ? make_float4(0.0f, 0.0f, 0.0f, 0.0f)
                                                           : make_float4(__uint_as_float(o[u]) * scale, __uint_as_float(o[u + 1]) * scale,
                                                                         __uint_as_float(o[u + 2]) * scale, __uint_as_float(o[u + 3]) * scale);
  }
}

// What the keys and values of a head of the expanded cache were divided by, into shared memory; then `bar` is told.
__device__ __forceinline__ void fetch_divisors(float (&to)[2], const Tile &p, int b, int kvh, int lane, uint64_t *bar) {
  if (lane < 2)
    to[lane] = p.divisors ? p.divisors[(b * 2 + lane) * p.kv.kv_heads + kvh] : 1.0f;
  __syncwarp();
  if (lane == 0)
    mbar_arrive(bar);
}

// This lane's box of a tile of keys (which = 0) or values: its row coordinate.
__device__ __forceinline__ int tile_box_row(const Tile &p, const PagedSequence &seq, const int32_t *table, int b, int kvh, int which, int key, bool mine, int *status) {
  if (!mine || key >= seq.length)
    return p.out_of_range;
  if (p.expanded_rows)
    return static_cast<int>(((static_cast<int64_t>(b) * 2 + which) * p.kv.kv_heads + kvh) * p.expanded_rows + key);
  const int page = table[key >> p.kv.page_shift];
  if (page >= 0 && page < p.kv.num_pages)
    return (((page * 2 + which) * p.kv.kv_heads + kvh) << p.kv.page_shift) + (key & ((1 << p.kv.page_shift) - 1));
  if (status)
    atomicOr(status, kStatusBadBatch);
  return p.out_of_range;
}

// Rows `past` and up of a tile of values in shared memory become zeros: 0 times whatever they hold is not 0.
template <int KT, int SLABS> __device__ __forceinline__ void zero_tail(uint8_t *tile, int past, int lane) {
  for (int u = lane; u < KT * 8 * SLABS; u += 32)
    if (u / 8 % KT >= past)
      *reinterpret_cast<uint4 *>(tile + u * 16) = make_uint4(0, 0, 0, 0);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

// Maps of the queries and the gates (another of the queries' where there are none).
struct RowMaps {
  CUtensorMap queries, gates;
};

} // namespace tc

cudaError_t launch_paged_narrow(int head_dim, bool f16, const CUtensorMap &values, const tc::RowMaps &maps, const tc::Tile &p, unsigned q_tiles, int *status, cudaStream_t stream);

} // namespace llmcp_b200
