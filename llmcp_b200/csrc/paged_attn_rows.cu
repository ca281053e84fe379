// Attention over the paged cache for few rows: the tokens of one sequence times the query heads that share a key head are
// at most 16 rows (one to a few new tokens of every sequence).
//
//   score s_rj = scale q_r . k_j (capped, biased, masked);  p = 2^(s log2 e - m);  o_r = sum_j p_rj v_j / sum_j p_rj
//
// Bound by HBM: every key and value is read once (4 bytes per dimension of a bf16 pair, 1.125 in 4 bits), and even one
// multiply-add per row and element on the CUDA cores would take longer than the read.  So both products run on mma.sync
// (m16n8k16) with the keys and the value dimensions as the 16-row side and the rows as the 8-column side (padded), one
// or two such columns: the instruction, not tcgen05, because a tile has 8 or 16 rows and its operands come straight from
// registers.  A tile's scores transposed, P^T, become the second product's operand by movmatrix.
//
// One CTA takes `chunk` keys of one (sequence, key head); its four warps take tiles of them in turn, each with a ring of
// its own that a lane or four of the warp feed by TMA (the hardware swizzle makes the ldmatrix reads free of conflicts),
// and running maximum, sum and output of its own; no barrier joins the warps before the end.  Several chunks of a
// sequence are joined by paged_merge_kernel.
//
// bf16 pages: weights are split into two bf16 values (high and rest) that both multiply V, so that their rounding (2^-17)
// does not show.
// 4-bit pages: codes + 8, 0 to 15, are used as f16 bit patterns in place: the four bits of an even nibble are the
// subnormal value code * 2^-24, those of an odd one 16 times that, so one mask makes two operands and the factors go
// into q (exactly: powers of two) or into the end.  For the keys the 8 is taken off the sum, for the values before the product, since a dimension in which a row's heavy key is 0 would
// otherwise be the difference of two large sums.  q is scaled by a power of two per row so that its largest element lies
// in [2^14, 2^15): f16 holds every bf16 value that matters beside it.  A block's score is multiplied by its key scale in
// f32 (the part of the 8s is one more product, scales times -8 sum q in two f16 pieces); the value scale goes into the
// weight, p' = f16(f16(p 2^k) d 2^j): k = 15, or less where the largest d so far would take p' past 2^15, and j = 0, or what
// takes that d to [1/2, 1) where it is less (at most 14; both move as the running maximum does).  Weights down to 2^-29 of the
// largest keep f16's relative rounding, 2^-11 twice, for d of 1 and less.
//
// One token of 64 sequences over 2000 to 8191 keys of 4 heads of 256 in bf16: 211 us, 6.5 TB/s.  Over 4 bits neither memory
// (45 % of its rate) nor issue (50 % of the slots, 1190 instructions for 32 keys of 256) is full: scores, maximum, weights and
// values of a warp's tile follow on one another, and three warps a scheduler do not hide their latencies.  One token over
// 131000 keys 43 us, 3.5 TB/s; three tokens of 20 heads of 128, 96 sequences over 1250 to 5000 keys, 93 us, 1.9 TB/s.

#include "common.cuh"
#include "paged.h"
#include "paged_attn.cuh"
#include "tc_common.cuh"

namespace llmcp_b200 {

namespace {

using namespace tc;

constexpr int kWarps = 4;
// A row's weights are 2^(score - reference): the reference is a score that none has outgrown by more than 2^8, so that sums
// and outputs are hardly ever rescaled.
constexpr float kHeadroom = 8.0f;

template <int D, bool Q4, int NT> struct Shape {
  static constexpr int keys = Q4 ? (D == 256 || NT == 2 ? 32 : 64) : 4096 / D; // keys per tile of a warp: 8 KB of bf16, 1 to 4 of codes
  static constexpr int row_bytes = Q4 ? D / 2 : 128;                // shared-memory row: the swizzle's span
  static constexpr int slabs = Q4 ? 1 : D / 64;                     // a bf16 row lies in slabs of 64 dimensions
  static constexpr int value_bytes = keys * row_bytes * slabs;
  static constexpr int scale_bytes = Q4 ? keys * D / 16 : 0;
  static constexpr int slot_bytes = (value_bytes + (D == 64 ? 2 : 1) * scale_bytes + 1023) / 1024 * 1024;
  static constexpr int slots = 3;
  static constexpr int blocks = D / 32;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t address) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool F16> __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t a0, const uint32_t a1, const uint32_t a2, const uint32_t a3, const uint32_t b0, const uint32_t b1) {
  if constexpr (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The first product of a sum: nothing to add to.
__device__ __forceinline__ void mma16816_f16_first(float (&d)[4], const uint32_t a0, const uint32_t a1, const uint32_t a2, const uint32_t a3, const uint32_t b0, const uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t mul_f16(uint32_t x, uint32_t y) {
  uint32_t z;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(z) : "r"(x), "r"(y));
  return z;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 f16_pair(uint32_t word) {
  float2 v;
  asm("{ .reg .b16 l, h; mov.b32 {l, h}, %2; cvt.f32.f16 %0, l; cvt.f32.f16 %1, h; }" : "=f"(v.x), "=f"(v.y) : "r"(word));
  return v;
}

__device__ __forceinline__ uint32_t sub_f16(uint32_t x, uint32_t y) {
  uint32_t z;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(z) : "r"(x), "r"(y));
  return z;
}

// N neighbouring words of shared memory.
template <int N> __device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint32_t *p) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4 *>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *p;
  }
}

// mbar_expect_tx and tma_load_2d on shared-memory addresses.
__device__ __forceinline__ void expect_at(uint32_t bar, uint32_t bytes) {
  asm volatile("{ .reg .b64 t; mbarrier.arrive.expect_tx.shared::cta.b64 t, [%0], %1; }" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_box(uint32_t to, const CUtensorMap *map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
               : "memory");
}

struct Rows {
  PagedKv kv;
  PagedBatch batch;
  PagedAttention call;
  int chunk, chunks, box_rows;
  int out_of_range; // a row coordinate past the last row of the cache: reads as zeros
  uint32_t spin_limit;
};

template <int D, bool Q4, int NT>
__global__ void __launch_bounds__(32 * kWarps, Q4 ? (NT * D <= 256 ? 3 : 2) : 2)
paged_rows_kernel(const __grid_constant__ CUtensorMap map_values, const __grid_constant__ CUtensorMap map_scales,
                  const __grid_constant__ Rows p, int *__restrict__ status) {
  using S = Shape<D, Q4, NT>;
  constexpr int KT = S::keys, M = KT / 16, NB = S::blocks, MT = D / 16;
  constexpr bool kQueriesShared = Q4 || NT * D > 256; // the queries' fragments in shared memory: registers are for warps
  extern __shared__ uint8_t raw_smem[];
  __shared__ uint64_t full[kWarps][S::slots];
  __shared__ float warp_max[kWarps][NT * 8], warp_sum[kWarps][NT * 8];
  __shared__ int sees[NT * 8];                       // keys below it
  __shared__ float slope[NT * 8];
  __shared__ int at[NT * 8], exponents[NT * 8]; // position; of the power of two that takes a row's products back
  __shared__ uint2 offsets_sm[Q4 ? NT : 1][32];
  __shared__ int failed;
  uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int chunk_index = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  if (lane == 0)
    for (int i = 0; i < S::slots; ++i)
      mbar_init(&full[warp][i], 1);
  if (tid == 0)
    failed = 0;
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncthreads();
  grid_dependency_sync();
  const PagedSequence seq = paged_sequence(p.batch, p.kv.page_shift, b, tid == 0 && chunk_index == 0 && kvh == 0 ? status : nullptr);
  const int group = p.call.heads / p.kv.kv_heads, rows = seq.count * group;
  const int key0 = chunk_index * p.chunk, key1 = min(seq.length, key0 + p.chunk);
  if (rows == 0 || (key0 >= key1 && chunk_index > 0))
    return;
  const int tiles_all = max(0, key1 - key0 + KT - 1) / KT, tiles = tiles_all > warp ? (tiles_all - warp + kWarps - 1) / kWarps : 0;

  // ---- the ring: item 2 i + which is tile i's keys or values; lanes below `boxes` issue a box each ----------------------
  const int sub_boxes = KT / p.box_rows, boxes = S::slabs * sub_boxes;
  const int slab = lane / sub_boxes, sub = lane % sub_boxes; // of this lane's box
  uint8_t *ring = base + warp * (S::slots * S::slot_bytes);
  const int32_t *table = p.batch.page_table + b * p.batch.table_stride;
  const int head_rows = p.kv.kv_heads << p.kv.page_shift;
  // scales of 16 rows; a box of them starts on a 128-byte boundary
  const int scale_pitch = D == 64 && p.box_rows == 16 ? 128 : D;
  auto first_key = [&](int i) { return key0 + (warp + i * kWarps) * KT; };
  auto page_of = [&](int i) { // of this lane's rows in tile i
    const int key = first_key(i) + sub * p.box_rows;
    return i < tiles && lane < boxes && key < seq.length ? table[key >> p.kv.page_shift] : -1;
  };
  auto row_of = [&](int i, int page) { // of this lane's box of keys in tile i; out of range past the sequence
    const int key = first_key(i) + sub * p.box_rows;
    if (i >= tiles || lane >= boxes || key >= seq.length)
      return p.out_of_range;
    if (page >= 0 && page < p.kv.num_pages)
      return page * 2 * head_rows + (kvh << p.kv.page_shift) + (key & ((1 << p.kv.page_shift) - 1));
    if (status)
      atomicOr(status, kStatusBadBatch);
    return p.out_of_range;
  };
  const uint32_t ring_address = smem_u32(ring), full_address = smem_u32(&full[warp][0]);
  const uint32_t box_at = (slab * KT + sub * p.box_rows) * S::row_bytes, scales_at = S::value_bytes + sub * (p.box_rows / 16) * scale_pitch;
  int next_tile = 0, issue_slot = 0, issued = 0; // the next items are next_tile's: its row, and the page of the tile behind it
  int row_next = row_of(0, page_of(0)), page_behind = page_of(1);
  auto copy = [&](int row) {
    const uint32_t bar = full_address + issue_slot * 8, slot = ring_address + issue_slot * S::slot_bytes;
    if (lane == 0)
      expect_at(bar, S::value_bytes + S::scale_bytes);
    __syncwarp();
    if (lane < boxes) {
      copy_box(slot + box_at, &map_values, slab * 64, row, bar);
      if (Q4)
        copy_box(slot + scales_at, &map_scales, 0, row >> 4, bar);
    }
    issue_slot = issue_slot + 1 == S::slots ? 0 : issue_slot + 1;
    ++issued;
  };
  auto issue_keys = [&]() {
    if (next_tile < tiles)
      copy(row_next);
  };
  auto issue_values = [&]() {
    if (next_tile < tiles) {
      copy(row_next == p.out_of_range ? row_next : row_next + head_rows);
      ++next_tile;
      row_next = row_of(next_tile, page_behind);
      page_behind = page_of(next_tile + 1);
    }
  };
  // three slots: the item behind a tile's values is the next but one tile's keys' place
  issue_keys();
  issue_values();
  issue_keys();

  // The sign of the scale goes into the queries, so that the largest product is the largest score; with a scale of 0 the
  // queries are zeros and the factor stays usable beside -infinity.
  const bool negative = p.call.scale < 0.0f, flat = p.call.scale == 0.0f;
  // ---- the queries: row 8 nt + g is token row / group, head kvh * group + row % group --------------------------------------
  uint32_t queries[kQueriesShared ? 1 : NT][Q4 ? NB * 4 : MT * 2];
  uint4 *queries_sm = reinterpret_cast<uint4 *>(base + kWarps * S::slots * S::slot_bytes);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (kQueriesShared && warp != nt)
      continue;
    const int row = nt * 8 + g;
    const uint16_t *q = p.call.q + (seq.first + row / group) * p.call.q_row + (kvh * group + row % group) * p.call.q_head;
    uint32_t fragment[Q4 ? NB * 4 : MT * 2];
    int exponent = 0;
    if constexpr (Q4) {
      uint4 raw[NB];
      float sums[NB];
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        raw[k] = row < rows && !flat ? *reinterpret_cast<const uint4 *>(q + 32 * k + 8 * t) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          top = max(top, max(w[i] & 0x7fffu, w[i] >> 16 & 0x7fffu));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int up = top == 0 ? 0 : min(126, 14 - (static_cast<int>(top >> 7) - 127)); // q * 2^up has its largest in [2^14, 2^15)
      const float mult = __uint_as_float(static_cast<uint32_t>(up + 127) << 23 | (negative ? 0x80000000u : 0u));
      exponent = 24 - up;
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
        float x[8], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16) * mult;
          sum += x[i];
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sums[k] = sum * (-8.0f / 16777216.0f);
        fragment[4 * k] = pack_f16(x[0], x[4]);
        fragment[4 * k + 1] = pack_f16(x[1] * 0.0625f, x[5] * 0.0625f);
        fragment[4 * k + 2] = pack_f16(x[2], x[6]);
        fragment[4 * k + 3] = pack_f16(x[3] * 0.0625f, x[7] * 0.0625f);
      }
      // place kk of the 16 belongs to block kk % NB: its sum rounded, then what that leaves, then nothing
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float v[2] = {0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < 16; ++kk)
          if (kk / 2 == t + 4 * h && kk < 2 * NB) {
            const float high = f16_pair(pack_f16(sums[kk % NB], 0.0f)).x;
            v[kk & 1] = kk < NB ? high : sums[kk % NB] - high;
          }
        reinterpret_cast<uint32_t *>(&offsets_sm[nt][lane])[h] = pack_f16(v[0], v[1]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < MT; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          fragment[2 * k + i] = row < rows && !flat ? *reinterpret_cast<const uint32_t *>(q + 16 * k + 8 * i + 2 * t) ^ (negative ? 0x80008000u : 0u) : 0;
    }
    if constexpr (kQueriesShared) {
#pragma unroll
      for (int k = 0; k < D / 32; ++k)
        queries_sm[(nt * (D / 32) + k) * 32 + lane] = make_uint4(fragment[4 * k], fragment[4 * k + 1], fragment[4 * k + 2], fragment[4 * k + 3]);
    } else {
#pragma unroll
      for (int k = 0; k < (Q4 ? NB * 4 : MT * 2); ++k)
        queries[nt][k] = fragment[k];
    }
    if (Q4 && t == 0)
      exponents[row] = exponent;
  }
  // what each row sees, and its bias
  if (tid < NT * 8) {
    const int position = seq.length - seq.count + tid / group;
    sees[tid] = tid < rows ? min(seq.length, max(position + 1, p.call.prefix ? p.call.prefix[b] : 0)) : seq.length;
    slope[tid] = p.call.slopes && tid < rows ? p.call.slopes[kvh * group + tid % group] * 1.4426950408889634f : 0.0f;
    at[tid] = position;
  }
  __syncthreads();
  uint32_t offsets[NT][2]; // 4 bits: what a block's scale is multiplied by to take the 8 off its codes, as f16 and its rest
  float factor[NT][2];     // what makes a column's products scores (in units of log 2, or before the cap)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if constexpr (Q4) {
      offsets[nt][0] = offsets_sm[nt][lane].x;
      offsets[nt][1] = offsets_sm[nt][lane].y;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      factor[nt][i] = flat ? 1.0f : fabsf(p.call.scale) * (p.call.softcap > 0.0f ? 1.0f : 1.4426950408889634f);
      if constexpr (Q4) { // -102 to 138: two powers of two, one may be past f32's end
        const int e = exponents[nt * 8 + 2 * t + i];
        factor[nt][i] = factor[nt][i] * __int_as_float((127 + e / 2) << 23) * __int_as_float((127 + e - e / 2) << 23);
      }
    }
  }
  // four words of the fragments of dimensions 32 k .. 32 k + 31
  auto query_words = [&](int nt, int k, uint32_t (&w)[4]) {
    if constexpr (kQueriesShared) {
      const uint4 v = queries_sm[(nt * (D / 32) + k) * 32 + lane];
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = queries[nt][4 * k + i];
    }
  };

  const int sees_least = min(seq.length, max(seq.length - seq.count + 1, p.call.prefix ? p.call.prefix[b] : 0)); // the first row
  const float cap = p.call.softcap, over_cap = cap > 0.0f ? 1.0f / cap : 0.0f;
  const bool biased = p.call.slopes != nullptr;

  float top[NT][2], sum[NT][2], out[MT][NT][4];
  float shift = Q4 ? kHeadroom - 15.0f : 0.0f; // references are kept without it; weights are 2^(score - maximum - shift)
  int lift = 14;                               // 4 bits: value scales, and outputs with them, are 2^lift times themselves
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    top[nt][0] = top[nt][1] = -INFINITY;
    sum[nt][0] = sum[nt][1] = 0.0f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        out[mt][nt][i] = 0.0f;
  }

  // where a lane reads for ldmatrix: row `row` of 16, 16-byte piece `piece` as the swizzle placed it; another even piece is
  // an exclusive or with it (rows and slots are aligned to the swizzle's span), another 16 rows an addition
  auto piece_offset = [&](int row, int piece) {
    if constexpr (S::row_bytes == 128)
      return row * 128 + ((piece ^ (row & 7)) << 4);
    else if constexpr (S::row_bytes == 64)
      return row * 64 + ((piece ^ (row >> 1 & 3)) << 4);
    else
      return row * 32 + ((piece ^ (row >> 2 & 1)) << 4);
  };
  // a row's scales in a slot, two to a word
  auto scale_words = [&](int s, int row) {
    return reinterpret_cast<const uint32_t *>(ring + s * S::slot_bytes + S::value_bytes + (row >> 4) * scale_pitch + (row & 15) * (D / 16));
  };
  const int lm_row = lane & 7, lm_matrix = lane >> 3;
  const int rows_first = piece_offset((lm_matrix & 1) * 8 + lm_row, lm_matrix >> 1);   // matrices: rows, then pieces
  const int pieces_first = piece_offset((lm_matrix >> 1) * 8 + lm_row, lm_matrix & 1); // pieces, then rows
  int slot_now = 0, phase_now = 0;
  auto next_slot = [&]() {
    if (++slot_now == S::slots) {
      slot_now = 0;
      phase_now ^= 1;
    }
  };
  bool ok = true;
  for (int i = 0; i < tiles; ++i) {
    const int j0 = first_key(i);
    // ---- scores -------------------------------------------------------------------------------------------------------------
    int s = slot_now;
    ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][s], phase_now, &failed, p.spin_limit));
    if (!ok)
      break;
    uint32_t slot = ring_address + s * S::slot_bytes;
    next_slot();
    float x[M][NT][4];
#pragma unroll
    for (int m = 0; m < M; ++m) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          x[m][nt][c] = 0.0f;
      if constexpr (Q4) {
        const uint32_t pair0 = scale_words(s, m * 16 + g)[t % (NB / 2)], pair1 = scale_words(s, m * 16 + g + 8)[t % (NB / 2)];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma16816_f16_first(x[m][nt], pair0, pair1, pair0, pair1, offsets[nt][0], offsets[nt][1]);
        uint32_t sw[2][NB / 2];
        load_words(sw[0], scale_words(s, m * 16 + g));
        load_words(sw[1], scale_words(s, m * 16 + g + 8));
#pragma unroll
        for (int k = 0; k < NB; k += 2) {
          uint32_t w[4]; // block k: rows g, g + 8; block k + 1 the same
          ldmatrix4(w, (slot + rows_first ^ k << 4) + m * 16 * S::row_bytes);
          const float2 scale0 = f16_pair(sw[0][k / 2]), scale1 = f16_pair(sw[1][k / 2]);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t lo = w[2 * u], hi = w[2 * u + 1], lo8 = lo >> 8, hi8 = hi >> 8;
            const uint32_t a[8] = {lo & 0x000f000fu, hi & 0x000f000fu, lo & 0x00f000f0u, hi & 0x00f000f0u,
                                   lo8 & 0x000f000fu, hi8 & 0x000f000fu, lo8 & 0x00f000f0u, hi8 & 0x00f000f0u};
            const float d0 = u ? scale0.y : scale0.x, d1 = u ? scale1.y : scale1.x;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              uint32_t q[4];
              query_words(nt, k + u, q);
              float acc[4];
              mma16816_f16_first(acc, a[0], a[1], a[2], a[3], q[0], q[1]);
              mma16816<true>(acc, a[4], a[5], a[6], a[7], q[2], q[3]);
              x[m][nt][0] = __fmaf_rn(acc[0], d0, x[m][nt][0]);
              x[m][nt][1] = __fmaf_rn(acc[1], d0, x[m][nt][1]);
              x[m][nt][2] = __fmaf_rn(acc[2], d1, x[m][nt][2]);
              x[m][nt][3] = __fmaf_rn(acc[3], d1, x[m][nt][3]);
            }
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < MT; k += 2) {
          uint32_t q[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            query_words(nt, k / 2, q[nt]);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t a[4];
            const int piece = 2 * (k + u);
            ldmatrix4(a, (slot + rows_first ^ (piece & 7) << 4) + (piece >> 3) * (KT * 128) + m * 16 * S::row_bytes);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              mma16816<false>(x[m][nt], a[0], a[1], a[2], a[3], q[nt][2 * u], q[nt][2 * u + 1]);
          }
        }
      }
    }
    __syncwarp();
    issue_values();
    // ---- weights ------------------------------------------------------------------------------------------------------------
    s = slot_now;
    ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][s], phase_now, &failed, p.spin_limit));
    if (!ok)
      break;
    slot = ring_address + s * S::slot_bytes;
    next_slot();
    const bool tail = j0 + KT > seq.length; // rows of the tile past the sequence: whatever they hold
    if (tail) { // their weights are 0, and so are their values (bf16) or scales now
      if constexpr (Q4) {
        for (int row = lane; row < KT; row += 32)
          if (j0 + row >= seq.length)
            for (int k = 0; k < NB / 2; ++k)
              const_cast<uint32_t *>(scale_words(s, row))[k] = 0;
      } else {
        for (int u = lane; u < KT * 8 * S::slabs; u += 32)
          if (j0 + u / 8 % KT >= seq.length)
            *reinterpret_cast<uint4 *>(ring + s * S::slot_bytes + u * 16) = make_uint4(0, 0, 0, 0);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // before the slot's next copy
      __syncwarp();
    }
    const float shift_before = shift;
    const int lift_before = lift;
    if constexpr (Q4) {
      // the largest value scale so far as a power of two above it: weights stay at 2^15 or below, and times a scale too
      uint32_t largest = 0;
#pragma unroll
      for (int n = 0; n < KT / 32; ++n)
#pragma unroll
        for (int k = 0; k < NB / 2; ++k)
          largest = __vmaxu2(largest, scale_words(s, n * 32 + lane)[k] & 0x7fff7fffu);
      largest = __reduce_max_sync(0xffffffffu, max(largest & 0xffffu, largest >> 16));
      shift = fmaxf(shift, static_cast<float>(static_cast<int>(largest >> 10) - 29) + kHeadroom);
      lift = min(lift, max(14 - static_cast<int>(largest >> 10), 0));
    }
    const bool masked = j0 + KT > sees_least; // some row does not see some key of the tile
    bool outgrown = shift != shift_before || lift != lift_before; // else the reference moves only where a score has outgrown it by 2^8
    float best[NT][2], scaled[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      scaled[nt][0] = factor[nt][0], scaled[nt][1] = factor[nt][1];
      if (cap > 0.0f) {
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int c = 0; c < 4; c += 2) {
            const float2 v = capped_log2(mul2(pair(x[m][nt][c], x[m][nt][c + 1]), pair(factor[nt][0], factor[nt][1])), cap, over_cap);
            x[m][nt][c] = v.x;
            x[m][nt][c + 1] = v.y;
          }
        scaled[nt][0] = scaled[nt][1] = 1.0f;
      }
      if (biased || masked) {
        float from[2]; // distances to the lane's first key: whole numbers are exact to 2^24, positions go past it
#pragma unroll
        for (int col = 0; col < 2; ++col)
          from[col] = static_cast<float>(at[nt * 8 + 2 * t + col] - j0 - g);
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int j = j0 + m * 16 + g + (c >> 1) * 8, row = nt * 8 + 2 * t + (c & 1);
            x[m][nt][c] = j < sees[row] ? x[m][nt][c] * scaled[nt][c & 1] - slope[row] * fabsf(from[c & 1] - static_cast<float>(m * 16 + (c >> 1) * 8)) : -INFINITY;
          }
        scaled[nt][0] = scaled[nt][1] = 1.0f;
      }
      best[nt][0] = best[nt][1] = -INFINITY;
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int col = 0; col < 2; ++col)
          best[nt][col] = fmaxf(best[nt][col], fmaxf(x[m][nt][col], x[m][nt][col + 2]));
#pragma unroll
      for (int col = 0; col < 2; ++col) {
        best[nt][col] = best[nt][col] == -INFINITY ? -INFINITY : best[nt][col] * scaled[nt][col];
        outgrown |= best[nt][col] > top[nt][col] + kHeadroom;
      }
    }
    if (__any_sync(0xffffffffu, outgrown)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float moved[2];
#pragma unroll
        for (int col = 0; col < 2; ++col) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1)
            best[nt][col] = fmaxf(best[nt][col], __shfl_xor_sync(0xffffffffu, best[nt][col], o));
          const float higher = best[nt][col] > top[nt][col] + kHeadroom ? best[nt][col] : top[nt][col];
          moved[col] = higher == -INFINITY ? 1.0f : exp2_approx((top[nt][col] + shift_before) - (higher + shift));
          top[nt][col] = higher;
          sum[nt][col] *= moved[col];
        }
        if constexpr (Q4) {
          const float lowered = __int_as_float((127 + lift - lift_before) << 23);
          moved[0] *= lowered;
          moved[1] *= lowered;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            out[mt][nt][c] *= moved[c & 1];
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float minus[2] = {top[nt][0] == -INFINITY ? 0.0f : -(top[nt][0] + shift), top[nt][1] == -INFINITY ? 0.0f : -(top[nt][1] + shift)};
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int c = 0; c < 4; ++c) // a row that has seen nothing: 2^(-inf - 0)
          x[m][nt][c] = exp2_approx(__fmaf_rn(x[m][nt][c], scaled[nt][c & 1], minus[c & 1]));
    }
    if constexpr (!Q4) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            sum[nt][c & 1] += x[m][nt][c];
    }
    // ---- values -------------------------------------------------------------------------------------------------------------
#pragma unroll
    for (int m = 0; m < M; ++m) {
      if constexpr (Q4) {
        uint32_t weights[NT][2]; // of keys 2 t, 2 t + 1 and 2 t + 8, 2 t + 9 in row g
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            sum[nt][c & 1] += x[m][nt][c];
          weights[nt][0] = transpose8x8(pack_f16(x[m][nt][0], x[m][nt][1]));
          weights[nt][1] = transpose8x8(pack_f16(x[m][nt][2], x[m][nt][3]));
        }
        uint32_t sw[4][NB / 2];
#pragma unroll
        for (int n = 0; n < 4; ++n)
          load_words(sw[n], scale_words(s, m * 16 + 2 * t + (n & 1) + (n >> 1) * 8));
        if (lift > 0) {
          const uint32_t power = static_cast<uint32_t>(15 + lift) * 0x04000400u;
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int k = 0; k < NB / 2; ++k)
              sw[n][k] = mul_f16(sw[n][k], power);
        }
#pragma unroll
        for (int k = 0; k < NB; k += 2) {
          uint32_t w[4]; // block k: keys 0-7, 8-15; block k + 1 the same
          ldmatrix4_trans(w, (slot + rows_first ^ k << 4) + m * 16 * S::row_bytes);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t lo = w[2 * u], hi = w[2 * u + 1], lo8 = lo >> 8, hi8 = hi >> 8;
            uint32_t a[8] = {lo & 0x000f000fu, lo & 0x00f000f0u, hi & 0x000f000fu, hi & 0x00f000f0u,
                             lo8 & 0x000f000fu, lo8 & 0x00f000f0u, hi8 & 0x000f000fu, hi8 & 0x00f000f0u};
#pragma unroll
            for (int n = 0; n < 8; ++n)
              a[n] = sub_f16(a[n], n & 1 ? 0x00800080u : 0x00080008u);
            const uint32_t d0 = __byte_perm(sw[0][k / 2], sw[1][k / 2], u ? 0x7632 : 0x5410);
            const uint32_t d1 = __byte_perm(sw[2][k / 2], sw[3][k / 2], u ? 0x7632 : 0x5410);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              const uint32_t b0 = mul_f16(weights[nt][0], d0), b1 = mul_f16(weights[nt][1], d1);
              mma16816<true>(out[2 * (k + u)][nt], a[0], a[1], a[2], a[3], b0, b1);
              mma16816<true>(out[2 * (k + u) + 1][nt], a[4], a[5], a[6], a[7], b0, b1);
            }
          }
        }
      } else {
        uint32_t high[NT][2], rest[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float p0 = x[m][nt][2 * h], p1 = x[m][nt][2 * h + 1];
            const uint32_t w = f32x2_to_bf16x2_hw(p0, p1);
            high[nt][h] = transpose8x8(w);
            rest[nt][h] = transpose8x8(f32x2_to_bf16x2_hw(p0 - __uint_as_float(w << 16), p1 - __uint_as_float(w & 0xffff0000u)));
          }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t a[4];
          const int piece = 2 * mt;
          ldmatrix4_trans(a, (slot + pieces_first ^ (piece & 7) << 4) + (piece >> 3) * (KT * 128) + m * 16 * S::row_bytes);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816<false>(out[mt][nt], a[0], a[1], a[2], a[3], high[nt][0], high[nt][1]);
            mma16816<false>(out[mt][nt], a[0], a[1], a[2], a[3], rest[nt][0], rest[nt][1]);
          }
        }
      }
    }
    __syncwarp();
    issue_keys();
  }
  if (!ok) // copies already requested still write into this CTA's shared memory
    for (int n = max(0, issued - S::slots); n < issued; ++n)
      mbar_wait_quiet(&full[warp][n % S::slots], (n / S::slots) & 1, p.spin_limit);

  // ---- the warps' parts joined --------------------------------------------------------------------------------------------------
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (Q4)
        top[nt][i] += shift; // of the weights as they were summed
#pragma unroll
      for (int o = 4; o < 32; o <<= 1)
        sum[nt][i] += __shfl_xor_sync(0xffffffffu, sum[nt][i], o);
      if (g == 0) {
        warp_max[warp][nt * 8 + 2 * t + i] = top[nt][i];
        warp_sum[warp][nt * 8 + 2 * t + i] = sum[nt][i];
      }
    }
  __syncthreads();
  if (failed) {
    if (tid == 0 && status)
      atomicOr(status, kStatusWaitRanOut);
    return;
  }
  float joined[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float all = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        all = fmaxf(all, warp_max[w][nt * 8 + 2 * t + i]);
      joined[nt][i] = top[nt][i] == -INFINITY ? 0.0f : exp2_approx(top[nt][i] - all);
      if (Q4)
        joined[nt][i] *= __int_as_float((127 - lift) << 23);
    }
  // row-major [warp][row][D + 4], over the rings (all copies have landed); the pad keeps the writes off each other's banks
  constexpr int kPitch = D + 4;
  float *parts = reinterpret_cast<float *>(base);
  float *mine = parts + warp * (NT * 8 * kPitch);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float v = out[mt][nt][c];
        int d;
        if constexpr (Q4) {
          // dims 32 k + 4 g + 2 j + (c >> 1) of m-tile 2 k + j; odd nibbles are 16 times their code
          d = (mt / 2) * 32 + 4 * g + 2 * (mt & 1) + (c >> 1);
          v *= c >> 1 ? 1048576.0f : 16777216.0f;
        } else {
          d = mt * 16 + g + (c >> 1) * 8;
        }
        mine[(nt * 8 + 2 * t + (c & 1)) * kPitch + d] = v * joined[nt][c & 1];
      }
  __syncthreads();
  const int head0 = kvh * group;
  for (int u = tid; u < rows * (D / 8); u += 32 * kWarps) {
    const int row = u / (D / 8), d = u % (D / 8) * 8;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    float all = -INFINITY, total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float *part = parts + (w * NT * 8 + row) * kPitch + d;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] += part[i];
      all = fmaxf(all, warp_max[w][row]);
    }
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      total += warp_max[w][row] == -INFINITY ? 0.0f : warp_sum[w][row] * exp2_approx(warp_max[w][row] - all);
    const int token = seq.first + row / group, head = head0 + row % group;
    if (p.chunks == 1) {
      const float inv = total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[i] *= inv;
      paged_store_row(p.call.out + paged_out_at<D>(p.call, token, head, d), make_float4(v[0], v[1], v[2], v[3]), make_float4(v[4], v[5], v[6], v[7]),
                      paged_gate(p.call, token, head, d), p.call.gate != nullptr);
    } else {
      paged_store_part(static_cast<float *>(p.call.workspace) + paged_out_at<D>(p.call, token, head, 0) * p.chunks + chunk_index * D + d,
                       make_float4(v[0], v[1], v[2], v[3]), make_float4(v[4], v[5], v[6], v[7]));
      if (d == 0)
        paged_store_sums<D>(p.call, p.batch.tokens, p.chunks, chunk_index, token, head, all, total);
    }
  }
}

template <int D, bool Q4, int NT>
cudaError_t launch(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, const PagedSplit &split, int *status, cudaStream_t stream) {
  using S = Shape<D, Q4, NT>;
  Rows p;
  p.kv = kv, p.batch = batch, p.call = call;
  p.chunk = split.chunk, p.chunks = split.chunks;
  p.box_rows = S::keys < (1 << kv.page_shift) ? S::keys : 1 << kv.page_shift;
  const int64_t rows = kv.num_pages * 2 * kv.kv_heads << kv.page_shift;
  p.out_of_range = static_cast<int>(rows);
  p.spin_limit = kSpinLimit<true>;
  CUtensorMap values, scales;
  if (!paged_value_map(&values, kv, rows, p.box_rows) || (Q4 && !paged_scale_map(&scales, kv, rows, p.box_rows)))
    return cudaErrorNotSupported;
  if (!Q4)
    scales = values;
  constexpr size_t ring = kWarps * S::slots * S::slot_bytes + (Q4 || NT * D > 256 ? NT * D * 16 : 0);
  constexpr size_t parts = sizeof(float) * kWarps * NT * 8 * (D + 4);
  constexpr size_t smem = 1024 + (ring > parts ? ring : parts);
  const auto kernel = paged_rows_kernel<D, Q4, NT>;
  if (cudaError_t e = opt_in_shared_memory(reinterpret_cast<const void *>(kernel), smem); e != cudaSuccess)
    return e;
  return launch_chained(kernel, dim3(split.chunks, kv.kv_heads, batch.sequences), dim3(32 * kWarps), smem, stream, values, scales, p, status);
}

template <int D, bool Q4>
cudaError_t launch(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, const PagedSplit &split, int *status, cudaStream_t stream) {
  return static_cast<int64_t>(batch.max_q) * (call.heads / kv.kv_heads) <= 8 ? launch<D, Q4, 1>(kv, batch, call, split, status, stream)
                                                                             : launch<D, Q4, 2>(kv, batch, call, split, status, stream);
}

} // namespace

int paged_rows_tile(const PagedKv &kv, int rows) {
  return kWarps * (kv.scales ? (kv.head_dim == 256 || rows > 8 ? 32 : 64) : 4096 / kv.head_dim);
}

cudaError_t launch_paged_rows(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, const PagedSplit &split, int *status,
                              cudaStream_t stream) {
  switch (kv.head_dim) {
  case 64:
    return kv.scales ? launch<64, true>(kv, batch, call, split, status, stream) : launch<64, false>(kv, batch, call, split, status, stream);
  case 128:
    return kv.scales ? launch<128, true>(kv, batch, call, split, status, stream) : launch<128, false>(kv, batch, call, split, status, stream);
  case 256:
    return kv.scales ? launch<256, true>(kv, batch, call, split, status, stream) : launch<256, false>(kv, batch, call, split, status, stream);
  default:
    return cudaErrorInvalidValue;
  }
}

} // namespace llmcp_b200
