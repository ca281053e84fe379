// Attention over the paged cache for many rows (prompts): both products on tcgen05.
//
//   S = Q K^T,  P = 2^(S scale log2 e - m),  O = sum P V / sum P,   128 rows (tokens x the query heads of one key head) a CTA
//
// Keys and values come as 16-bit tiles by TMA: bf16 straight from the pages; a 4-bit cache is expanded once per call into
// f16 rows (paged_expand_kernel), value = code * scale / 8 rounded to f16 (2^-11; the 8 keeps the largest below f16's
// end and goes into the factors), because every tile of rows would otherwise unpack the same keys again.
//
// One CTA, 384 threads (warp 11 only hands over its registers):
//   warps 0-7  softmax, a thread per row: warps 0-3 take the even key tiles, 4-7 the odd ones.  A thread reads its scores
//              from tensor memory, writes P over them and, when its row's reference moves, rescales its row of O there.
//              The reference (a score that none has outgrown by more than 2^8) passes from tile to tile, between the two
//              warps that share 32 rows, through shared memory; the exponentials of two tiles run side by side.
//   warp 8     one thread issues the MMAs: Q and P from tensor memory, K (K-major) and V (MN-major: rows are keys) from shared memory,
//              both with the 128-byte swizzle.  Scores are issued two or three tiles ahead of P V.
//   warp 9     issues the TMA loads into a ring of tiles, in the order in which the MMAs take them: K0 K1 K2 V0 K3 V1 ...
//   warp 10    zeroes the rows of the last value tile that lie past the sequence: 0 times whatever they hold is not 0.
// Q is written to tensor (or shared) memory from registers, so queries may have any strides.
//
// Every wait on a barrier is bounded; one that runs out raises a flag that all roles observe, the loader waits (bounded)
// for its copies in flight, tensor memory is released and the status bit is set.

#include "common.cuh"
#include "paged.h"
#include "paged_attn.cuh"
#include "tc_common.cuh"

namespace llmcp_b200 {

namespace {

using namespace tc;

constexpr int kRows = 128;
constexpr int kSoftmaxWarps = 8, kMmaWarp = 8, kLoadWarp = 9, kThreads = 384;
// Registers a thread: 168 at launch (all there are for 12 warps), then 208 for the two softmax warpgroups, 88 for the third.
constexpr int kSoftmaxRegisters = 208, kOtherRegisters = 88;
static_assert(2 * kSoftmaxRegisters + kOtherRegisters == 3 * 168, "registers of the block");
constexpr float kHeadroom = 8.0f;

template <int D> struct Shape {
  static constexpr int keys = D == 256 ? 64 : 128; // per tile
  static constexpr int slabs = D / 64;
  static constexpr int slot_bytes = keys * D * 2;
  // Tensor memory: score buffers, O, Q.  Three buffers let a warpgroup begin its next tile before the product of its last
  // one is done; with 256 dimensions there is room for two only, with 128 Q goes to shared memory for the third's sake.
  static constexpr int buffers = D == 256 ? 2 : 3;
  static constexpr bool q_shared = D == 128;
  static constexpr int o_column = buffers * keys, q_column = o_column + D;
  static_assert(q_column + (q_shared ? 0 : D / 2) <= 512, "tensor memory");
  static constexpr int q_bytes = q_shared ? kRows * D * 2 : 0;
  static constexpr int slots = (6 * 32768 - q_bytes) / slot_bytes; // 192 KB: one CTA on an SM, as tensor memory is one CTA's
  static constexpr int q_slot = slots - kRows * D * 2 / slot_bytes; // where Q waits on its way to tensor memory
  static constexpr size_t smem = 1024 + q_bytes + static_cast<size_t>(slots) * slot_bytes;
};

struct Tile {
  PagedKv kv;
  PagedBatch batch;
  PagedAttention call;
  int chunk, chunks, box_rows;
  int tokens_per_tile;
  int64_t expanded_rows; // rows of a sequence's keys in the expanded cache; 0: pages
  int out_of_range;
  uint32_t spin_limit;
};

// D = f32, A and B 16 bits (bf16 or f16), M = 128; B either K-major or MN-major.
template <bool F16, int N, bool MN> constexpr uint32_t kInstruction =
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

// Two f32 values in one register pair.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <int SLOTS> struct Barriers {
  uint64_t full[SLOTS], empty[SLOTS]; // a tile of keys or values
  uint64_t s_full[3];                 // [buffer]: scores of a tile are in tensor memory
  uint64_t p_full[3];                 // its weights are
  uint64_t o_full;                    // every tile's P V has been added
  uint64_t tail_here, tail_ready;     // the last tile of a sequence's values has landed; its rows past the end are zeros
  uint64_t q_full;                    // the queries are
  uint64_t o_done[2];                 // [tile & 1]: P V of a tile has been added
  uint64_t reference[2][4];           // [tile & 1][32 rows]: the reference after a tile
  uint32_t tmem_base;
  int abort_flag;
};

template <int D, bool F16>
__global__ void __launch_bounds__(kThreads, 1)
paged_tile_kernel(const __grid_constant__ CUtensorMap map_values, const __grid_constant__ Tile p, int *__restrict__ status) {
  using S = Shape<D>;
  constexpr int KT = S::keys;
  extern __shared__ uint8_t raw_smem[];
  __shared__ Barriers<S::slots> bars;
  __shared__ float references[kRows], last_reference[2][kRows], sums[2][kRows];
  uint8_t *q_sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  uint8_t *ring = q_sm + S::q_bytes;
  volatile int *abort_flag = &bars.abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.x % p.kv.kv_heads, b = blockIdx.y, chunk_index = blockIdx.z;
  const int q_tile = (gridDim.x - 1 - blockIdx.x) / p.kv.kv_heads; // the longest rows first

  if (tid == 0) {
    for (int i = 0; i < S::slots; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 4);
    }
    mbar_init(&bars.o_full, 1);
    mbar_init(&bars.tail_here, 1);
    mbar_init(&bars.tail_ready, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.o_done[i], 1);
      for (int w = 0; w < 4; ++w)
        mbar_init(&bars.reference[i][w], 1);
    }
    mbar_init(&bars.q_full, kSoftmaxWarps);
    bars.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  grid_dependency_sync();
  const PagedSequence seq = paged_sequence(p.batch, p.kv.page_shift, b, tid == 0 && blockIdx.x == 0 && chunk_index == 0 ? status : nullptr);
  const unsigned group = static_cast<unsigned>(p.call.heads) / static_cast<unsigned>(p.kv.kv_heads);
  const int token0 = q_tile * p.tokens_per_tile, tokens = min(p.tokens_per_tile, seq.count - token0);
  if (tokens <= 0)
    return;
  const int prefix = p.call.prefix ? p.call.prefix[b] : 0;
  // keys below these are seen by the tile's first and last token
  const int sees_least = max(0, min(seq.length, max(seq.length - seq.count + token0 + 1, prefix)));
  const int sees_most = max(0, min(seq.length, max(seq.length - seq.count + token0 + tokens, prefix)));
  const int key0 = chunk_index * p.chunk, key1 = min(sees_most, key0 + p.chunk);
  if (key0 >= key1 && chunk_index > 0)
    return;
  const int tiles = max(0, key1 - key0 + KT - 1) / KT;

  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem_base;

  if (warp >= kSoftmaxWarps) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
  if (warp == kLoadWarp) {
    // ---- loader: the first `ahead` tiles of keys, then values and keys in turn, as the MMAs take them; a box per lane -------------
    const int sub_boxes = KT / p.box_rows, boxes = S::slabs * sub_boxes;
    const int slab = lane / sub_boxes, sub = lane % sub_boxes;
    const int32_t *table = p.batch.page_table + b * p.batch.table_stride;
    const int head_rows = p.kv.kv_heads << p.kv.page_shift;
    const int ahead = min(S::buffers, tiles);
    int issued = 0, keys_issued = 0, values_issued = 0;
    bool ok = true;
    const int items = 2 * tiles;
    for (int n = 0; n < items && ok; ++n) {
      // K0 K1 (K2) V0 K.. V1 K.. ...: keys while fewer than `ahead` tiles lie between them and the values, and while there are any
      const int which = keys_issued < tiles && keys_issued - values_issued < ahead ? 0 : 1;
      const int i = which ? values_issued++ : keys_issued++;
      const int key = key0 + i * KT + sub * p.box_rows;
      int row = p.out_of_range;
      if (lane < boxes && key < seq.length) {
        if (p.expanded_rows) {
          row = static_cast<int>(((static_cast<int64_t>(b) * 2 + which) * p.kv.kv_heads + kvh) * p.expanded_rows + key);
        } else {
          const int page = table[key >> p.kv.page_shift];
          if (page >= 0 && page < p.kv.num_pages)
            row = (page * 2 + which) * head_rows + (kvh << p.kv.page_shift) + (key & ((1 << p.kv.page_shift) - 1));
          else if (status)
            atomicOr(status, kStatusBadBatch);
        }
      }
      const int s = n % S::slots;
      if (!S::q_shared && n == S::q_slot)
        ok = __all_sync(0xffffffffu, mbar_wait<false>(&bars.q_full, 0, abort_flag, p.spin_limit));
      if (ok && n >= S::slots)
        ok = __all_sync(0xffffffffu, mbar_wait<false>(&bars.empty[s], (n / S::slots - 1) & 1, abort_flag, p.spin_limit));
      if (!ok)
        break;
      if (lane == 0)
        mbar_expect_tx(&bars.full[s], S::slot_bytes);
      __syncwarp();
      issued = n + 1;
      if (lane < boxes)
        tma_load_2d(ring + s * S::slot_bytes + (slab * KT + sub * p.box_rows) * 128, &map_values, slab * 64, row, &bars.full[s]);
    }
    if (*abort_flag) // copies already requested still write into this CTA's shared memory
      for (int n = max(0, issued - S::slots); n < issued; ++n)
        mbar_wait_quiet<false>(&bars.full[n % S::slots], (n / S::slots) & 1, p.spin_limit);
  } else if (warp == kMmaWarp) {
    // ---- MMA issue: one thread ---------------------------------------------------------------------------------------------------
    if (elect_one()) {
      auto wait = [&](uint64_t *bar, int parity) { return mbar_wait<false>(bar, parity, abort_flag, p.spin_limit); };
      const uint32_t ring_address = smem_u32(ring);
      const uint64_t q_descriptor = operand_descriptor(smem_u32(q_sm)); // addresses in descriptors count in units of 16 bytes
      int slot = 0, phase = 0, s_buffer = 0;
      auto next_slot = [&]() {
        if (++slot == S::slots) {
          slot = 0;
          phase ^= 1;
        }
      };
      auto scores = [&]() {
        if (!wait(&bars.full[slot], phase))
          return false;
        tc_fence_after();
        const uint64_t k = operand_descriptor(ring_address + slot * S::slot_bytes);
        const uint32_t to = tmem + s_buffer * KT;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          if constexpr (S::q_shared)
            mma_ss(to, q_descriptor + ((n / 4) * (kRows * 128) + (n % 4) * 32) / 16, k + ((n / 4) * (KT * 128) + (n % 4) * 32) / 16, kInstruction<F16, KT, false>, n != 0);
          else
            mma_ts(to, tmem + S::q_column + n * 8, k + ((n / 4) * (KT * 128) + (n % 4) * 32) / 16, kInstruction<F16, KT, false>, n != 0);
        }
        mma_commit(&bars.s_full[s_buffer]);
        mma_commit(&bars.empty[slot]);
        next_slot();
        s_buffer = s_buffer + 1 == S::buffers ? 0 : s_buffer + 1;
        return true;
      };
      bool ok = tiles > 0 && wait(&bars.q_full, 0);
      int scored = 0;
      for (; ok && scored < min(S::buffers, tiles); ++scored) {
        tc_fence_after();
        ok = scores();
      }
      int p_buffer = 0, p_phase = 0;
      for (int i = 0; i < tiles && ok; ++i) {
        ok = wait(&bars.full[slot], phase);
        if (ok && i == tiles - 1 && seq.length - key0 - i * KT < KT) { // rows past the sequence: whatever they hold
          mbar_arrive(&bars.tail_here);
          ok = wait(&bars.tail_ready, 0);
        }
        ok = ok && wait(&bars.p_full[p_buffer], p_phase);
        if (!ok)
          break;
        tc_fence_after();
        const uint64_t v = mn_descriptor(ring_address + slot * S::slot_bytes, KT * 128);
#pragma unroll
        for (int n = 0; n < KT / 16; ++n)
          mma_ts(tmem + S::o_column, tmem + p_buffer * KT + n * 8, v + n * (2048 / 16), kInstruction<F16, D, true>, i != 0 || n != 0);
        mma_commit(&bars.o_done[i & 1]);
        mma_commit(&bars.empty[slot]);
        next_slot();
        if (++p_buffer == S::buffers) {
          p_buffer = 0;
          p_phase ^= 1;
        }
        if (scored < tiles) { // into the buffer that this tile's weights leave: products run in the order of their issue
          ok = scores();
          ++scored;
        }
      }
      if (ok)
        mma_commit(&bars.o_full);
    }
    __syncwarp();
  } else if (warp == kMmaWarp + 2 && tiles > 0) {
    // ---- values of the last tile past the sequence ----------------------------------------------------------------------------------
    const int past = seq.length - key0 - (tiles - 1) * KT;
    if (past < KT && __all_sync(0xffffffffu, mbar_wait(&bars.tail_here, 0, abort_flag, p.spin_limit))) {
      uint8_t *tile = ring + (2 * tiles - 1) % S::slots * S::slot_bytes;
      for (int u = lane; u < KT * 8 * S::slabs; u += 32)
        if (u / 8 % KT >= past)
          *reinterpret_cast<uint4 *>(tile + u * 16) = make_uint4(0, 0, 0, 0);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&bars.tail_ready);
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));
    // ---- softmax: a thread per row -----------------------------------------------------------------------------------------------
    const int half = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const bool valid = row < static_cast<int>(tokens * group);
    const int head0 = kvh * static_cast<int>(group), token_first = seq.first + token0;
    float factor = p.call.scale * (p.call.softcap > 0.0f ? 1.0f : 1.4426950408889634f);
    const bool negative = factor < 0.0f; // goes into the queries: the largest product is the largest score
    const bool flat = factor == 0.0f;    // every score is 0: so are the queries, and the factor stays usable beside -infinity
    factor = flat ? 1.0f : fabsf(factor);
    // Rows come in whole, a lane 16 bytes of one; they go to shared memory as the swizzle has them, K-major slabs of 64
    // dimensions: where the MMAs read them, or in the ring's last slots for the threads that take them to tensor memory.
    constexpr int kLanes = D / 8, kSide = 32 / kLanes;
    uint8_t *staged = S::q_shared ? q_sm : ring + S::q_slot * S::slot_bytes;
    constexpr int kStep = kSoftmaxWarps * kSide, kMine = kRows / kStep; // rows of a lane: all requested at once
    const int piece = lane % kLanes, first_row = warp * kSide + lane / kLanes;
    uint4 pieces[kMine];
#pragma unroll
    for (int n = 0; n < kMine; ++n) {
      const unsigned r = first_row + n * kStep;
      pieces[n] = make_uint4(0, 0, 0, 0);
      if (r < static_cast<unsigned>(tokens * group) && !flat)
        pieces[n] = *reinterpret_cast<const uint4 *>(p.call.q + (token_first + r / group) * p.call.q_row + (head0 + r % group) * p.call.q_head + piece * 8);
    }
#pragma unroll
    for (int n = 0; n < kMine; ++n) {
      const int r = first_row + n * kStep;
      const uint4 v = pieces[n];
      uint32_t w[4] = {v.x, v.y, v.z, v.w};
      if constexpr (F16) { // a power of two per row takes the largest |q| into [2^14, 2^15); keys are 1 / 8 of themselves
        uint32_t top2 = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          top2 = __vmaxu2(top2, w[i] & 0x7fff7fffu);
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1)
          top2 = __vmaxu2(top2, __shfl_xor_sync(0xffffffffu, top2, o));
        const uint32_t top = max(top2 & 0xffffu, top2 >> 16);
        const int up = top == 0 ? 0 : min(126, 14 - (static_cast<int>(top >> 7) - 127));
        const float mult = __uint_as_float(static_cast<uint32_t>(up + 127) << 23 | (negative ? 0x80000000u : 0u));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = pack16<true>(__uint_as_float(w[i] << 16) * mult, __uint_as_float(w[i] & 0xffff0000u) * mult);
        if (piece == 0)
          references[r] = __int_as_float(min(254, 3 - up + 127) << 23);
      } else if (negative) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] ^= 0x80008000u;
      }
      *reinterpret_cast<uint4 *>(staged + (piece / 8) * (kRows * 128) + r * 128 + ((piece % 8 ^ r & 7) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if constexpr (S::q_shared)
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("bar.sync 1, 256;" ::: "memory"); // the softmax warps
    if constexpr (F16)
      factor *= references[row];
    if constexpr (!S::q_shared) {
#pragma unroll
      for (int c = 0; c < D / 2 / 32; ++c) { // 32 dimensions = 16 columns at a time; half of them each
        const int d = half * (D / 2) + c * 32;
        uint32_t w[16];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint4 v = *reinterpret_cast<const uint4 *>(staged + (d / 64) * (kRows * 128) + row * 128 + ((d % 64 / 8 + k ^ row & 7) << 4));
          w[4 * k] = v.x, w[4 * k + 1] = v.y, w[4 * k + 2] = v.z, w[4 * k + 3] = v.w;
        }
        tmem_store16(lanes + S::q_column + d / 2, w);
      }
      tmem_wait_stores();
      tc_fence_before();
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the loader's copies into these slots come after
    }
    __syncwarp();
    if (lane == 0)
      mbar_arrive(&bars.q_full);
    if constexpr (F16)
      asm volatile("bar.sync 1, 256;" ::: "memory"); // the factors have been read: their place is the references' now

    const int position = seq.length - seq.count + token0 + static_cast<int>(row / group);
    const int sees = valid ? max(0, min(seq.length, max(position + 1, prefix))) : 0;
    const float cap = p.call.softcap, over_cap = cap > 0.0f ? 1.0f / cap : 0.0f;
    const bool biased = p.call.slopes != nullptr;
    const float slope = biased && valid ? p.call.slopes[head0 + row % group] * 1.4426950408889634f : 0.0f, at = static_cast<float>(position);
    float reference = -INFINITY, sum = 0.0f;
    auto o_wait = [&](int i) { return __all_sync(0xffffffffu, mbar_wait<false>(&bars.o_done[i & 1], (i >> 1) & 1, abort_flag, p.spin_limit)); };
    bool ok = true;
    int buffer = half, buffer_phase = 0; // tile i is in buffer i % buffers
    for (int i = half; i < tiles; i += 2) {
      const int j0 = key0 + i * KT;
      ok = __all_sync(0xffffffffu, mbar_wait<false>(&bars.s_full[buffer], buffer_phase, abort_flag, p.spin_limit));
      if (!ok)
        break;
      tc_fence_after();
      const uint32_t s_at = lanes + buffer * KT;
      uint32_t x[KT / 32][32];
#pragma unroll
      for (int c = 0; c < KT / 32; ++c)
        tmem_issue32(s_at + c * 32, x[c]);
#pragma unroll
      for (int c = 0; c < KT / 32; ++c)
        tmem_wait_loads_into(x[c]);
      float scaled = factor;
      if (cap > 0.0f) {
#pragma unroll
        for (int c = 0; c < KT / 32; ++c)
#pragma unroll
          for (int u = 0; u < 32; ++u)
            x[c][u] = __float_as_uint(capped_log2(__uint_as_float(x[c][u]) * factor, cap, over_cap));
        scaled = 1.0f;
      }
      if (biased) {
#pragma unroll
        for (int c = 0; c < KT / 32; ++c)
#pragma unroll
          for (int u = 0; u < 32; ++u)
            x[c][u] = __float_as_uint(__uint_as_float(x[c][u]) * scaled - slope * fabsf(at - static_cast<float>(j0 + c * 32 + u)));
        scaled = 1.0f;
      }
      if (j0 + KT > sees_least) {
#pragma unroll
        for (int c = 0; c < KT / 32; ++c)
#pragma unroll
          for (int u = 0; u < 32; ++u)
            if (j0 + c * 32 + u >= sees)
              x[c][u] = 0xff800000u;
      }
      float most[8]; // side by side: one chain of maxima would take as long as everything else
#pragma unroll
      for (int u = 0; u < 8; ++u)
        most[u] = -INFINITY;
#pragma unroll
      for (int c = 0; c < KT / 32; ++c)
#pragma unroll
        for (int u = 0; u < 32; ++u)
          most[u & 7] = fmaxf(most[u & 7], __uint_as_float(x[c][u]));
      float best = fmaxf(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])), fmaxf(fmaxf(most[4], most[5]), fmaxf(most[6], most[7])));
      best = best == -INFINITY ? best : best * scaled;
      // the reference after the tile in front
      float before = -INFINITY;
      if (i > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait<false>(&bars.reference[half ^ 1][quarter], ((i - 1) >> 1) & 1, abort_flag, p.spin_limit));
        if (!ok)
          break;
        before = references[row];
      }
      const float now = best > before + kHeadroom ? best : before;
      references[row] = now;
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&bars.reference[half][quarter]);
      if (now != reference) { // moved by this tile or the one in front
        sum *= reference == -INFINITY ? 0.0f : exp2_approx(reference - now);
        reference = now;
      }
      if (__any_sync(0xffffffffu, now != before) && i > 0) {
        // O holds every tile up to i - 1 once the product of that one is done.  (A wait by parity tells a phase from its
        // neighbours only: the one before, tile i - 3, is done, or the scores of this one would not be there.)
        ok = o_wait(i - 1);
        if (!ok)
          break;
        tc_fence_after();
        const float moved = now == before ? 1.0f : before == -INFINITY ? 0.0f : exp2_approx(before - now);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_load32(lanes + S::o_column + c * 32, o);
#pragma unroll
          for (int u = 0; u < 32; ++u)
            o[u] = __float_as_uint(moved == 0.0f ? 0.0f : __uint_as_float(o[u]) * moved);
          tmem_store32(lanes + S::o_column + c * 32, o);
        }
        tmem_wait_stores();
      }
      // f16 weights lie between 2^7 (a row's largest, at least) and 2^15, and keep their precision down to 2^-14
      const float minus = (now == -INFINITY ? 0.0f : -now) + (F16 ? 15.0f - kHeadroom : 0.0f);
      uint64_t added[4] = {0, 0, 0, 0}; // pairs of sums
      const uint64_t scaled2 = pair(scaled, scaled), minus2 = pair(minus, minus);
#pragma unroll
      for (int c = 0; c < KT / 32; ++c) {
        uint32_t w[16];
#pragma unroll
        for (int u = 0; u < 32; u += 2) {
          const float2 y = halves(fma2(pair(__uint_as_float(x[c][u]), __uint_as_float(x[c][u + 1])), scaled2, minus2));
          const float p0 = exp2_approx(y.x), p1 = exp2_approx(y.y);
          added[u >> 1 & 3] = add2(added[u >> 1 & 3], pair(p0, p1));
          w[u >> 1] = pack16<F16>(p0, p1);
        }
        tmem_store16(s_at + c * 16, w);
      }
      const float2 added2 = halves(add2(add2(added[0], added[1]), add2(added[2], added[3])));
      sum += added2.x + added2.y;
      tmem_wait_stores();
      tc_fence_before();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&bars.p_full[buffer]);
      buffer += 2;
      if (buffer >= S::buffers) {
        buffer -= S::buffers;
        buffer_phase ^= 1;
      }
    }
    // ---- epilogue: the two halves' sums, then half of the dimensions each -----------------------------------------------------------
    last_reference[half][row] = reference;
    sums[half][row] = sum;
    asm volatile("bar.sync 1, 256;" ::: "memory"); // the softmax warps
    if (p.call.gate && p.chunks == 1) { // on their way while the last products run
#pragma unroll
      for (int n = 0; n < kMine; ++n) {
        const unsigned r = first_row + n * kStep;
        if (r < static_cast<unsigned>(tokens * group))
          pieces[n] = paged_gate<D>(p.call, token_first + r / group, head0 + r % group, piece * 8);
      }
    }
    if (ok && tiles > 0)
      ok = __all_sync(0xffffffffu, mbar_wait<false>(&bars.o_full, 0, abort_flag, p.spin_limit));
    if (ok) {
      tc_fence_after();
      const float final_reference = tiles > 0 ? references[row] : -INFINITY;
      float total = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        total += last_reference[h][row] == -INFINITY ? 0.0f : sums[h][row] * exp2_approx(last_reference[h][row] - final_reference);
      // rows of O by thread into shared memory (the ring is done with), then whole rows out
      constexpr int kPitch = D + 4;
      float *rows_out = reinterpret_cast<float *>(ring);
      // values are 1 / 8 of themselves in f16; where a row has seen nothing O may hold anything
      const float unscale = (F16 ? 8.0f : 1.0f) * (total == 0.0f ? 0.0f : p.chunks == 1 ? __fdiv_rn(1.0f, total) : 1.0f);
#pragma unroll 1
      for (int c = 0; c < D / 2 / 32; ++c) {
        const int d = half * (D / 2) + c * 32;
        uint32_t o[32];
        __syncwarp();
        tmem_load32(lanes + S::o_column + d, o);
#pragma unroll
        for (int u = 0; u < 32; u += 4) {
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (total != 0.0f)
            v = make_float4(__uint_as_float(o[u]) * unscale, __uint_as_float(o[u + 1]) * unscale, __uint_as_float(o[u + 2]) * unscale,
                            __uint_as_float(o[u + 3]) * unscale);
          *reinterpret_cast<float4 *>(rows_out + row * kPitch + d + u) = v;
        }
      }
      if (p.chunks > 1 && half == 0 && valid)
        paged_store_sums<D>(p.call, p.batch.tokens, p.chunks, chunk_index, token_first + row / group, head0 + row % group, final_reference, total);
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (ok) {
      const float *rows_out = reinterpret_cast<const float *>(ring);
#pragma unroll
      for (int n = 0; n < kMine; ++n) {
        const unsigned r = first_row + n * kStep;
        if (r >= static_cast<unsigned>(tokens * group))
          break;
        const int d = piece * 8, token = token_first + r / group, head = head0 + r % group;
        const float4 x = *reinterpret_cast<const float4 *>(rows_out + r * (D + 4) + d), y = *reinterpret_cast<const float4 *>(rows_out + r * (D + 4) + d + 4);
        if (p.chunks == 1)
          paged_store_row<D>(p.call, token, head, d, x, y, pieces[n]);
        else
          paged_store_part<D>(p.call, p.chunks, chunk_index, token, head, d, x, y);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
  if (tid == 0 && bars.abort_flag && status)
    atomicOr(status, kStatusWaitRanOut);
}

// A 4-bit cache's rows of the batch's sequences as f16 / 8: [sequence][keys, values][kv head][rows][D], zeros from a
// sequence's length to the end of its last tile.  A warp takes a row of a head's keys or values per lane group.
template <int D>
__global__ void __launch_bounds__(256)
paged_expand_kernel(PagedKv kv, PagedBatch batch, uint4 *__restrict__ out, int64_t rows, int *__restrict__ status) {
  constexpr int kLanes = D / 32; // a block of 32 dimensions (16 bytes of codes) per thread
  grid_dependency_sync();
  const int b = blockIdx.z, which = blockIdx.y / kv.kv_heads, head = blockIdx.y % kv.kv_heads;
  const PagedSequence s = paged_sequence(batch, kv.page_shift, b, nullptr);
  if (s.count == 0)
    return;
  const int padded = (s.length + 127) / 128 * 128;
  for (int64_t u = blockIdx.x * static_cast<int64_t>(256) + threadIdx.x; u < static_cast<int64_t>(padded) * kLanes; u += static_cast<int64_t>(gridDim.x) * 256) {
    const int key = static_cast<int>(u / kLanes), block = static_cast<int>(u % kLanes);
    uint4 codes = make_uint4(0, 0, 0, 0);
    uint32_t scale = 0;
    if (key < s.length) {
      const int64_t row = paged_row(kv, batch, b, key, which, head);
      if (row >= 0) {
        codes = *reinterpret_cast<const uint4 *>(kv.pages + row * (D / 2) + block * 16);
        scale = kv.scales[row * (D / 32) + block];
      } else if (status) {
        atomicOr(status, kStatusBadBatch);
      }
    }
    uint32_t d2; // scale / 8 twice
    const uint32_t pair = scale | scale << 16, eighth = 0x30003000u;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d2) : "r"(pair), "r"(eighth));
    const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
    uint4 *dst = out + (((static_cast<int64_t>(b) * 2 + which) * kv.kv_heads + head) * rows + key) * (D / 8) + block * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // code + 8 in the low bits of 1024, 1024 off again: exact; nibbles n and n + 4 come together
      uint32_t v[4], r[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint32_t biased = (w[i] >> (4 * n) & 0x000f000fu) | 0x64006400u, offset = 0x64086408u;
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(v[n]) : "r"(biased), "r"(offset));
        asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(v[n]) : "r"(v[n]), "r"(d2));
      }
      r[0] = __byte_perm(v[0], v[1], 0x5410), r[1] = __byte_perm(v[2], v[3], 0x5410);
      r[2] = __byte_perm(v[0], v[1], 0x7632), r[3] = __byte_perm(v[2], v[3], 0x7632);
      dst[i] = make_uint4(r[0], r[1], r[2], r[3]);
    }
  }
}

int64_t expanded_rows(const PagedBatch &batch) { return (static_cast<int64_t>(batch.max_kv) + 127) / 128 * 128; }

size_t expanded_bytes(const PagedKv &kv, const PagedBatch &batch) {
  return kv.scales ? static_cast<size_t>(batch.sequences) * 2 * kv.kv_heads * expanded_rows(batch) * kv.head_dim * 2 : 0;
}

template <int D, bool F16>
cudaError_t launch(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, const PagedSplit &split, int *status, cudaStream_t stream) {
  using S = Shape<D>;
  const int group = call.heads / kv.kv_heads;
  Tile p;
  p.kv = kv, p.batch = batch, p.call = call;
  p.chunk = split.chunk, p.chunks = split.chunks;
  p.tokens_per_tile = kRows / group;
  p.spin_limit = kSpinLimit<false>;
  const int page = 1 << kv.page_shift;
  PagedKv source = kv;
  int64_t rows = kv.num_pages * 2 * kv.kv_heads << kv.page_shift;
  p.expanded_rows = 0;
  p.box_rows = S::keys < page ? S::keys : page;
  if (F16) {
    p.expanded_rows = expanded_rows(batch);
    p.box_rows = S::keys;
    rows = static_cast<int64_t>(batch.sequences) * 2 * kv.kv_heads * p.expanded_rows;
    if (rows > (int64_t(1) << 31) - 1)
      return cudaErrorInvalidValue;
    source.pages = static_cast<uint8_t *>(call.workspace) + (paged_parts_bytes(kv, batch, call.heads, split) + 255) / 256 * 256;
    source.scales = nullptr;
    const int64_t blocks = (p.expanded_rows * (D / 32) + 255) / 256;
    if (cudaError_t e = launch_chained(paged_expand_kernel<D>, dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096), 2 * kv.kv_heads, batch.sequences), dim3(256), 0,
                                       stream, kv, batch, reinterpret_cast<uint4 *>(source.pages), p.expanded_rows, status);
        e != cudaSuccess)
      return e;
  }
  p.out_of_range = static_cast<int>(rows);
  CUtensorMap values;
  if (!paged_value_map(&values, source, rows, p.box_rows))
    return cudaErrorNotSupported;
  const auto kernel = paged_tile_kernel<D, F16>;
  if (cudaError_t e = opt_in_shared_memory(reinterpret_cast<const void *>(kernel), S::smem); e != cudaSuccess)
    return e;
  const unsigned q_tiles = static_cast<unsigned>((batch.max_q + p.tokens_per_tile - 1) / p.tokens_per_tile);
  return launch_chained(kernel, dim3(kv.kv_heads * q_tiles, batch.sequences, split.chunks), dim3(kThreads), S::smem, stream, values, p, status);
}

} // namespace

size_t paged_tile_workspace(const PagedKv &kv, const PagedBatch &batch, int heads, const PagedSplit &split) {
  return (paged_parts_bytes(kv, batch, heads, split) + 255) / 256 * 256 + expanded_bytes(kv, batch);
}

PagedSplit paged_tile_split(const PagedKv &kv, const PagedBatch &batch, int heads, int sms) {
  const int tokens_per_tile = kRows / (heads / kv.kv_heads);
  const int64_t ctas = static_cast<int64_t>((batch.max_q + tokens_per_tile - 1) / tokens_per_tile) * kv.kv_heads * batch.sequences;
  const int64_t tile = kv.head_dim == 256 ? 64 : 128, tiles = (batch.max_kv + tile - 1) / tile;
  // pieces of at least four tiles, as many as fill the SMs once
  int64_t pieces = sms / ctas;
  pieces = pieces > tiles / 4 ? tiles / 4 : pieces;
  pieces = pieces > kMaxChunks ? kMaxChunks : pieces;
  if (pieces <= 1)
    return PagedSplit{batch.max_kv > 0 ? static_cast<int>(tiles * tile) : 1, 1};
  const int64_t each = (tiles + pieces - 1) / pieces;
  return PagedSplit{static_cast<int>(each * tile), static_cast<int>((tiles + each - 1) / each)};
}

cudaError_t launch_paged_tile(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, const PagedSplit &split, int *status,
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
