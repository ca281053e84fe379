// Attention over the paged cache for many rows (prompts), 256 dimensions: both products on tcgen05.  (64 and 128 dimensions:
// paged_attn_narrow.cu, launched from here.)
//
//   S = Q K^T,  P = 2^(S scale log2 e - m),  O = sum P V / sum P,   128 rows (tokens x the query heads of one key head) a CTA
//
// Keys and values come as 16-bit tiles by TMA: bf16 straight from the pages; a 4-bit cache is expanded once per call into
// f16 rows (paged_expand_kernel), value = code * scale rounded to f16, because every tile of rows would otherwise unpack the
// same keys again.  The rounding is 2^-11 for every scale, f16's subnormal ones too: a whole number of its steps stays one.
// A sequence's head whose largest scale is 8192 or more (7 times that may leave f16) has its codes divided by 8 (exactly),
// and its factors are that much larger; what a small block beside such a large one loses then is 2^-22, 2^-37 of the
// largest value.  paged_largest_scale_kernel finds those.
//
// One CTA, 352 threads, all 512 columns of tensor memory (O 256, Q 128, two tiles of 64 scores):
//   warps 0-7  softmax, a thread per row: warps 0-3 take the even key tiles, 4-7 the odd ones.  A thread reads its scores
//              from tensor memory, writes P over them and, when its row's reference moves, rescales its row of O there.
//              The reference (a score that none has outgrown by more than 2^8) passes from tile to tile, between the two
//              warps that share 32 rows, through shared memory; the exponentials of two tiles run side by side.
//   warp 8     one thread issues the MMAs: Q and P from tensor memory, K (K-major) and V (MN-major: rows are keys) from
//              shared memory, both with the 128-byte swizzle.  Scores are issued two tiles ahead of P V.
//   warps 9, 10  issue the TMA loads of keys (and queries and gates) and of values into a ring of tiles, in the order in
//              which the MMAs take them: K0 K1 V0 K2 V1 ...  Warp 10 zeroes the rows of the last value tile that lie past
//              the sequence, too: 0 times whatever they hold is not 0.
// Queries come in as whole rows through ring slots that are not in use yet, results leave as whole rows through the ring.
//
// A key tile is 1024 cycles of products beside a softmax of about 1300; the gates' sigmoids and the results take 7 thousand
// cycles a CTA.  4 prompts of 1024 to 2048 tokens of 16 heads, gated: 119 us in a captured graph, 740 TFLOP/s (141 us with one
// loading warp), 132 to 134 us as a call among others.
//
// Every wait on a barrier is bounded; one that runs out raises a flag that all roles observe, the loader waits (bounded)
// for its copies in flight, tensor memory is released and the status bit is set.

#include "paged_attn_tc.cuh"

namespace llmcp_b200 {

namespace {

using namespace tc;

constexpr int D = 256;
constexpr int KT = 64; // keys per tile
constexpr int kSlabs = D / 64, kSlotBytes = KT * D * 2, kSlots = 6;
constexpr int kQSlot = kSlots - kRows * D * 2 / kSlotBytes; // where Q waits on its way to tensor memory
constexpr size_t kSmem = 1024 + static_cast<size_t>(kSlots) * kSlotBytes;
// Tensor memory, in columns: two score buffers, O, Q.
constexpr int kOColumn = 2 * KT, kQColumn = kOColumn + D;
static_assert(kQColumn + D / 2 <= 512, "tensor memory");
constexpr int kSoftmaxWarps = 8, kMmaWarp = 8, kLoadWarp = 9, kValueWarp = 10, kThreads = 352;

struct Barriers {
  uint64_t full[kSlots], empty[kSlots]; // a tile of keys or values
  uint64_t s_full[2];                 // [buffer]: scores of a tile are in tensor memory
  uint64_t p_full[2];                 // its weights are
  uint64_t o_full;                    // every tile's P V has been added
  uint64_t tail_here, tail_ready;     // the last tile of a sequence's values has landed; its rows past the end are zeros
  uint64_t q_here;                    // the queries (and the divisors) have landed
  uint64_t q_full;                    // ... and are in tensor memory
  uint64_t o_done[2];                 // [tile & 1]: P V of a tile has been added
  uint64_t reference[2][4];           // [tile & 1][32 rows]: the reference after a tile
  uint32_t tmem_base;
  int abort_flag;
  float divisors[2];                  // of the expanded keys and values
};

template <bool F16>
__global__ void __launch_bounds__(kThreads, 1)
paged_tile_kernel(const __grid_constant__ CUtensorMap map_values, const __grid_constant__ RowMaps maps, const __grid_constant__ Tile p, int *__restrict__ status) {
  extern __shared__ uint8_t raw_smem[];
  __shared__ Barriers bars;
  __shared__ float references[kRows], last_reference[2][kRows], sums[2][kRows];
  uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  volatile int *abort_flag = &bars.abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kvh = blockIdx.x % p.kv.kv_heads, b = blockIdx.y, chunk_index = blockIdx.z;
  const int q_tile = (gridDim.x - 1 - blockIdx.x) / p.kv.kv_heads; // the longest rows first

  if (tid == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1);
    }
    mbar_init(&bars.o_full, 1);
    mbar_init(&bars.tail_here, 1);
    mbar_init(&bars.tail_ready, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 4);
      mbar_init(&bars.o_done[i], 1);
      for (int w = 0; w < 4; ++w)
        mbar_init(&bars.reference[i][w], 1);
    }
    mbar_init(&bars.q_here, F16 ? 2 : 1);
    mbar_init(&bars.q_full, kSoftmaxWarps);
    bars.abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  grid_dependency_sync();
  const PagedSequence seq = paged_sequence(p.batch, p.kv.page_shift, b, tid == 0 && blockIdx.x == 0 && chunk_index == 0 ? status : nullptr);
  const unsigned group = p.group;
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

  // ---- loaders: a warp for the keys, one for the values; K0 K1 V0 K2 V1 ... as the MMAs take them, a box per lane ------------------
  int issued = -1; // this warp's last item of the ring
  // Parity tells a phase from its neighbours only; the one before is over: for a warp's own items because it waited for them,
  // for the last values (in a slot of keys) and the gates because the items before them have been there.
  auto slot_free = [&](int n, bool others) {
    bool ok = true;
    if (others) // these slots may still hold the queries
      ok = __all_sync(0xffffffffu, mbar_wait<false>(&bars.q_full, 0, abort_flag, p.spin_limit));
    if (ok && n >= kSlots)
      ok = __all_sync(0xffffffffu, mbar_wait<false>(&bars.empty[n % kSlots], (n / kSlots - 1) & 1, abort_flag, p.spin_limit));
    return ok;
  };
  auto load_tiles = [&](int which) {
    const int sub_boxes = KT / p.box_rows;
    const int slab = lane / sub_boxes, sub = lane % sub_boxes;
    const int32_t *table = p.batch.page_table + b * p.batch.table_stride;
    bool ok = true;
    for (int i = 0; i < tiles && ok; ++i) {
      const int n = which ? (i == tiles - 1 ? 2 * tiles - 1 : 2 * i + 2) : max(0, 2 * i - 1);
      const int row = tile_box_row(p, seq, table, b, kvh, which, key0 + i * KT + sub * p.box_rows, slab < kSlabs, status);
      ok = slot_free(n, n >= kQSlot && n < kSlots);
      if (!ok)
        break;
      const int s = n % kSlots;
      if (lane == 0)
        mbar_expect_tx(&bars.full[s], kSlotBytes);
      __syncwarp();
      issued = n;
      if (slab < kSlabs)
        tma_load_2d(ring + s * kSlotBytes + (slab * KT + sub * p.box_rows) * 128, &map_values, slab * 64, row, &bars.full[s]);
    }
    return ok;
  };
  auto wait_for_copies = [&]() { // after an abort: they still write into this CTA's shared memory
    for (int n = max(0, issued - kSlots + 1); n <= issued; ++n)
      mbar_wait_quiet<false>(&bars.full[n % kSlots], (n / kSlots) & 1, p.spin_limit);
  };

  if (warp == kLoadWarp) {
    const int slab_bytes = p.tokens_per_tile * p.group * 128, token_first = seq.first + token0, head0 = kvh * p.group;
    if (lane == 0) {
      mbar_expect_tx(&bars.q_here, kSlabs * slab_bytes);
      for (int k = 0; k < kSlabs; ++k)
        load_slab(ring + kQSlot * kSlotBytes + k * (kRows * 128), &maps.queries, k * 64, head0, token_first, &bars.q_here);
    }
    bool ok = load_tiles(0);
    if (p.call.gate && p.chunks == 1)
      for (int half = 0; half < 2 && ok; ++half) { // the gates are the last two items: half of the dimensions each
        const int n = 2 * tiles + half, s = n % kSlots;
        ok = slot_free(n, half == 0);
        if (!ok)
          break;
        if (lane == 0)
          mbar_expect_tx(&bars.full[s], kSlabs / 2 * slab_bytes);
        __syncwarp();
        issued = n;
        if (lane < kSlabs / 2)
          load_slab(ring + s * kSlotBytes + lane * (kRows * 128), &maps.gates, half * (D / 2) + lane * 64, head0, token_first, &bars.full[s]);
      }
    if (*abort_flag) {
      mbar_wait_quiet<false>(&bars.q_here, 0, p.spin_limit);
      wait_for_copies();
    }
  } else if (warp == kMmaWarp) {
    // ---- MMA issue: one thread ---------------------------------------------------------------------------------------------------
    if (elect_one()) {
      auto wait = [&](uint64_t *bar, int parity) { return mbar_wait<false>(bar, parity, abort_flag, p.spin_limit); };
      const uint32_t ring_address = smem_u32(ring);
      int slot = 0, phase = 0, scored = 0;
      auto next_slot = [&]() {
        if (++slot == kSlots) {
          slot = 0;
          phase ^= 1;
        }
      };
      auto scores = [&]() {
        tc_fence_after();
        const uint64_t k = operand_descriptor(ring_address + slot * kSlotBytes); // addresses count in units of 16 bytes
#pragma unroll
        for (int n = 0; n < D / 16; ++n)
          mma_ts(tmem + (scored & 1) * KT, tmem + kQColumn + n * 8, k + ((n / 4) * (KT * 128) + (n % 4) * 32) / 16, kInstruction<F16, KT, false>, n != 0);
        mma_commit(&bars.s_full[scored & 1]);
        mma_commit(&bars.empty[slot]);
        next_slot();
        ++scored;
      };
      bool ok = tiles > 0 && wait(&bars.q_full, 0);
      while (ok && scored < min(2, tiles)) {
        ok = wait(&bars.full[slot], phase);
        if (ok)
          scores();
      }
      for (int i = 0; i < tiles && ok; ++i) {
        ok = wait_for_both(&bars.full[slot], phase, &bars.p_full[i & 1], (i >> 1) & 1, abort_flag, p.spin_limit);
        if (ok && i == tiles - 1 && seq.length - key0 - i * KT < KT) { // rows past the sequence: whatever they hold
          mbar_arrive(&bars.tail_here);
          ok = wait(&bars.tail_ready, 0);
        }
        if (!ok)
          break;
        tc_fence_after();
        const uint64_t v = mn_descriptor(ring_address + slot * kSlotBytes, KT * 128);
#pragma unroll
        for (int n = 0; n < KT / 16; ++n)
          mma_ts(tmem + kOColumn, tmem + (i & 1) * KT + n * 8, v + n * (2048 / 16), kInstruction<F16, D, true>, i != 0 || n != 0);
        mma_commit(&bars.o_done[i & 1]);
        mma_commit(&bars.empty[slot]);
        next_slot();
        if (scored < tiles) { // into the buffer that this tile's weights leave: products run in the order of their issue
          ok = wait(&bars.full[slot], phase);
          if (ok)
            scores();
        }
      }
      if (ok)
        mma_commit(&bars.o_full);
    }
    __syncwarp();
  } else if (warp == kValueWarp) {
    if constexpr (F16)
      fetch_divisors(bars.divisors, p, b, kvh, lane, &bars.q_here);
    load_tiles(1);
    const int past = seq.length - key0 - (tiles - 1) * KT;
    if (tiles > 0 && past < KT && __all_sync(0xffffffffu, mbar_wait<false>(&bars.tail_here, 0, abort_flag, p.spin_limit))) {
      zero_tail<KT, kSlabs>(ring + (2 * tiles - 1) % kSlots * kSlotBytes, past, lane);
      if (lane == 0)
        mbar_arrive(&bars.tail_ready);
    }
    if (*abort_flag)
      wait_for_copies();
  } else {
    // ---- softmax: a thread per row -----------------------------------------------------------------------------------------------
    const int half = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const unsigned rows = tokens * group;
    const bool valid = row < static_cast<int>(rows);
    const int head0 = kvh * static_cast<int>(group), token_first = seq.first + token0;
    float factor = p.call.scale * (p.call.softcap > 0.0f ? 1.0f : 1.4426950408889634f);
    const bool negative = factor < 0.0f; // goes into the queries: the largest product is the largest score
    const bool flat = factor == 0.0f;    // every score is 0: so are the queries, and the factor stays usable beside -infinity
    factor = flat ? 1.0f : fabsf(factor);
    const uint8_t *staged = ring + kQSlot * kSlotBytes; // the loader leaves these slots until the queries have gone on
    auto all_wait = [&](uint64_t *bar, int parity) { return __all_sync(0xffffffffu, mbar_wait<false>(bar, parity, abort_flag, p.spin_limit)); };
    bool ok = all_wait(&bars.q_here, 0);
    float multiplier = 1.0f, unscale = 1.0f;
    if constexpr (F16)
      multiplier = query_multiplier<D>(staged, row, negative, &unscale);
    factor *= F16 ? unscale * bars.divisors[0] : 1.0f;
#pragma unroll 1
    for (int c = half * (D / 64); c < (half + 1) * (D / 64); ++c) { // 32 dimensions = 16 columns at a time; half of them each
      uint32_t w[16];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 v = query_piece<F16>(*reinterpret_cast<const uint4 *>(staged + piece_at(row, c * 4 + k)), multiplier, negative, flat);
        w[4 * k] = v.x, w[4 * k + 1] = v.y, w[4 * k + 2] = v.z, w[4 * k + 3] = v.w;
      }
      tmem_store16(lanes + kQColumn + c * 16, w);
    }
    tmem_wait_stores();
    tc_fence_before();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // the loader's copies into these slots come after
    __syncwarp();
    if (lane == 0)
      mbar_arrive(&bars.q_full);

    RowScores r;
    const int position = seq.length - seq.count + token0 + static_cast<int>(row / group);
    r.factor = factor;
    r.cap = p.call.softcap, r.over_cap = r.cap > 0.0f ? 1.0f / r.cap : 0.0f;
    r.biased = p.call.slopes != nullptr;
    r.slope = r.biased && valid ? p.call.slopes[head0 + row % group] * 1.4426950408889634f : 0.0f, r.at = position;
    r.sees = valid ? max(0, min(seq.length, max(position + 1, prefix))) : 0, r.sees_least = sees_least;
    float reference = -INFINITY, sum = 0.0f;
    for (int i = half; i < tiles && ok; i += 2) {
      ok = all_wait(&bars.s_full[half], (i >> 1) & 1);
      if (!ok)
        break;
      tc_fence_after();
      uint32_t x[KT / 32][32];
      load_scores<KT>(x, lanes + half * KT);
      const float scaled = shape_scores<KT>(x, r, key0 + i * KT);
      const float best = largest_score<KT>(x, scaled);
      // the reference after the tile in front
      float before = -INFINITY;
      if (i > 0) {
        ok = all_wait(&bars.reference[half ^ 1][quarter], ((i - 1) >> 1) & 1);
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
        ok = all_wait(&bars.o_done[(i - 1) & 1], ((i - 1) >> 1) & 1);
        if (!ok)
          break;
        tc_fence_after();
        rescale_row<D>(lanes + kOColumn, now == before ? 1.0f : before == -INFINITY ? 0.0f : exp2_approx(before - now));
      }
      sum += store_weights<KT, F16, 0>(x, lanes + half * KT, scaled, now);
      tc_fence_before();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&bars.p_full[half]);
    }
    // ---- epilogue: the two halves' sums, then half of the dimensions each -----------------------------------------------------------
    last_reference[half][row] = reference;
    sums[half][row] = sum;
    // Gates, then results, lie in the two slots after the ring's last item, a half's in its own: what was in them six items
    // before was done with before the last scores that either half has seen.
    const TileRows mine{rows, group, p.one_over_group, token_first, head0};
    const int place = 2 * tiles + half;
    uint8_t *rows_out = ring + place % kSlots * kSlotBytes;
    const bool gated = p.call.gate && p.chunks == 1;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (ok && gated)
      ok = all_wait(&bars.full[place % kSlots], (place / kSlots) & 1);
    if (ok && tiles > 0)
      ok = all_wait(&bars.o_full, 0);
    if (ok) {
      tc_fence_after();
      const float final_reference = tiles > 0 ? references[row] : -INFINITY;
      float total = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        total += last_reference[h][row] == -INFINITY ? 0.0f : sums[h][row] * exp2_approx(last_reference[h][row] - final_reference);
      // where a row has seen nothing O may hold anything
      const float scale = (F16 ? bars.divisors[1] : 1.0f) * (p.chunks == 1 && total != 0.0f ? __fdiv_rn(1.0f, total) : 1.0f);
      const uint32_t o_at = lanes + kOColumn + half * (D / 2);
      if (p.chunks == 1) {
        unload_row<D / 2>(rows_out, row, o_at, scale, total == 0.0f, gated);
      } else {
        const int64_t part = (mine.at(row, p.call.heads, 1) * p.chunks + chunk_index) * D + half * (D / 2);
        unload_part<D / 2>(static_cast<float *>(p.call.workspace) + (valid ? part : 0), o_at, scale, total == 0.0f, valid);
        if (half == 0 && valid)
          paged_store_sums<D>(p.call, p.batch.tokens, p.chunks, chunk_index, token_first + row / group, head0 + row % group, final_reference, total);
      }
    }
    if (half == 0)
      asm volatile("bar.sync 2, 128;" ::: "memory");
    else
      asm volatile("bar.sync 3, 128;" ::: "memory");
    if (ok && p.chunks == 1)
      copy_rows_out<D / 2, 4>(p.call.out + half * (D / 2), static_cast<int64_t>(p.call.heads) * D, D, rows_out, mine, quarter, lane);
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

// The largest scale (its bits) of every sequence's keys and values by head, in `gridDim.x` parts: [sequence][keys, values]
// [kv head][kScaleParts].
constexpr int kScaleParts = 32;

template <int DIM>
__global__ void __launch_bounds__(256)
paged_largest_scale_kernel(PagedKv kv, PagedBatch batch, uint32_t *__restrict__ out) {
  constexpr int kWords = DIM / 64, kAhead = 4; // two scales to a word; a key per thread, four at a time
  __shared__ uint32_t tops[8];
  grid_dependency_sync();
  const int b = blockIdx.z, which = blockIdx.y / kv.kv_heads, head = blockIdx.y % kv.kv_heads;
  const PagedSequence s = paged_sequence(batch, kv.page_shift, b, nullptr);
  if (s.count == 0)
    return;
  const uint32_t *scales = reinterpret_cast<const uint32_t *>(kv.scales);
  const int step = gridDim.x * 256;
  uint32_t top = 0;
  for (int first = blockIdx.x * 256 + threadIdx.x; first < s.length; first += kAhead * step) {
    int64_t row[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
      row[a] = first + a * step < s.length ? paged_row(kv, batch, b, first + a * step, which, head) : -1;
    uint32_t words[kAhead][kWords];
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int k = 0; k < kWords; ++k)
        words[a][k] = row[a] >= 0 ? scales[row[a] * kWords + k] : 0;
#pragma unroll
    for (int a = 0; a < kAhead; ++a)
#pragma unroll
      for (int k = 0; k < kWords; ++k)
        top = __vmaxu2(top, words[a][k] & 0x7fff7fffu);
  }
  top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
  if (threadIdx.x % 32 == 0)
    tops[threadIdx.x / 32] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w)
      top = max(top, tops[w]);
    out[((static_cast<int64_t>(b) * 2 + which) * kv.kv_heads + head) * kScaleParts + blockIdx.x] = top;
  }
}

// A 4-bit cache's rows of the batch's sequences as f16: [sequence][keys, values][kv head][rows][D], zeros from a
// sequence's length to the end of its last tile; an eighth of the values where the head's largest scale needs it.
// 16000 rows of 8 heads of 128: 21 us, of 13 that its bytes take, after 6 us for the largest scales.
template <int DIM>
__global__ void __launch_bounds__(256)
paged_expand_kernel(PagedKv kv, PagedBatch batch, uint4 *__restrict__ out, int64_t rows, const uint32_t *largest, int parts,
                    float *__restrict__ divisors, int *__restrict__ status) {
  constexpr int kLanes = DIM / 8, kAhead = 4; // eight dimensions (4 bytes of codes, 16 bytes out) per thread, of four keys at a time
  grid_dependency_sync();
  const int b = blockIdx.z, which = blockIdx.y / kv.kv_heads, head = blockIdx.y % kv.kv_heads;
  const PagedSequence s = paged_sequence(batch, kv.page_shift, b, nullptr);
  if (s.count == 0)
    return;
  const int64_t of_head = (static_cast<int64_t>(b) * 2 + which) * kv.kv_heads + head;
  const int lane = threadIdx.x & 31;
  const bool large = __reduce_max_sync(0xffffffffu, lane < parts ? largest[of_head * kScaleParts + lane] : 0) >= 0x7000; // 8192
  if (blockIdx.x == 0 && threadIdx.x == 0)
    divisors[of_head] = large ? 8.0f : 1.0f;
  // code + 8 in the low bits of 1024, 1032 off again: exact; in those of 128 it is an eighth
  const uint32_t base = large ? 0x58005800u : 0x64006400u, offset = base | 0x00080008u;
  const int padded = (s.length + 127) / 128 * 128;
  const int piece = threadIdx.x % kLanes, step = gridDim.x * (256 / kLanes);
  uint4 *to = out + of_head * rows * kLanes + piece;
  const uint8_t *from = kv.pages + piece * 4;
  const uint16_t *scales = kv.scales + piece / 4;
  for (int first = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes; first < padded; first += kAhead * step) {
    uint32_t codes[kAhead], scale[kAhead];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int key = first + a * step;
      codes[a] = scale[a] = 0;
      if (key < s.length) {
        const int64_t row = paged_row(kv, batch, b, key, which, head);
        if (row >= 0) {
          codes[a] = *reinterpret_cast<const uint32_t *>(from + row * (DIM / 2));
          scale[a] = scales[row * (DIM / 32)];
        } else if (status) {
          atomicOr(status, kStatusBadBatch);
        }
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const int key = first + a * step;
      if (key >= padded)
        break;
      const uint32_t d2 = scale[a] | scale[a] << 16;
      uint32_t v[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const uint32_t biased = (codes[a] >> (4 * n) & 0x000f000fu) | base; // nibbles n and n + 4 come together
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(v[n]) : "r"(biased), "r"(offset));
        asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(v[n]) : "r"(v[n]), "r"(d2));
      }
      to[static_cast<int64_t>(key) * kLanes] = make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632));
    }
  }
}

// Tiles of a sequence's rows.
int64_t row_tiles(const PagedBatch &batch, int per_tile) { return (static_cast<int64_t>(batch.max_q) + per_tile - 1) / per_tile; }

int64_t expanded_rows(const PagedBatch &batch) { return (static_cast<int64_t>(batch.max_kv) + 127) / 128 * 128; }

size_t expanded_bytes(const PagedKv &kv, const PagedBatch &batch) {
  return kv.scales ? static_cast<size_t>(batch.sequences) * 2 * kv.kv_heads * expanded_rows(batch) * kv.head_dim * 2 : 0;
}

// Behind them: the largest scales' parts, and the divisors.
int64_t expanded_heads(const PagedKv &kv, const PagedBatch &batch) { return kv.scales && batch.max_kv > 0 ? static_cast<int64_t>(batch.sequences) * 2 * kv.kv_heads : 0; }

// The expanded copy in the workspace.
template <int DIM>
cudaError_t expand(const PagedKv &kv, const PagedBatch &batch, uint8_t *to, uint32_t *largest, float *divisors, int *status, cudaStream_t stream) {
  const int64_t rows = expanded_rows(batch), blocks = (rows * (DIM / 8) + 1023) / 1024; // a turn of the kernel's loop each
  const unsigned heads = 2 * kv.kv_heads, sequences = batch.sequences;
  const int parts = static_cast<int>(rows > kScaleParts * 1024 ? kScaleParts : (rows + 1023) / 1024); // likewise
  if (cudaError_t e = launch_chained(paged_largest_scale_kernel<DIM>, dim3(parts, heads, sequences), dim3(256), 0, stream, kv, batch, largest); e != cudaSuccess)
    return e;
  return launch_chained(paged_expand_kernel<DIM>, dim3(static_cast<unsigned>(blocks < 4096 ? blocks : 4096), heads, sequences), dim3(256), 0, stream,
                        kv, batch, reinterpret_cast<uint4 *>(to), rows, largest, parts, divisors, status);
}

template <bool F16> cudaError_t launch_wide(const CUtensorMap &values, const RowMaps &maps, const Tile &p, unsigned q_tiles, int *status, cudaStream_t stream) {
  const auto kernel = paged_tile_kernel<F16>;
  if (cudaError_t e = opt_in_shared_memory(reinterpret_cast<const void *>(kernel), kSmem); e != cudaSuccess)
    return e;
  return launch_chained(kernel, dim3(p.kv.kv_heads * q_tiles, p.batch.sequences, p.chunks), dim3(kThreads), kSmem, stream, values, maps, p, status);
}

} // namespace

size_t paged_tile_workspace(const PagedKv &kv, const PagedBatch &batch, int heads, const PagedSplit &split) {
  return (paged_parts_bytes(kv, batch, heads, split) + 255) / 256 * 256 + expanded_bytes(kv, batch) +
         expanded_heads(kv, batch) * (kScaleParts + 1) * sizeof(uint32_t);
}

PagedSplit paged_tile_split(const PagedKv &kv, const PagedBatch &batch, int heads, int sms) {
  const int64_t ctas = row_tiles(batch, kRows / (heads / kv.kv_heads)) * kv.kv_heads * batch.sequences;
  const int64_t tiles = (batch.max_kv + KT - 1) / KT;
  // Pieces of at least four tiles, as many as the SMs take at a time.  64 rows of 16 heads of 256 over 4000 keys: 28 us with
  // eight tiles and more, 23 with four, 23 with two; 60 of 32 heads of 128 over 1000, twice: 21, 16, 19.  Of at least eight
  // where a piece's sums take more than 4 MB to write and read again: 512 of 32 heads of 128, 20 us with four, 15 with eight.
  const int64_t least = static_cast<int64_t>(batch.tokens) * heads * kv.head_dim * 4 > 4 << 20 ? 8 : 4;
  int64_t pieces = static_cast<int64_t>(sms) * (kv.head_dim == D ? 1 : 2) / ctas;
  pieces = pieces > tiles / least ? tiles / least : pieces;
  pieces = pieces > kMaxChunks ? kMaxChunks : pieces;
  if (pieces <= 1)
    return PagedSplit{batch.max_kv > 0 ? static_cast<int>(tiles * KT) : 1, 1};
  const int64_t each = (tiles + pieces - 1) / pieces;
  return PagedSplit{static_cast<int>(each * KT), static_cast<int>((tiles + each - 1) / each)};
}

cudaError_t launch_paged_tile(const PagedKv &kv, const PagedBatch &batch, const PagedAttention &call, const PagedSplit &split, int *status,
                              cudaStream_t stream) {
  const bool f16 = kv.scales != nullptr;
  Tile p;
  p.kv = kv, p.batch = batch, p.call = call;
  p.chunk = split.chunk, p.chunks = split.chunks;
  p.group = call.heads / kv.kv_heads, p.one_over_group = (65536 + p.group - 1) / p.group;
  p.tokens_per_tile = kRows / p.group;
  p.spin_limit = kSpinLimit<false>;
  p.expanded_rows = 0;
  p.divisors = nullptr;
  p.box_rows = KT < 1 << kv.page_shift ? KT : 1 << kv.page_shift;
  PagedKv source = kv;
  int64_t rows = kv.num_pages * 2 * kv.kv_heads << kv.page_shift;
  if (f16) {
    p.box_rows = KT;
    source.scales = nullptr;
    rows = 1; // without keys nothing is expanded, and no tile comes through the map
  }
  if (f16 && batch.max_kv > 0) {
    p.expanded_rows = expanded_rows(batch);
    rows = static_cast<int64_t>(batch.sequences) * 2 * kv.kv_heads * p.expanded_rows; // the entry has seen that they are less than 2^31
    source.pages = static_cast<uint8_t *>(call.workspace) + (paged_parts_bytes(kv, batch, call.heads, split) + 255) / 256 * 256;
    uint32_t *largest = reinterpret_cast<uint32_t *>(source.pages + expanded_bytes(kv, batch));
    float *divisors = reinterpret_cast<float *>(largest + expanded_heads(kv, batch) * kScaleParts);
    p.divisors = divisors;
    const auto run = kv.head_dim == 64 ? expand<64> : kv.head_dim == 128 ? expand<128> : expand<256>;
    if (const cudaError_t e = run(kv, batch, source.pages, largest, divisors, status, stream); e != cudaSuccess)
      return e;
  }
  p.out_of_range = static_cast<int>(rows);
  CUtensorMap values;
  if (!paged_value_map(&values, source, rows, p.box_rows))
    return cudaErrorNotSupported;
  RowMaps maps;
  if (!paged_rows_map(&maps.queries, call.q, kv.head_dim, call.heads, batch.tokens, call.q_head, call.q_row, p.group, p.tokens_per_tile))
    return cudaErrorNotSupported;
  maps.gates = maps.queries;
  if (call.gate && !paged_rows_map(&maps.gates, call.gate, kv.head_dim, call.heads, batch.tokens, call.gate_head, call.gate_row, p.group, p.tokens_per_tile))
    return cudaErrorNotSupported;
  const unsigned q_tiles = static_cast<unsigned>(row_tiles(batch, p.tokens_per_tile));
  if (kv.head_dim != D)
    return launch_paged_narrow(kv.head_dim, f16, values, maps, p, q_tiles, status, stream);
  return f16 ? launch_wide<true>(values, maps, p, q_tiles, status, stream) : launch_wide<false>(values, maps, p, q_tiles, status, stream);
}

} // namespace llmcp_b200
