// Attention over the paged cache for many rows (prompts), 64 and 128 dimensions: as paged_attn_tile.cu, but O leaves room in
// tensor memory, so two CTAs share an SM: while one loads, waits or writes, the other computes.  Each has 128 rows, a
// thread per row, two buffers of 64 scores and O in 256 columns, the queries in shared memory.  (One CTA with two tiles of
// rows that share the keys measured the same on long prompts and 15 % longer on short ones, where its longest tile
// decides.)
//
// A tile of 64 keys costs 512 cycles of exponentials (16 a cycle, less what the multipliers take over) and, at 128
// dimensions, 640 cycles of products: the scores' operands both come from shared memory, 128 bytes a cycle.
//
//   warps 0-3  softmax;  4  MMA issue (one thread);  5  TMA loads of queries, keys and gates;  6  of values, the last of which
//              it gives zeros past the sequence.  (An item costs its warp some 1100 cycles, the wait for its slot and the
//              issue of its boxes among them: one warp for both bound every tile.)
//
// 1024 tokens over 7000 keys in 4 bits, twice, 32 heads of 128: 276 us in a captured graph, 910 TFLOP/s, 29 us of it the
// expansion; 295 to 302 us as a call among others.  3 x up to 1501 tokens of 8 heads of 64, capped: 46 us a call, of
// which the longest rows' 25 tiles of 2000 cycles and a CTA's start and end account for some 31.  A row's scores over two threads (eight softmax
// warps) measured 5 % (64) to 15 % (128) slower.

#include "paged_attn_tc.cuh"

namespace llmcp_b200 {

namespace {

using namespace tc;

constexpr int KT = 64;

constexpr int kMmaWarp = 4, kLoadWarp = 5, kValueWarp = 6, kThreads = 224;

template <int D> struct Shape {
  static constexpr int slabs = D / 64;
  static constexpr int slot_bytes = KT * D * 2;
  static constexpr int q_bytes = kRows * D * 2;
  static constexpr int slots = D == 128 ? 4 : 8; // 64 KB
  static constexpr int o_column = 2 * KT;        // tensor memory: two score buffers, O
  static_assert(o_column + D <= 256, "tensor memory of one of two CTAs");
  static constexpr size_t smem = 1024 + q_bytes + slots * slot_bytes;
};

template <int SLOTS> struct Barriers {
  uint64_t full[SLOTS], empty[SLOTS]; // a tile of keys or values
  uint64_t q_here;                    // the queries (and the divisors) have landed
  uint64_t q_full;                    // ... and are as the products take them
  uint64_t gates_here;
  uint64_t s_full[2];                 // [key tile & 1]: scores are in tensor memory
  uint64_t p_full[2];                 // their weights are
  uint64_t o_done[2];                 // P V has been added
  uint64_t o_full;                    // all of it
  uint64_t tail_here, tail_ready;     // the last tile of a sequence's values has landed; its rows past the end are zeros
  uint32_t tmem_base;
  int abort_flag;
  float divisors[2];                  // of the expanded keys and values
};

template <int D, bool F16>
__global__ void __launch_bounds__(kThreads, 2)
paged_narrow_kernel(const __grid_constant__ CUtensorMap map_values, const __grid_constant__ RowMaps maps, const __grid_constant__ Tile p, int *__restrict__ status) {
  using S = Shape<D>;
  extern __shared__ uint8_t raw_smem[];
  __shared__ Barriers<S::slots> bars;
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
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_full[i], 4);
      mbar_init(&bars.o_done[i], 1);
    }
    mbar_init(&bars.q_here, F16 ? 2 : 1);
    mbar_init(&bars.q_full, 4);
    mbar_init(&bars.gates_here, 1);
    mbar_init(&bars.o_full, 1);
    mbar_init(&bars.tail_here, 1);
    mbar_init(&bars.tail_ready, 1);
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
  const int key0 = chunk_index * p.chunk, tiles = max(0, min(sees_most, key0 + p.chunk) - key0 + KT - 1) / KT;
  if (tiles == 0 && chunk_index > 0)
    return;

  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars.tmem_base)), "r"(256) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem_base;

  // ---- loaders: a warp for the keys, one for the values; K0 K1 V0 K2 V1 ... as the MMAs take them, a box per lane ------------------
  int issued = -1; // this warp's last item of the ring
  auto load_tiles = [&](int which) {
    const int sub_boxes = KT / p.box_rows;
    const int slab = lane / sub_boxes, sub = lane % sub_boxes;
    const int32_t *table = p.batch.page_table + b * p.batch.table_stride;
    bool ok = true;
    for (int i = 0; i < tiles; ++i) {
      const int n = which ? (i == tiles - 1 ? 2 * tiles - 1 : 2 * i + 2) : max(0, 2 * i - 1);
      const int row = tile_box_row(p, seq, table, b, kvh, which, key0 + i * KT + sub * p.box_rows, slab < S::slabs, status);
      const int s = n % S::slots;
      // Parity tells a phase from its neighbours only; the one before is over: for a warp's own items because it waited for
      // them, for the last values (in a slot of keys) because those before them have been there.
      if (n >= S::slots)
        ok = __all_sync(0xffffffffu, mbar_wait<false>(&bars.empty[s], (n / S::slots - 1) & 1, abort_flag, p.spin_limit));
      if (!ok)
        break;
      if (lane == 0)
        mbar_expect_tx(&bars.full[s], S::slot_bytes);
      __syncwarp();
      issued = n;
      if (slab < S::slabs)
        tma_load_2d(ring + s * S::slot_bytes + (slab * KT + sub * p.box_rows) * 128, &map_values, slab * 64, row, &bars.full[s]);
    }
    return ok;
  };
  auto wait_for_copies = [&]() { // after an abort: they still write into this CTA's shared memory
    for (int n = max(0, issued - S::slots + 1); n <= issued; ++n)
      mbar_wait_quiet<false>(&bars.full[n % S::slots], (n / S::slots) & 1, p.spin_limit);
  };

  if (warp == kLoadWarp) {
    const int slab_bytes = p.tokens_per_tile * p.group * 128, token_first = seq.first + token0, head0 = kvh * p.group;
    if (lane == 0) {
      mbar_expect_tx(&bars.q_here, S::slabs * slab_bytes);
      for (int k = 0; k < S::slabs; ++k)
        load_slab(q_sm + k * (kRows * 128), &maps.queries, k * 64, head0, token_first, &bars.q_here);
    }
    const bool ok = load_tiles(0);
    // the gates take the queries' place, once the last keys' product is done (or nobody has wanted them)
    bool gates = false;
    if (ok && p.call.gate && p.chunks == 1) {
      const int last = tiles == 1 ? 0 : 2 * tiles - 3; // the ring's item
      gates = __all_sync(0xffffffffu, tiles > 0 ? mbar_wait<false>(&bars.empty[last % S::slots], (last / S::slots) & 1, abort_flag, p.spin_limit)
                                                 : mbar_wait<false>(&bars.q_full, 0, abort_flag, p.spin_limit));
      if (gates && lane == 0) {
        mbar_expect_tx(&bars.gates_here, S::slabs * slab_bytes);
        for (int k = 0; k < S::slabs; ++k)
          load_slab(q_sm + k * (kRows * 128), &maps.gates, k * 64, head0, token_first, &bars.gates_here);
      }
    }
    if (*abort_flag) { // copies already requested still write into this CTA's shared memory
      mbar_wait_quiet<false>(&bars.q_here, 0, p.spin_limit);
      if (gates)
        mbar_wait_quiet<false>(&bars.gates_here, 0, p.spin_limit);
      wait_for_copies();
    }
  } else if (warp == kMmaWarp) {
    // ---- MMA issue: one thread ---------------------------------------------------------------------------------------------------
    if (elect_one()) {
      auto wait = [&](uint64_t *bar, int parity) { return mbar_wait<false>(bar, parity, abort_flag, p.spin_limit); };
      const uint64_t k0 = operand_descriptor(smem_u32(ring)), v0 = mn_descriptor(smem_u32(ring), KT * 128); // addresses in descriptors
      const uint64_t q_descriptor = operand_descriptor(smem_u32(q_sm));                                     // count in units of 16 bytes
      int slot = 0, phase = 0;
      auto next_slot = [&]() {
        mma_commit(&bars.empty[slot]);
        if (++slot == S::slots) {
          slot = 0;
          phase ^= 1;
        }
      };
      auto scores = [&](int i) {
        tc_fence_after();
        const uint64_t k = k0 + static_cast<uint32_t>(slot) * (S::slot_bytes / 16);
#pragma unroll
        for (int n = 0; n < D / 16; ++n)
          mma_ss(tmem + (i & 1) * KT, q_descriptor + ((n / 4) * (kRows * 128) + (n % 4) * 32) / 16, k + ((n / 4) * (KT * 128) + (n % 4) * 32) / 16,
                 kInstruction<F16, KT, false>, n != 0);
        mma_commit(&bars.s_full[i & 1]);
        next_slot();
      };
      bool ok = tiles > 0 && wait(&bars.q_full, 0);
      for (int i = 0; i < min(2, tiles) && ok; ++i) {
        ok = wait(&bars.full[slot], phase);
        if (ok)
          scores(i);
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
        const uint64_t v = v0 + static_cast<uint32_t>(slot) * (S::slot_bytes / 16);
#pragma unroll
        for (int n = 0; n < KT / 16; ++n)
          mma_ts(tmem + S::o_column, tmem + (i & 1) * KT + n * 8, v + n * (2048 / 16), kInstruction<F16, D, true>, i != 0 || n != 0);
        mma_commit(&bars.o_done[i & 1]);
        next_slot();
        if (i + 2 < tiles) { // into the buffer that these weights leave: products run in the order of their issue
          ok = wait(&bars.full[slot], phase);
          if (ok)
            scores(i + 2);
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
      zero_tail<KT, S::slabs>(ring + (2 * tiles - 1) % S::slots * S::slot_bytes, past, lane);
      if (lane == 0)
        mbar_arrive(&bars.tail_ready);
    }
    if (*abort_flag)
      wait_for_copies();
  } else {
    // ---- softmax: a thread per row -----------------------------------------------------------------------------------------------
    const int row = warp * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const unsigned rows = tokens * group;
    const bool valid = row < static_cast<int>(rows);
    const int head0 = kvh * static_cast<int>(group), token_first = seq.first + token0;
    RowScores r;
    r.factor = p.call.scale * (p.call.softcap > 0.0f ? 1.0f : 1.4426950408889634f);
    const bool negative = r.factor < 0.0f; // goes into the queries: the largest product is the largest score
    const bool flat = r.factor == 0.0f;    // every score is 0: so are the queries, and the factor stays usable beside -infinity
    r.factor = flat ? 1.0f : fabsf(r.factor);
    auto all_wait = [&](uint64_t *bar, int parity) { return __all_sync(0xffffffffu, mbar_wait<false>(bar, parity, abort_flag, p.spin_limit)); };
    bool ok = all_wait(&bars.q_here, 0);
    if (F16 || negative || flat) { // in place, a row per thread
      float multiplier = 1.0f, unscale = 1.0f;
      if constexpr (F16)
        multiplier = query_multiplier<D>(q_sm, row, negative, &unscale);
      r.factor *= F16 ? unscale * bars.divisors[0] : 1.0f;
#pragma unroll 2
      for (int piece = 0; piece < D / 8; ++piece) {
        uint4 *at = reinterpret_cast<uint4 *>(q_sm + piece_at(row, piece));
        *at = query_piece<F16>(*at, multiplier, negative, flat);
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // visible to the tensor core's reads
    __syncwarp();
    if (lane == 0)
      mbar_arrive(&bars.q_full);
    const int position = seq.length - seq.count + token0 + static_cast<int>(row / group);
    r.cap = p.call.softcap, r.over_cap = r.cap > 0.0f ? 1.0f / r.cap : 0.0f;
    r.biased = p.call.slopes != nullptr;
    r.slope = r.biased && valid ? p.call.slopes[head0 + row % group] * 1.4426950408889634f : 0.0f, r.at = position;
    r.sees = valid ? max(0, min(seq.length, max(position + 1, prefix))) : 0, r.sees_least = sees_least;
    float reference = -INFINITY, sum = 0.0f;
    for (int i = 0; i < tiles && ok; ++i) {
      ok = all_wait(&bars.s_full[i & 1], (i >> 1) & 1);
      if (!ok)
        break;
      tc_fence_after();
      const uint32_t s_at = lanes + (i & 1) * KT;
      uint32_t x[KT / 32][32];
      load_scores<KT>(x, s_at);
      const float scaled = shape_scores<KT>(x, r, key0 + i * KT);
      const float best = largest_score<KT>(x, scaled);
      if (__any_sync(0xffffffffu, best > reference + kHeadroom)) {
        const float now = best > reference + kHeadroom ? best : reference;
        const float moved = now == reference ? 1.0f : reference == -INFINITY ? 0.0f : exp2_approx(reference - now);
        sum *= moved;
        if (i > 0) {
          // O holds every tile up to i - 1 once the product of that one is done.  (A wait by parity tells a phase from its
          // neighbours only: the one before, tile i - 3, is done, or the scores of this one would not be there.)
          ok = all_wait(&bars.o_done[(i - 1) & 1], ((i - 1) >> 1) & 1);
          if (!ok)
            break;
          tc_fence_after();
          rescale_row<D>(lanes + S::o_column, moved);
        }
        reference = now;
      }
      // a masked score is -infinity, whose weight has to be 0
      sum += key0 + i * KT + KT > r.sees_least ? store_weights<KT, F16, 0>(x, s_at, scaled, reference) : store_weights<KT, F16, 2>(x, s_at, scaled, reference);
      tc_fence_before();
      __syncwarp();
      if (lane == 0)
        mbar_arrive(&bars.p_full[i & 1]);
    }
    // ---- epilogue -------------------------------------------------------------------------------------------------------------------
    // Gates, then results, lie in the queries' place.
    const TileRows mine{rows, group, p.one_over_group, token_first, head0};
    const bool gated = p.call.gate && p.chunks == 1;
    if (ok && gated)
      ok = all_wait(&bars.gates_here, 0);
    if (ok && tiles > 0)
      ok = all_wait(&bars.o_full, 0);
    if (ok) {
      tc_fence_after();
      // where a row has seen nothing O may hold anything
      const float scale = (F16 ? bars.divisors[1] : 1.0f) * (p.chunks == 1 && sum != 0.0f ? __fdiv_rn(1.0f, sum) : 1.0f);
      if (p.chunks == 1) {
        unload_row<D>(q_sm, row, lanes + S::o_column, scale, sum == 0.0f, gated);
      } else {
        const int64_t part = (mine.at(row, p.call.heads, 1) * p.chunks + chunk_index) * D;
        unload_part<D>(static_cast<float *>(p.call.workspace) + (valid ? part : 0), lanes + S::o_column, scale, sum == 0.0f, valid);
        if (valid)
          paged_store_sums<D>(p.call, p.batch.tokens, p.chunks, chunk_index, token_first + row / group, head0 + row % group, reference, sum);
      }
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (ok && p.chunks == 1)
      copy_rows_out<D, 4>(p.call.out, static_cast<int64_t>(p.call.heads) * D, D, q_sm, mine, warp, lane);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256) : "memory");
  }
  if (tid == 0 && bars.abort_flag && status)
    atomicOr(status, kStatusWaitRanOut);
}

template <int D, bool F16> cudaError_t launch(const CUtensorMap &values, const RowMaps &maps, const Tile &p, unsigned q_tiles, int *status, cudaStream_t stream) {
  const auto kernel = paged_narrow_kernel<D, F16>;
  if (cudaError_t e = opt_in_shared_memory(reinterpret_cast<const void *>(kernel), Shape<D>::smem); e != cudaSuccess)
    return e;
  return launch_chained(kernel, dim3(p.kv.kv_heads * q_tiles, p.batch.sequences, p.chunks), dim3(kThreads), Shape<D>::smem, stream, values, maps, p, status);
}

} // namespace

cudaError_t launch_paged_narrow(int head_dim, bool f16, const CUtensorMap &values, const RowMaps &maps, const Tile &p, unsigned q_tiles, int *status, cudaStream_t stream) {
  if (head_dim == 64)
    return f16 ? launch<64, true>(values, maps, p, q_tiles, status, stream) : launch<64, false>(values, maps, p, q_tiles, status, stream);
  return f16 ? launch<128, true>(values, maps, p, q_tiles, status, stream) : launch<128, false>(values, maps, p, q_tiles, status, stream);
}

} // namespace llmcp_b200
