// C entry points of the paged key/value cache: every argument is checked here, before anything touches the GPU.

#include <algorithm>
#include <cmath>
#include <stdexcept>
#include <string>

#include "../../include/llmcp_b200.h"
#include "common.cuh"
#include "paged.h"

namespace llmcp_b200 {
void report_error(const std::string &message); // api.cu
void count_launches(uint64_t launches);
} // namespace llmcp_b200

using namespace llmcp_b200;

namespace {

void require(bool ok, const char *what) {
  if (!ok)
    throw std::runtime_error(std::string("paged cache: ") + what);
}

bool on(const void *p, size_t boundary) { return reinterpret_cast<uintptr_t>(p) % boundary == 0; }

PagedKv to_kv(const llmcp_b200_paged_kv *kv) {
  require(kv && kv->pages, "the cache has no pages");
  require(kv->head_dim == 64 || kv->head_dim == 128 || kv->head_dim == 256, "head_dim has to be 64, 128 or 256");
  require(kv->page_size >= 16 && kv->page_size <= 256 && (kv->page_size & (kv->page_size - 1)) == 0,
          "page_size has to be 16, 32, 64, 128 or 256");
  require(kv->kv_heads >= 1 && kv->kv_heads <= 1024, "kv_heads has to be 1 to 1024");
  // rows of all pages are numbered in 31 bits by the copies
  require(kv->num_pages >= 1 && kv->num_pages <= ((int64_t(1) << 31) - 1) / (2 * kv->kv_heads * kv->page_size),
          "num_pages has to be at least 1, with fewer than 2^31 rows in all");
  require(on(kv->pages, 16) && on(kv->scales, 16), "pages and scales have to start on a 16-byte boundary");
  int shift = 4;
  while ((1 << shift) < kv->page_size)
    ++shift;
  return PagedKv{static_cast<uint8_t *>(kv->pages), kv->scales, kv->num_pages, shift, static_cast<int>(kv->kv_heads),
                 static_cast<int>(kv->head_dim)};
}

PagedBatch to_batch(const llmcp_b200_paged_batch *b, const PagedKv &kv) {
  require(b != nullptr, "no batch");
  constexpr int64_t most = int64_t(1) << 30; // arithmetic on positions and tiles stays in 31 bits
  require(b->sequences >= 0 && b->sequences <= 65535, "sequences has to be 0 to 65535");
  require(b->tokens >= 0 && b->tokens <= most && b->max_q >= 0 && b->max_q <= most && b->max_kv >= 0 && b->max_kv <= most,
          "tokens, max_q and max_kv have to be 0 to 2^30");
  require(b->table_width >= 0 && b->table_width <= most && (b->table_stride >= b->table_width || b->sequences <= 1),
          "a row of the page table has table_width entries, rows lie table_stride apart");
  require(b->sequences == 0 || b->tokens == 0 || (b->q_start && b->kv_len && (b->page_table || b->table_width == 0)),
          "q_start, kv_len or page_table is missing");
  PagedBatch out;
  out.q_start = b->q_start;
  out.kv_len = b->kv_len;
  out.page_table = b->page_table;
  out.table_stride = b->table_stride;
  out.sequences = static_cast<int>(b->sequences);
  out.table_width = static_cast<int>(b->table_width);
  out.tokens = static_cast<int>(b->tokens);
  // no sequence has more rows than the call, or more keys than its pages hold: wider bounds would only lay out empty work, or
  // choose the kernel for rows that are not there
  out.max_q = static_cast<int>(std::min(b->max_q, b->tokens));
  out.max_kv = static_cast<int>(std::min(b->max_kv, b->table_width << kv.page_shift));
  return out;
}

bool nothing(const PagedBatch &b) { return b.sequences == 0 || b.tokens == 0 || b.max_q == 0; }

void check(cudaError_t e, const char *what) {
  if (e != cudaSuccess) {
    cudaGetLastError();
    throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
  }
}

template <typename F> int entry(F &&body) {
  try {
    body();
    return 0;
  } catch (const std::exception &e) {
    report_error(e.what());
    return 1;
  }
}

} // namespace

extern "C" int llmcp_dev_paged_append(const llmcp_b200_paged_kv *kv, const llmcp_b200_paged_batch *batch, const uint16_t *q, int64_t q_row,
                                      int64_t q_head, int64_t heads, const uint16_t *k, int64_t k_row, int64_t k_head, const uint16_t *v,
                                      int64_t v_row, int64_t v_head, const uint16_t *q_norm, const uint16_t *k_norm, float eps,
                                      const float *cos, const float *sin, int64_t cos_rows, int64_t rot, uint16_t *q_out, int *status,
                                      void *stream) {
  return entry([&] {
    const PagedKv c = to_kv(kv);
    const PagedBatch b = to_batch(batch, c);
    require(heads >= 0 && heads <= 16384, "heads has to be 0 to 16384");
    require(rot >= 0 && rot <= c.head_dim && rot % (c.head_dim / 16) == 0, "rot has to be a multiple of head_dim / 16, at most head_dim");
    require(cos_rows >= 0, "cos_rows is negative");
    require(eps >= 0.0f && std::isfinite(eps), "eps has to be finite and not negative");
    if (nothing(b))
      return;
    require(heads == 0 || (q && q_out), "q or q_out is missing");
    require(k && v, "k or v is missing");
    require(rot == 0 || (cos && sin), "cos or sin is missing");
    require(on(q, 2) && on(k, 2) && on(v, 2) && on(q_norm, 2) && on(k_norm, 2) && on(cos, 4) && on(sin, 4) && on(q_out, 16),
            "q_out has to start on a 16-byte boundary, every other tensor on one of its elements");
    PagedAppend a = {};
    a.q = q, a.k = k, a.v = v;
    a.q_row = q_row, a.q_head = q_head, a.k_row = k_row, a.k_head = k_head, a.v_row = v_row, a.v_head = v_head;
    a.q_norm = q_norm, a.k_norm = k_norm, a.eps = eps;
    a.cos = cos, a.sin = sin, a.cos_rows = cos_rows;
    a.heads = static_cast<int>(heads), a.rot = static_cast<int>(rot);
    a.q_out = q_out;
    int sms = 0;
    check(current_sm_count(&sms), "paged append");
    check(launch_paged_append(c, b, a, status, sms, static_cast<cudaStream_t>(stream)), "paged append");
    count_launches(1);
  });
}

extern "C" int llmcp_dev_paged_read(const llmcp_b200_paged_kv *kv, const llmcp_b200_paged_batch *batch, void *k_out, void *v_out,
                                    int out_dtype, int *status, void *stream) {
  return entry([&] {
    const PagedKv c = to_kv(kv);
    const PagedBatch b = to_batch(batch, c);
    require(out_dtype == kF32 || out_dtype == kBF16, "out_dtype has to be 0 (f32) or 1 (bf16)");
    if (nothing(b))
      return;
    require(k_out && v_out && on(k_out, 16) && on(v_out, 16), "k_out and v_out have to start on a 16-byte boundary");
    int sms = 0;
    check(current_sm_count(&sms), "paged read");
    check(launch_paged_read(c, b, k_out, v_out, out_dtype, status, sms, static_cast<cudaStream_t>(stream)), "paged read");
    count_launches(1);
  });
}

namespace {
int checked_heads(const PagedKv &c, const PagedBatch &b, int64_t max_q, int64_t heads) {
  require(heads >= 1 && heads <= 16384 && heads % c.kv_heads == 0, "heads has to be a multiple of kv_heads, at most 16384");
  require(heads / c.kv_heads <= 128, "at most 128 query heads share a key head");
  // prompts over 4 bits work on rows of 16 bits, numbered in 31 bits too
  require(!c.scales || max_q * (heads / c.kv_heads) <= 16 ||
              static_cast<int64_t>(b.sequences) * 2 * c.kv_heads * ((b.max_kv + int64_t(127)) / 128 * 128) < (int64_t(1) << 31),
          "sequences * 2 * kv_heads * max_kv has to stay below 2^31 for prompts over 4 bits; make several calls");
  return static_cast<int>(heads);
}
} // namespace

extern "C" int64_t llmcp_dev_paged_attention_workspace(const llmcp_b200_paged_kv *kv, const llmcp_b200_paged_batch *batch, int64_t heads) {
  int64_t bytes = -1;
  entry([&] {
    const PagedKv c = to_kv(kv);
    const PagedBatch b = to_batch(batch, c);
    const int h = checked_heads(c, b, batch->max_q, heads);
    if (nothing(b)) {
      bytes = 0;
      return;
    }
    int sms = 0;
    check(current_sm_count(&sms), "paged attention workspace");
    bytes = static_cast<int64_t>(paged_attention_workspace(c, b, h, sms));
  });
  return bytes;
}

extern "C" int llmcp_dev_paged_attention(const llmcp_b200_paged_kv *kv, const llmcp_b200_paged_batch *batch, const uint16_t *q, int64_t q_row,
                                         int64_t q_head, int64_t heads, float scale, float softcap, const float *slopes,
                                         const int32_t *prefix, const uint16_t *gate, int64_t gate_row, int64_t gate_head, uint16_t *out,
                                         void *workspace, int64_t workspace_bytes, int *status, void *stream) {
  return entry([&] {
    const PagedKv c = to_kv(kv);
    const PagedBatch b = to_batch(batch, c);
    const int h = checked_heads(c, b, batch->max_q, heads);
    require(std::isfinite(scale) && std::isfinite(softcap) && softcap >= 0.0f, "scale and softcap have to be finite, softcap not negative");
    if (nothing(b))
      return;
    require(q && out, "q or out is missing");
    // the stride of a dimension with one entry means nothing
    if (b.tokens == 1)
      q_row = gate_row = int64_t(8);
    if (h == 1)
      q_head = gate_head = int64_t(8);
    require(on(q, 16) && q_row % 8 == 0 && q_head % 8 == 0 && on(out, 16) && on(gate, 16) && (!gate || (gate_row % 8 == 0 && gate_head % 8 == 0)),
            "rows of q, gate and out have to start on 16-byte boundaries");
    require(q_row > 0 && q_head > 0 && (!gate || (gate_row > 0 && gate_head > 0)), "strides of q and gate have to be positive");
    require(on(slopes, 4) && on(prefix, 4), "slopes and prefix have to start on one of their elements");
    int sms = 0;
    check(current_sm_count(&sms), "paged attention");
    const size_t need = paged_attention_workspace(c, b, h, sms);
    require(need == 0 || (workspace && on(workspace, 16) && workspace_bytes >= 0 && static_cast<size_t>(workspace_bytes) >= need),
            "the workspace is smaller than llmcp_dev_paged_attention_workspace says, or off a 16-byte boundary");
    PagedAttention a = {};
    a.q = q, a.q_row = q_row, a.q_head = q_head, a.heads = h;
    // A cap whose ratio to a score (or its reciprocal) could leave f32: above 2^64 it changes nothing that f32 scores show, and
    // below 2^-64 what it leaves of them is 0.
    if (softcap > 0.0f && softcap < 0x1p-64f)
      scale = 0.0f;
    if (softcap > 0x1p64f || softcap < 0x1p-64f)
      softcap = 0.0f;
    a.scale = scale, a.softcap = softcap, a.slopes = slopes, a.prefix = prefix;
    a.gate = gate, a.gate_row = gate_row, a.gate_head = gate_head;
    a.out = out, a.workspace = workspace;
    int launches = 0;
    check(launch_paged_attention(c, b, a, status, sms, static_cast<cudaStream_t>(stream), &launches), "paged attention");
    count_launches(static_cast<uint64_t>(launches));
  });
}
