// C ABI of the attention-side kernels (declared in include/jeeves_attention.h):
// argument validation and launches only.
#include <cmath>

#include "../../include/jeeves_attention.h"
#include "../../include/jeeves_fp8.h"
#include "attention.h"

namespace {

using jv::fail;
using jv::hip_status;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Rows of a call: its grids then stay below 2^24 workgroups of 256 threads.
constexpr int64_t kMaxRows = (int64_t(1) << 28) - 1;
// Keys that a query can see.
constexpr int64_t kMaxKeys = int64_t(1) << 30;

int check_heads(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t dim) {
  if (dim != 64 && dim != 128 && dim != 256) return fail(JV_ERR_VALUE, "heads of 64, 128 or 256 channels, got %lld", (long long)dim);
  if (tokens < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads > 65536 || kv_heads > 65536 ||
      tokens > kMaxRows / (q_heads + 2 * kv_heads))
    return fail(JV_ERR_VALUE, "bad sizes: %lld tokens, %lld query heads, %lld key heads", (long long)tokens, (long long)q_heads,
                (long long)kv_heads);
  return JV_OK;
}

// Rows of [tokens, heads, dim] that 16-byte loads reach.
int check_rows(const char* name, const void* p, int64_t ts, int64_t hs) {
  if (!p) return fail(JV_ERR_VALUE, "%s is missing", name);
  if (!aligned16(p) || ts % 8 || hs % 8) return fail(JV_ERR_VALUE, "%s needs 16-byte aligned rows", name);
  return JV_OK;
}

int check_rope(const float* rope, int64_t n_pos, int64_t rotary, const void* pos, int64_t dim) {
  if (!rope) return JV_OK;
  if (rotary <= 0 || rotary % 16 || rotary > dim)
    return fail(JV_ERR_VALUE, "the rotation takes a multiple of 16 channels up to %lld, got %lld", (long long)dim, (long long)rotary);
  if (n_pos < 1 || !pos || !aligned16(rope))
    return fail(JV_ERR_VALUE, "the rotation needs positions and a 16-byte aligned table of one position at least");
  return JV_OK;
}

int page_shift_of(int64_t page_size) {
  for (int s = 4; s <= 10; ++s)
    if (page_size == (int64_t)1 << s) return s;
  return -1;
}

int check_cache(const void* k_pages, const void* v_pages, int64_t pages, int64_t page_size) {
  if (page_shift_of(page_size) < 0)
    return fail(JV_ERR_VALUE, "the page size is a power of two from 16 to 1024, got %lld", (long long)page_size);
  if (pages <= 0 || pages > INT32_MAX) return fail(JV_ERR_VALUE, "bad page count %lld", (long long)pages);
  if (!k_pages || !v_pages || !aligned16(k_pages) || !aligned16(v_pages))
    return fail(JV_ERR_VALUE, "the cache needs 16-byte aligned pages of keys and values");
  return JV_OK;
}

// Sizes the attention's grids and 32-bit counts hold.
int check_batch(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t prefix_len) {
  if (int rc = check_heads(tokens, q_heads, kv_heads, dim)) return rc;
  if (q_heads % kv_heads)
    return fail(JV_ERR_VALUE, "%lld query heads are no multiple of %lld key heads", (long long)q_heads, (long long)kv_heads);
  if (batch < 0 || batch > (1 << 20) || prefix_len < 0 || prefix_len > (1 << 30))
    return fail(JV_ERR_VALUE, "bad sizes: batch %lld, prefix of %lld keys", (long long)batch, (long long)prefix_len);
  if ((tokens * q_heads / kv_heads + batch * 16) * kv_heads > INT32_MAX / 4)
    return fail(JV_ERR_VALUE, "too many rows for one call: %lld tokens, %lld heads", (long long)tokens, (long long)q_heads);
  return JV_OK;
}

// Counters of a plan: one a unit and key head, where the last unit of a tile joins its parts.
int64_t counters_of(const jv::AttnPlan& p, int64_t kv_heads) {
  return p.split && !p.prefix_tiles ? p.own_units * kv_heads : 0;
}

}  // namespace

extern "C" {

int jv_norm_rope(const void* q, int64_t q_ts, int64_t q_hs, const void* k, int64_t k_ts, int64_t k_hs, const float* rope,
                 int64_t n_pos, int64_t rotary, const void* pos, int pos64, const float* q_weight, const float* k_weight,
                 float eps, void* q_out, void* k_out, int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t dim, int fp16,
                 void* stream) {
  if (int rc = check_heads(tokens, q_heads, kv_heads, dim)) return rc;
  if (int rc = check_rope(rope, n_pos, rotary, pos, dim)) return rc;
  if (tokens == 0) return JV_OK;
  if (int rc = check_rows("q", q, q_ts, q_hs)) return rc;
  if (int rc = check_rows("k", k, k_ts, k_hs)) return rc;
  if (int rc = check_rows("the output", q_out, 0, 0)) return rc;
  if (int rc = check_rows("the output", k_out, 0, 0)) return rc;
  jv::RopeArgs a{};
  a.q = (const uint16_t*)q, a.k = (const uint16_t*)k;
  a.q_ts = q_ts, a.q_hs = q_hs, a.k_ts = k_ts, a.k_hs = k_hs;
  a.rope = rope, a.pos = pos, a.n_pos = n_pos, a.pos64 = pos64, a.rotary = rope ? (int)rotary : 0;
  a.q_weight = q_weight, a.k_weight = k_weight, a.eps = eps;
  a.q_out = (uint16_t*)q_out, a.k_out = (uint16_t*)k_out;
  a.tokens = (int)tokens, a.q_heads = (int)q_heads, a.kv_heads = (int)kv_heads;
  return hip_status(jv::norm_rope(a, (int)dim, fp16 != 0, (hipStream_t)stream), "norm and rotation launch");
}

int jv_append_kv(const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts, int64_t v_hs, const void* slots,
                 int slot64, void* k_pages, void* v_pages, int64_t pages, int64_t page_size, const float* rope, int64_t n_pos,
                 int64_t rotary, const void* pos, int pos64, const float* k_weight, float eps, const void* q, int64_t q_ts,
                 int64_t q_hs, const float* q_weight, void* q_out, int64_t q_heads, int64_t tokens, int64_t kv_heads,
                 int64_t dim, int fp16, void* stream) {
  if (int rc = check_heads(tokens, q ? q_heads : 1, kv_heads, dim)) return rc;
  if (int rc = check_cache(k_pages, v_pages, pages, page_size)) return rc;
  if (int rc = check_rope(rope, n_pos, rotary, pos, dim)) return rc;
  if (tokens == 0) return JV_OK;
  if (int rc = check_rows("k", k, k_ts, k_hs)) return rc;
  if (int rc = check_rows("v", v, v_ts, v_hs)) return rc;
  if (q) {
    if (int rc = check_rows("q", q, q_ts, q_hs)) return rc;
    if (int rc = check_rows("the output", q_out, 0, 0)) return rc;
  }
  if (!slots) return fail(JV_ERR_VALUE, "the append needs the tokens' slots");
  jv::RopeArgs a{};
  a.q = (const uint16_t*)q, a.k = (const uint16_t*)k, a.v = (const uint16_t*)v;
  a.q_ts = q_ts, a.q_hs = q_hs, a.k_ts = k_ts, a.k_hs = k_hs, a.v_ts = v_ts, a.v_hs = v_hs;
  a.rope = rope, a.pos = pos, a.n_pos = n_pos, a.pos64 = pos64, a.rotary = rope ? (int)rotary : 0;
  a.q_weight = q_weight, a.k_weight = k_weight, a.eps = eps;
  a.q_out = (uint16_t*)q_out;
  a.k_pages = (uint16_t*)k_pages, a.v_pages = (uint16_t*)v_pages;
  a.slots = slots, a.slot64 = slot64, a.page_shift = page_shift_of(page_size), a.n_slots = pages * page_size;
  a.tokens = (int)tokens, a.q_heads = q ? (int)q_heads : 0, a.kv_heads = (int)kv_heads;
  return hip_status(jv::norm_rope(a, (int)dim, fp16 != 0, (hipStream_t)stream), "cache append launch");
}

int jv_narrow_indices(const int64_t* src, int64_t rows, int64_t cols, int64_t row_stride, int64_t col_stride, int32_t* dst,
                      void* stream) {
  if (rows < 0 || cols < 0 || (cols > 0 && rows > INT32_MAX / cols))
    return fail(JV_ERR_VALUE, "bad sizes: %lld rows of %lld indices", (long long)rows, (long long)cols);
  if (rows == 0 || cols == 0) return JV_OK;
  if (!src || !dst) return fail(JV_ERR_VALUE, "the indices or their output are missing");
  return hip_status(jv::narrow_indices(src, (int)rows, (int)cols, row_stride, col_stride, dst, (hipStream_t)stream),
                    "index launch");
}

int64_t jv_paged_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                           int64_t prefix_len, int ragged) {
  if (check_batch(tokens, batch, q_heads, kv_heads, dim, prefix_len)) return -1;
  if (tokens == 0 || batch == 0) return 0;
  const int cus = jv::cu_count_of(-1);
  if (cus <= 0) return -1;
  return jv::attention_workspace(jv::attention_plan(tokens, batch, q_heads, kv_heads, dim, prefix_len, ragged != 0, cus), batch,
                                 kv_heads, dim);
}

int64_t jv_paged_attention_counters_needed(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                           int64_t prefix_len, int ragged) {
  if (check_batch(tokens, batch, q_heads, kv_heads, dim, prefix_len)) return -1;
  if (tokens == 0 || batch == 0) return 0;
  const int cus = jv::cu_count_of(-1);
  if (cus <= 0) return -1;
  return counters_of(jv::attention_plan(tokens, batch, q_heads, kv_heads, dim, prefix_len, ragged != 0, cus), kv_heads);
}

int jv_paged_attention(const void* q, int64_t q_ts, int64_t q_hs, const void* k_pages, const void* v_pages, int64_t pages,
                       int64_t page_size, const int32_t* table, int64_t table_stride, int64_t table_cols,
                       const int32_t* lengths, const int32_t* starts, int64_t batch, const int32_t* prefix_pages,
                       int64_t prefix_len, float scale, void* out, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                       int64_t dim, int fp16, void* workspace, int64_t workspace_bytes, int32_t* counters, int64_t n_counters,
                       void* stream) {
  if (int rc = check_batch(tokens, batch, q_heads, kv_heads, dim, prefix_len)) return rc;
  if (int rc = check_cache(k_pages, v_pages, pages, page_size)) return rc;
  if (!(scale > 0.0f) || !std::isfinite(scale)) return fail(JV_ERR_VALUE, "the scale must be positive and finite, got %g", scale);
  if (!starts && tokens != batch)
    return fail(JV_ERR_VALUE, "without query starts each of the %lld sequences has one token, got %lld", (long long)batch,
                (long long)tokens);
  if (table_cols < 0 || table_stride < 0 || table_cols > kMaxKeys / page_size || table_cols * page_size + prefix_len > kMaxKeys)
    return fail(JV_ERR_VALUE, "page table of %lld columns for a batch of %lld is too large", (long long)table_cols, (long long)batch);
  if (tokens == 0) return JV_OK;
  if (batch == 0) return fail(JV_ERR_VALUE, "%lld tokens of no sequence", (long long)tokens);
  if (int rc = check_rows("q", q, q_ts, q_hs)) return rc;
  if (int rc = check_rows("the output", out, 0, 0)) return rc;
  if (!lengths || (!table && table_cols > 0) || (!prefix_pages && prefix_len > 0))
    return fail(JV_ERR_VALUE, "the attention needs the lengths and the pages of its keys");
  const int cus = jv::cu_count_of(-1);
  if (cus <= 0) return fail(JV_ERR_HIP, "cannot query the device's compute units");
  jv::AttnArgs a{};
  a.p = jv::attention_plan(tokens, batch, q_heads, kv_heads, dim, prefix_len, starts != nullptr, cus);
  const int64_t need = jv::attention_workspace(a.p, batch, kv_heads, dim);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return fail(JV_ERR_VALUE, "workspace needs %lld bytes, 256-byte aligned", (long long)need);
  // where keys are split, the 32-bit sum of the tiles' keys in steps of 16 and more
  if (a.p.split && a.p.tiles * ((table_cols * page_size + prefix_len) / 16 + 1 + a.p.tiles) > INT32_MAX)
    return fail(JV_ERR_VALUE, "page table of %lld columns for a batch of %lld is too large", (long long)table_cols, (long long)batch);
  const int64_t units = (int64_t)a.p.own_units * kv_heads, shares = (int64_t)a.p.prefix_tiles * a.p.prefix_splits * kv_heads;
  if (units + shares >= int64_t(1) << 24 || (shares && tokens * q_heads >= int64_t(1) << 26))
    return fail(JV_ERR_VALUE, "too many rows for one call: %lld tokens, %lld heads", (long long)tokens, (long long)q_heads);
  if (const int64_t n = counters_of(a.p, kv_heads); n && (!counters || n_counters < n))
    return fail(JV_ERR_VALUE, "%lld units exceed the %lld counters", (long long)n, (long long)n_counters);
  a.counters = counters;
  a.q = (const uint16_t*)q, a.q_ts = q_ts, a.q_hs = q_hs;
  a.k_pages = (const uint16_t*)k_pages, a.v_pages = (const uint16_t*)v_pages;
  a.pages = (int)pages, a.page_shift = page_shift_of(page_size);
  a.table = table, a.table_stride = table_stride, a.table_cols = (int)table_cols;
  a.lengths = lengths, a.starts = starts;
  a.prefix_pages = prefix_pages, a.prefix_len = (int)prefix_len;
  a.tokens = (int)tokens, a.batch = (int)batch, a.q_heads = (int)q_heads, a.kv_heads = (int)kv_heads;
  a.group = (int)(q_heads / kv_heads);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = (uint16_t*)out;
  return hip_status(jv::paged_attention(a, (int)dim, fp16 != 0, workspace, (hipStream_t)stream), "attention launch");
}

}  // extern "C"
