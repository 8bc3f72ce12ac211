/*
 * jeeves_attention.h -- C ABI of what lies between the q/k/v and the o
 * projections of a served model (libjeeves_fp8.so, MI355X / gfx950): norms and
 * rotation of queries and keys, the paged key/value cache's append, and the
 * attention that reads the cache.
 *
 * Conventions are those of jeeves_fp8.h: device pointers, a hipStream_t, a
 * JV_* status with jv_fp8_last_error(), launches only (no allocation, no host
 * synchronisation), so that every call may be captured into a HIP graph.
 *
 * Tensors are bf16 (fp16 = 0) or fp16 (fp16 = 1). Queries, keys and values are
 * [tokens, heads, dim] with strides in elements for tokens (`ts`) and heads
 * (`hs`), unit stride over dim and 16-byte aligned rows; dim is 64, 128 or 256.
 * The cache is two contiguous arrays [pages, kv_heads, page_size, dim], the
 * page size a power of two from 16 to 1024. Token `offset` of page `page` is
 * slot page * page_size + offset. A call takes less than 2^28 rows (tokens times
 * heads of q, k and v) and queries that can see up to 2^30 keys, in all fewer
 * than 2^35 for the row tiles of a call that splits its keys over workgroups.
 */
#ifndef JEEVES_ATTENTION_H
#define JEEVES_ATTENTION_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Per-head RMS norms and rotation of q and k into contiguous q_out and k_out.
 * A head row x becomes y = x w / sqrt(mean(x^2) + eps) (y = x where the weight
 * is NULL; weights are float32 [dim]), and with a table its channels i and
 * i + rotary / 2 (i < rotary / 2) are turned by the angle of the token's
 * position: fp32 throughout, rounded once.
 * rope: float32 [n_pos, rotary], each position's rotary / 2 cosines, then its
 * sines, 16-byte aligned, n_pos at least 1 (NULL: no rotation); rotary a
 * multiple of 16 up to dim. pos: int32 [tokens], int64 with pos64. A token whose
 * position the table does not have comes out as NaN. The role of _rotary
 * (model/triton_kernels.py:54) and of the q and k norms before it.
 */
int jv_norm_rope(const void* q, int64_t q_ts, int64_t q_hs, const void* k, int64_t k_ts, int64_t k_hs, const float* rope,
                 int64_t n_pos, int64_t rotary, const void* pos, int pos64, const float* q_weight, const float* k_weight,
                 float eps, void* q_out, void* k_out, int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t dim, int fp16,
                 void* stream);

/*
 * Keys, normed and rotated as by jv_norm_rope, and values into their slots of
 * the cache; with q (may be NULL) the queries into q_out in the same launch.
 * slots: int32 [tokens], int64 with slot64; a token whose slot is negative or
 * past the cache is left out. Two tokens with one slot: either's row may stay.
 * The role of _rotate_into_cache (model/triton_kernels.py:214).
 */
int jv_append_kv(const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts, int64_t v_hs, const void* slots,
                 int slot64, void* k_pages, void* v_pages, int64_t pages, int64_t page_size, const float* rope, int64_t n_pos,
                 int64_t rotary, const void* pos, int pos64, const float* k_weight, float eps, const void* q, int64_t q_ts,
                 int64_t q_hs, const float* q_weight, void* q_out, int64_t q_heads, int64_t tokens, int64_t kv_heads,
                 int64_t dim, int fp16, void* stream);

/*
 * int64 page tables, lengths or starts [rows, cols] as the contiguous int32
 * that jv_paged_attention takes, values past 32 bits held at their ends.
 * Strides in elements; fewer than 2^31 values.
 */
int jv_narrow_indices(const int64_t* src, int64_t rows, int64_t cols, int64_t row_stride, int64_t col_stride, int32_t* dst,
                      void* stream);

#define JV_ATTENTION_COUNTERS 65536

/* Bytes of workspace jv_paged_attention needs for these sizes on the current
 * device (0: none); -1 if it cannot be queried or the sizes are refused. */
int64_t jv_paged_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                           int64_t prefix_len, int ragged);
/* Counters that it needs (0: none, they may be NULL); -1 as above. */
int64_t jv_paged_attention_counters_needed(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim,
                                           int64_t prefix_len, int ragged);

/*
 * Attention of a batch over the cache. Sequence b has the tokens starts[b] ..
 * starts[b + 1] - 1 of q (starts: int32 [batch + 1], not decreasing, from 0 to
 * tokens; NULL: one token each, tokens = batch) and lengths[b] own keys (int32), which lie in
 * the pages table[b * table_stride ..] in order; its token i of n sees the own
 * keys up to lengths[b] - n + i, and the first prefix_len keys of the pages
 * prefix_pages, which the whole batch shares (prefix_len 0: none). Query head h
 * reads kv head h / (q_heads / kv_heads). out [tokens, q_heads, dim],
 * contiguous, is the softmax-weighted sum of the values, scores times `scale`;
 * 0 where a token sees no key or belongs to no sequence. Keys that a token
 * does not see have no effect, whatever their values; a NaN score that it sees
 * makes its row NaN, a NaN value the channel. Lengths are taken up to
 * the table's width, page ids into the cache's range.
 * workspace: 256-byte aligned. counters: int32, JV_ATTENTION_COUNTERS of them
 * serve every call; zero before the first call and left at zero by each, one
 * set for each stream whose calls can overlap. The role of _decode_attention_split and
 * _decode_attention_combine (model/triton_kernels.py:118-171).
 */
int jv_paged_attention(const void* q, int64_t q_ts, int64_t q_hs, const void* k_pages, const void* v_pages, int64_t pages,
                       int64_t page_size, const int32_t* table, int64_t table_stride, int64_t table_cols,
                       const int32_t* lengths, const int32_t* starts, int64_t batch, const int32_t* prefix_pages,
                       int64_t prefix_len, float scale, void* out, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                       int64_t dim, int fp16, void* workspace, int64_t workspace_bytes, int32_t* counters,
                       int64_t n_counters, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* JEEVES_ATTENTION_H */
