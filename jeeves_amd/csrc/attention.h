// Shared by the attention-side kernels (rotation and norms of q and k, the
// paged cache's append, the attention over it) and their C entry points:
// 16-bit types, launch arguments and the host-side plan.
//
// The cache: K and V as [pages, kv_heads, page_size, head_dim] of bf16 or
// fp16, page_size a power of two from 16. One head's keys of a page are one
// run of memory, and a group of 16 keys that starts at a multiple of 16 lies
// in one page.
#pragma once

#include <algorithm>

#include "fp8_common.h"
#include "status.h"

namespace jv {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// The two 16-bit types: packing of two floats (round to nearest even),
// unpacking, the MFMA that multiplies them with fp32 sums, and the bits of
// +infinity (all exponent bits).
struct Bf16 {
  static constexpr uint32_t kInf = 0x7F80u;
  static constexpr float kShift = 0.0f;  // exponent added to softmax weights
  static __device__ __forceinline__ float lo(uint32_t v) { return __uint_as_float(v << 16); }
  static __device__ __forceinline__ float hi(uint32_t v) { return __uint_as_float(v & 0xFFFF0000u); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  // c + both halves of v
  static __device__ __forceinline__ float add2(uint32_t v, float c) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, v), __builtin_bit_cast(bf16x2, 0x3F803F80u), c, false);
  }
  static __device__ __forceinline__ f32x16 mfma32(i32x4 a, i32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(i32x4 a, i32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16k16(s16x4 a, s16x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
  }
};

struct Fp16 {
  static constexpr uint32_t kInf = 0x7C00u;
  static constexpr float kShift = 7.0f;
  static __device__ __forceinline__ float lo(uint32_t v) { return (float)__builtin_bit_cast(_Float16, (uint16_t)v); }
  static __device__ __forceinline__ float hi(uint32_t v) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(v >> 16)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16);
  }
  static __device__ __forceinline__ float add2(uint32_t v, float c) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, v), __builtin_bit_cast(f16x2, 0x3C003C00u), c, false);
  }
  static __device__ __forceinline__ f32x16 mfma32(i32x4 a, i32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16(i32x4 a, i32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mfma16k16(s16x4 a, s16x4 b, f32x4 c) {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
  }
};

// ---------------------------------------------------------------------------
// Norms, rotation, append (rope.hip).
// ---------------------------------------------------------------------------
struct RopeArgs {
  const uint16_t *q, *k, *v;                  // q, v may be null
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;  // token and head strides, elements
  const float* rope;                          // [positions, rotary]: cosines, then sines; null: no rotation
  const void* pos;                            // int32 or int64 [tokens]
  int64_t n_pos;
  int pos64, rotary;
  const float *q_weight, *k_weight;  // null: no norm
  float eps;
  uint16_t *q_out, *k_out;  // [tokens, heads, dim], contiguous; k_out null when appending
  uint16_t *k_pages, *v_pages;
  const void* slots;  // int32 or int64 [tokens]
  int slot64, page_shift;
  int64_t n_slots;
  int tokens, q_heads, kv_heads;
};

hipError_t norm_rope(const RopeArgs& a, int dim, bool fp16, hipStream_t stream);

// int64 indices [rows, cols] into contiguous int32, held in range (rope.hip).
hipError_t narrow_indices(const int64_t* src, int rows, int cols, int64_t row_stride, int64_t col_stride, int32_t* dst,
                          hipStream_t stream);

// ---------------------------------------------------------------------------
// Attention (attention.hip).
// ---------------------------------------------------------------------------
// Query rows of one kv head are (token, head in the group) pairs, token major:
// row = token * group + g. A sequence's rows are cut into tiles of `rows`
// (kFewRows or kManyRows); sequence b's tiles take the tile slots from
// floor(start_b * group / rows) + b on, which never meet those of b + 1
// (ceil(x - y) <= floor(x) - floor(y) + 1), so that the grid follows from the
// token and sequence counts alone while the starts stay on the device.
constexpr int kFewRows = 16, kManyRows = 128;

// Counters a call may use at most; keys that would need more are not split.
constexpr int64_t kAttnCounters = 65536;

struct AttnPlan {
  bool few_own, few_prefix;  // tiles of kFewRows rows instead of kManyRows
  bool split;                // the keys of a row tile may go to several workgroups
  int tiles;                 // at least the batch's row tiles
  int at_once;               // workgroups of a head that the device holds at a time
  int cu_units;              // workgroups of a head that come to the device's CUs first, one a CU
  int own_units;             // tile slots, or with a split the most units (tile, key chunk) that there can be
  int prefix_tiles, prefix_splits;  // where the prefix is gone through apart, for all tokens' rows
};

struct AttnArgs {
  const uint16_t* q;
  int64_t q_ts, q_hs;
  const uint16_t *k_pages, *v_pages;
  int pages, page_shift;
  const int32_t* table;
  int64_t table_stride;
  int table_cols;
  const int32_t *lengths, *starts;  // starts null: one token for each sequence
  const int32_t* prefix_pages;
  int prefix_len;
  int tokens, batch, q_heads, kv_heads, group;
  float scale_log2;  // scale * log2(e)
  uint16_t* out;     // [tokens, q_heads, dim]
  float *part_o, *prefix_o;      // partial results: [unit, kv_head, rows, dim]
  float2 *part_ml, *prefix_ml;   // their references and sums: [unit, kv_head, rows]
  int32_t* counters;             // 0 before and after each call
  int2* info;                    // a sequence's first unit and its tiles' chunks, for join_kernel
  AttnPlan p;
};

// Chosen by the sizes that the host knows.
AttnPlan attention_plan(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t prefix_len,
                        bool ragged, int cus);
int64_t attention_workspace(const AttnPlan& p, int64_t batch, int64_t kv_heads, int64_t dim);
hipError_t paged_attention(AttnArgs a, int dim, bool fp16, void* workspace, hipStream_t stream);

}  // namespace jv
