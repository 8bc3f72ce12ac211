// Shared by the kernels between the projections of a layer with linear
// attention (the norms around a block, the short convolution, the linear
// attention) and their C entry points: launch arguments and elementwise
// functions.
#pragma once

#include "attention.h"

namespace jv {

constexpr float kLog2e = 1.4426950408889634f;

// 1 / sqrt(m): the hardware's, which takes a subnormal m for 0 (so those go
// through it scaled), and one Newton step (none where m is 0, inf or NaN).
__device__ __forceinline__ float inv_sqrt(float m) {
  const bool tiny = m < 0x1p-100f;
  m *= tiny ? 0x1p60f : 1.0f;
  float r = __builtin_amdgcn_rsqf(m);
  const float n = r * __builtin_fmaf(-0.5f * m * r, r, 1.5f);
  if (m > 0.0f && m < __builtin_inff()) r = n;
  return r * (tiny ? 0x1p30f : 1.0f);
}

// 1 / d, d at least 1: the hardware's with one Newton step, which on this chip
// gives the division's bits for every float (the tests go through all of them:
// from any reciprocal within one unit the step would miss some); past 2^126, where
// the hardware has no quotient, the division (five instructions instead of ten:
// 16 prompts through the convolution 96 -> 84 us).
__device__ __forceinline__ float inverse(float d) {
  if (d >= 0x1p126f) return 1.0f / d;
  const float r = __builtin_amdgcn_rcpf(d);
  return __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
}

// 1 / (1 + e^-x) and x / (1 + e^-x) in the steps of the elementary operations
// (exponential, sum, quotient, product), each rounded.
__device__ __forceinline__ float sigmoid(float x) { return inverse(1.0f + expf(-x)); }
__device__ __forceinline__ float silu(float x) { return x * sigmoid(x); }

// The first by the hardware's 2^x alone, for what is then rounded to 16 or 8 bits:
// the product's rounding puts |x| 2^-24 into the exponential, which counts where
// that is not small against 1 (4099 rows of 4096 to codes 21 us, with expf 25).
__device__ __forceinline__ float quick_sigmoid(float x) { return inverse(1.0f + __builtin_amdgcn_exp2f(-x * kLog2e)); }

// log(1 + e^x) = max(x, 0) + log1p(u), u = e^-|x| <= 1, with log1p(u) =
// 2 atanh(s), s = u / (2 + u) <= 1/3, by the series s + s^3/3 + .. + s^15/15
// (what follows is below 2^-29 of it). Far below 0 u is all that is left, so it is
// the exponential itself, one for a token and head: 2^x of a rounded product would
// be off by |x| 2^-24.
__device__ __forceinline__ float softplus(float x) {
  const float u = expf(-__builtin_fabsf(x));
  const float s = u / (2.0f + u), t = s * s;
  float p = 1.0f / 15;
#pragma unroll
  for (int n = 13; n > 0; n -= 2) p = __builtin_fmaf(p, t, 1.0f / n);
  const float l = 2.0f * s * p;
  return x > 0.0f ? x + l : x != x ? x : l;
}

// Sum over the wave, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int s = 1; s < 64; s *= 2) v += __shfl_xor(v, s);
  return v;
}

// ---------------------------------------------------------------------------
// Norms around a block (norm.hip).
// ---------------------------------------------------------------------------
struct NormArgs {
  const uint16_t *x, *residual, *gate;  // residual, gate may be null
  int64_t x_ts, x_hs, residual_ts, gate_ts, gate_hs;
  int activation;
  const float *post_weight, *weight;  // null: no norm
  float scale, eps;
  uint16_t *h_out, *y_out;  // may be null
  uint8_t* codes;           // null: none
  int64_t ldc;              // 0: packed
  float* scales;
  int tokens, heads, dim, cols;
};
hipError_t block_norm(const NormArgs& a, bool fp16, hipStream_t stream);

// ---------------------------------------------------------------------------
// Sequences of a batch and the slots of what they carry on.
// ---------------------------------------------------------------------------
struct Batch {
  const int32_t *starts, *slots, *from;  // starts null: one token each
  int64_t n_slots;
  int tokens, batch;
};

// A value that the whole wave reads, through the scalar cache; the index is
// uniform and the array is not written by the kernel.
__device__ __forceinline__ int32_t uniform_at(const int32_t* p, int i) {
  typedef const __attribute__((address_space(4))) int32_t* constant_ptr;
  return *(constant_ptr)(uintptr_t)(p + __builtin_amdgcn_readfirstlane(i));
}

__device__ __forceinline__ float uniform_f32(const float* p, int i) {
  typedef const __attribute__((address_space(4))) float* constant_ptr;
  return *(constant_ptr)(uintptr_t)(p + __builtin_amdgcn_readfirstlane(i));
}

struct ConvArgs {
  const uint16_t* x;
  int64_t x_ts;
  const float *weight, *bias;
  int activation;
  uint16_t* states;
  Batch b;
  uint16_t* out;
  int channels;
};
hipError_t causal_conv(const ConvArgs& a, int width, bool fp16, hipStream_t stream);

struct LinearArgs {
  const uint16_t *q, *k, *v;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
  const void *decay, *beta;  // beta null: no correction
  int64_t decay_ts, beta_ts;
  int gates16;
  const float *rate, *decay_bias;  // rate null: gates as they are
  float norm_eps;                  // 0: no norm
  float* states;
  Batch b;
  float scale;
  uint16_t* out;
  int k_heads, v_heads, group;
  uint8_t* workspace;
};
constexpr int kChunk = 64;
// Chunks of a batch: sequence b's take the places from floor(start_b / 64) + b
// on, which never meet those of b + 1.
__host__ __device__ inline int64_t linear_chunks(int64_t tokens, int64_t batch) { return tokens / kChunk + batch; }
// Of the batch's 64 tokens from `place` x 64 on those that there are: batches of
// many sequences have places past the last token, 2^20 of them and more.
__host__ __device__ inline int rows_at(int place, int tokens) {
  const int n = tokens - place * kChunk;
  return n < 0 ? 0 : n < kChunk ? n : kChunk;
}
int64_t linear_workspace(int64_t tokens, int64_t batch, int64_t k_heads, int64_t v_heads, int64_t k_dim);
hipError_t linear_step(const LinearArgs& a, int k_dim, int v_dim, bool fp16, hipStream_t stream);
hipError_t linear_prompt(const LinearArgs& a, int k_dim, int v_dim, bool fp16, hipStream_t stream);

}  // namespace jv
