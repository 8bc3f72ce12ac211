// Per-head RMS norms and the position rotation of queries and keys, and the
// append of keys and values to the paged cache, in one pass over the rows.
//
// A head's row x of `dim` channels: y = x w / sqrt(mean(x^2) + eps) (y = x
// without a weight), then, for i < rotary / 2 and the angle t of the token's
// position, z_i = y_i cos t_i - y_{i + rotary/2} sin t_i and
// z_{i + rotary/2} = y_{i + rotary/2} cos t_i + y_i sin t_i; the channels from
// `rotary` on stay y. All of it in fp32, rounded once when z is stored.
//
// The rows are read and written once, so HBM bounds it: 7921 tokens of 40 heads
// of 128 take 35 us, 4.7 TB/s of the 4.9 that a copy reaches; few tokens take
// the 3 us of a launch and its two dependent loads. A group of dim / 8 lanes
// holds a row, 16 bytes a lane; the rotation's partner channels come from
// another lane of the group. A group takes kHeads heads of one token, with the
// token's angles and the head weights in registers (they would be eight of the
// nine loads of every 16 bytes otherwise). Two heads: with one those 7921 tokens
// take 41 us and the append of 4096 tokens of 4 heads of 256 10.6 us; with two
// 35.4 and 9.8; with four, which leave the device fewer waves, 34.6 and 11.3,
// and 7.5 instead of 7.3 us for 800 tokens.
#include "attention.h"

namespace jv {

__device__ __forceinline__ int64_t load_index(const void* p, int wide, int i) {
  return wide ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t)reinterpret_cast<const int32_t*>(p)[i];
}

constexpr int kHeads = 2;

template <class H, int D>
__global__ __launch_bounds__(256) void norm_rope_kernel(RopeArgs a, uint32_t q_blocks, uint32_t kv_blocks, uint32_t per_token,
                                                        uint32_t tasks) {
  constexpr int LPH = D / 8;  // lanes of a head
  const uint32_t task = blockIdx.x * (256 / LPH) + threadIdx.x / LPH;
  if (task >= tasks) return;
  const int token = (int)(task / per_token);
  const uint32_t j = task % per_token;
  const int c = threadIdx.x % LPH;  // this lane's 8 channels: 8 c ..
  const bool is_q = j < q_blocks, is_v = j >= q_blocks + kv_blocks;
  const int h0 = (int)(is_q ? j : is_v ? j - q_blocks - kv_blocks : j - q_blocks) * kHeads;
  const int heads = is_q ? a.q_heads : a.kv_heads;
  const uint16_t* src = is_q ? a.q + token * a.q_ts : is_v ? a.v + token * a.v_ts : a.k + token * a.k_ts;
  const int64_t hs = is_q ? a.q_hs : is_v ? a.v_hs : a.k_hs;
  uint4 x[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) x[i] = *reinterpret_cast<const uint4*>(src + min(h0 + i, heads - 1) * hs + c * 8);

  // Where the row goes: q and k rows to their outputs, or k and v to a slot.
  uint16_t* dst;
  int64_t dst_hs = D;
  bool keep = true;
  if (is_q || a.k_out) {
    dst = (is_q ? a.q_out : a.k_out) + (int64_t)token * heads * D;
  } else {
    const int64_t slot = load_index(a.slots, a.slot64, token);
    keep = slot >= 0 && slot < a.n_slots;
    dst_hs = (int64_t)D << a.page_shift;
    dst = (is_v ? a.v_pages : a.k_pages) + (slot >> a.page_shift) * a.kv_heads * dst_hs +
          (slot & (((int64_t)1 << a.page_shift) - 1)) * D;
  }
  dst += c * 8;

  if (!is_v) {
    const float* weight = is_q ? a.q_weight : a.k_weight;
    const int half = a.rotary >> 4;  // lanes of half the rotated channels
    const bool rot = a.rope && c < 2 * half;
    const int pc = !rot ? c : c < half ? c + half : c - half;  // the partner's lane
    const int partner = (int)(threadIdx.x & 63) - c + pc;
    float cs[8], sn[8], w[8], wp[8];
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) cs[e] = 1.0f, sn[e] = 0.0f, w[e] = 1.0f, wp[e] = 1.0f;
    if (weight) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = weight[c * 8 + e], wp[e] = weight[pc * 8 + e];
    }
    if (a.rope) {
      const int64_t pos = load_index(a.pos, a.pos64, token);
      bad = pos < 0 || pos >= a.n_pos;
      if (rot) {
        const float* t = a.rope + (bad ? 0 : pos) * a.rotary + (c < half ? c : pc) * 8;
        const float sign = c < half ? -1.0f : 1.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) cs[e] = t[e], sn[e] = sign * t[8 * half + e];
      }
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const uint32_t xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      float f[8], g[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t p = (uint32_t)__shfl((int)xs[e], partner);
        f[2 * e] = H::lo(xs[e]), f[2 * e + 1] = H::hi(xs[e]);
        g[2 * e] = H::lo(p), g[2 * e + 1] = H::hi(p);
      }
      float r = 1.0f;
      if (weight) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(f[e], f[e], ss);
#pragma unroll
        for (int s = 1; s < LPH; s *= 2) ss += __shfl_xor(ss, s);
        float m = ss * (1.0f / D) + a.eps;
        // the hardware's 1 / sqrt, which takes a subnormal m for 0 (so those go
        // through it scaled), and one Newton step (none where m is 0, inf or NaN)
        const bool tiny = m < 0x1p-100f;
        m *= tiny ? 0x1p60f : 1.0f;
        r = __builtin_amdgcn_rsqf(m);
        const float n = r * __builtin_fmaf(-0.5f * m * r, r, 1.5f);
        if (m > 0.0f && m < __builtin_inff()) r = n;
        r *= tiny ? 0x1p30f : 1.0f;
      }
      // a position that the table does not have: no angle, so no row
      if (bad) r = __builtin_nanf("");
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = f[e] * r * w[e];
        z[e] = rot ? __builtin_fmaf(g[e] * r * wp[e], sn[e], y * cs[e]) : y;
      }
      x[i] = uint4{H::pack(z[0], z[1]), H::pack(z[2], z[3]), H::pack(z[4], z[5]), H::pack(z[6], z[7])};
    }
  }
#pragma unroll
  for (int i = 0; i < kHeads; ++i)
    if (keep && h0 + i < heads) *reinterpret_cast<uint4*>(dst + (h0 + i) * dst_hs) = x[i];
}

// A few thousand values at most: a launch's time.
__global__ __launch_bounds__(256) void narrow_kernel(const int64_t* src, uint32_t n, uint32_t cols, int64_t row_stride,
                                                     int64_t col_stride, int32_t* dst) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int64_t v = src[(int64_t)(i / cols) * row_stride + (int64_t)(i % cols) * col_stride];
  dst[i] = (int32_t)(v < INT32_MIN ? INT32_MIN : v > INT32_MAX ? INT32_MAX : v);
}

hipError_t narrow_indices(const int64_t* src, int rows, int cols, int64_t row_stride, int64_t col_stride, int32_t* dst,
                          hipStream_t stream) {
  const uint32_t n = (uint32_t)rows * (uint32_t)cols;
  narrow_kernel<<<(n + 255) / 256, 256, 0, stream>>>(src, n, (uint32_t)cols, row_stride, col_stride, dst);
  return hipGetLastError();
}

template <class H, int D>
static void launch_norm_rope(const RopeArgs& a, hipStream_t stream) {
  const auto blocks = [](int heads) { return (uint32_t)((heads + kHeads - 1) / kHeads); };
  const uint32_t qb = a.q ? blocks(a.q_heads) : 0, kb = blocks(a.kv_heads), per = qb + kb + (a.v ? kb : 0);
  const uint32_t tasks = per * (uint32_t)a.tokens, groups = 256 / (D / 8);
  norm_rope_kernel<H, D><<<(tasks + groups - 1) / groups, 256, 0, stream>>>(a, qb, kb, per, tasks);
}

hipError_t norm_rope(const RopeArgs& a, int dim, bool fp16, hipStream_t stream) {
  if (dim == 64) fp16 ? launch_norm_rope<Fp16, 64>(a, stream) : launch_norm_rope<Bf16, 64>(a, stream);
  else if (dim == 128) fp16 ? launch_norm_rope<Fp16, 128>(a, stream) : launch_norm_rope<Bf16, 128>(a, stream);
  else if (dim == 256) fp16 ? launch_norm_rope<Fp16, 256>(a, stream) : launch_norm_rope<Bf16, 256>(a, stream);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

}  // namespace jv
