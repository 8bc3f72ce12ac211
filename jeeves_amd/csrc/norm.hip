// Norms around a block: one pass over a token's row that ends the block
// (its output's norm, its gate, the residual) and begins the next (that sum's
// norm, and the e4m3 codes that the next FP8 projection multiplies).
//
// Bound by bytes, each read and written once: 8192 rows of 4096, with a gate, a
// residual and both norms, in 65 us (336 MB, 5.2 TB/s, VALU 62%); 4099 rows of
// 4096 with a gate to codes in 21 us as a call among others (84 MB, 4.0 TB/s, VALU
// 67%: the sigmoids, and quotients for the codes), 28 by itself under a tracer, start
// and end included. One row by itself: 3.3 us, a launch and memory's latency.
#include "kernels.h"
#include "layer.h"

namespace jv {

// Largest |value| pattern over the workgroup's waves.
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* lds, int waves) {
  v = wave_max_u32(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  uint32_t m = lds[0];
  for (int w = 1; w < waves; ++w) m = max(m, lds[w]);
  return m;
}

__device__ __forceinline__ float block_sum(float v, float* lds, int waves) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = lds[0];
  for (int w = 1; w < waves; ++w) s += lds[w];
  return s;
}

// A workgroup takes a row, each thread NC chunks of 8 channels, which stay in
// registers. HEADS: the first norm is over heads of dim = 8 LPH channels.
template <class H, int NC, int LPH>
__global__ __launch_bounds__(512) void block_norm_kernel(NormArgs a) {
  constexpr bool kHeads = LPH > 0;
  __shared__ float sums[2][8];
  __shared__ uint32_t maxima[8];
  const int threads = blockDim.x, waves = threads >> 6, chunks = a.cols >> 3;
  const bool packed = a.codes && a.ldc == 0;
  // Packed codes: the rows of a 16-token tile on one XCD, whose L2 then joins
  // the pieces that they write into each fragment; rows past the last token
  // are padding, whose codes are 0.
  int row = blockIdx.x;
  bool active = true;
  if (packed) {
    const int tiles = (a.tokens + 15) >> 4, j = row >> 3, t = (row & 7) + 8 * (j >> 4);
    active = t < tiles;
    row = active ? t * 16 + (j & 15) : 0;
  }
  const bool real = active && row < a.tokens;
  const int src = min(row, a.tokens - 1);

  uint4 xv[NC], rv[NC], gv[NC];
  float f[NC][8];
  int at[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = min((int)threadIdx.x + i * threads, chunks - 1);
    at[i] = c;
    const int head = kHeads ? c / (kHeads ? LPH : 1) : 0;
    const int in = (c - head * LPH) * 8;
    xv[i] = *reinterpret_cast<const uint4*>(a.x + src * a.x_ts + head * a.x_hs + in);
    if (a.residual) rv[i] = *reinterpret_cast<const uint4*>(a.residual + src * a.residual_ts + c * 8);
    if (a.gate) gv[i] = *reinterpret_cast<const uint4*>(a.gate + src * a.gate_ts + head * a.gate_hs + in);
  }
  const auto unpack = [](uint4 v, float (&o)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) o[2 * e] = H::lo(w[e]), o[2 * e + 1] = H::hi(w[e]);
  };
#pragma unroll
  for (int i = 0; i < NC; ++i) unpack(xv[i], f[i]);

  if (a.post_weight) {
    float r[NC];
    if constexpr (kHeads) {
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(f[i][e], f[i][e], ss);
#pragma unroll
        for (int s = 1; s < LPH; s *= 2) ss += __shfl_xor(ss, s);
        r[i] = inv_sqrt(ss * (1.0f / (8 * LPH)) + a.eps);
      }
    } else {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < NC; ++i)
        if ((int)threadIdx.x + i * threads < chunks)
#pragma unroll
          for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(f[i][e], f[i][e], ss);
      const float m = inv_sqrt(block_sum(ss, sums[0], waves) / (float)a.cols + a.eps);
#pragma unroll
      for (int i = 0; i < NC; ++i) r[i] = m;
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const float* w = a.post_weight + (kHeads ? at[i] % (kHeads ? LPH : 1) : at[i]) * 8;
      const float4 w0 = *reinterpret_cast<const float4*>(w), w1 = *reinterpret_cast<const float4*>(w + 4);
      const float ws[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) f[i][e] = f[i][e] * r[i] * ws[e];
    }
  }
  if (a.gate) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      float g[8];
      unpack(gv[i], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float s = a.activation ? quick_sigmoid(g[e]) : g[e];
        f[i][e] *= a.activation == 2 ? g[e] * s : s;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    float g[8];
    if (a.residual) unpack(rv[i], g);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[i][e] = a.residual ? __builtin_fmaf(a.scale, f[i][e], g[e]) : a.scale * f[i][e];
  }
  const auto store = [&](uint16_t* out) {
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if (real && (int)threadIdx.x + i * threads < chunks)
        *reinterpret_cast<uint4*>(out + (int64_t)row * a.cols + at[i] * 8) =
            uint4{H::pack(f[i][0], f[i][1]), H::pack(f[i][2], f[i][3]), H::pack(f[i][4], f[i][5]), H::pack(f[i][6], f[i][7])};
  };
  if (a.h_out) store(a.h_out);
  if (a.weight) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
      if ((int)threadIdx.x + i * threads < chunks)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(f[i][e], f[i][e], ss);
    const float r = inv_sqrt(block_sum(ss, sums[1], waves) / (float)a.cols + a.eps);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const float4 w0 = *reinterpret_cast<const float4*>(a.weight + at[i] * 8);
      const float4 w1 = *reinterpret_cast<const float4*>(a.weight + at[i] * 8 + 4);
      const float ws[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) f[i][e] = f[i][e] * r * ws[e];
    }
  }
  if (a.y_out) store(a.y_out);
  if (!a.codes) return;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < NC; ++i)
    if ((int)threadIdx.x + i * threads < chunks)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[i][e]) & 0x7FFFFFFFu);  // NaN is above infinity
  top = block_max(top, maxima, waves);
  const float scale = scale_from_amax_f32(__uint_as_float(top));
  if (threadIdx.x == 0 && real) a.scales[row] = scale;
  const bool finite = top < 0x7F800000u;
  const float inv = 1.0f / scale;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    float q[8];
    // with the correctly rounded 1 / scale the corrected product is the IEEE quotient
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = finite ? __builtin_copysignf(quotient(f[i][e], scale, inv), f[i][e]) : f[i][e] / scale;
    uint2 code = {0u, 0u};
    if (finite) {
      int lo = cvt_pk_fp8<false>(q[0], q[1], 0), hi = cvt_pk_fp8<false>(q[4], q[5], 0);
      lo = cvt_pk_fp8<true>(q[2], q[3], lo), hi = cvt_pk_fp8<true>(q[6], q[7], hi);
      code = uint2{(uint32_t)lo, (uint32_t)hi};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) code.x |= e4m3_encode_sw(q[e]) << (8 * e), code.y |= e4m3_encode_sw(q[4 + e]) << (8 * e);
    }
    if (active && (packed || real) && (int)threadIdx.x + i * threads < chunks) {
      const int64_t off = packed ? packed_x_offset(row, at[i] * 8, a.cols >> 7) : (int64_t)row * a.ldc + at[i] * 8;
      *reinterpret_cast<uint2*>(a.codes + off) = real ? code : uint2{0u, 0u};
    }
  }
}

template <class H, int NC>
static void launch_block_norm(const NormArgs& a, hipStream_t stream) {
  const int chunks = a.cols / 8, threads = ((chunks + NC - 1) / NC + 63) / 64 * 64;
  const uint32_t tiles = (uint32_t)(a.tokens + 15) / 16;
  const uint32_t grid = a.codes && a.ldc == 0 ? (tiles + 7) / 8 * 128 : (uint32_t)a.tokens;
  switch (a.heads > 1 ? a.dim : 0) {
    case 64: block_norm_kernel<H, NC, 8><<<grid, threads, 0, stream>>>(a); break;
    case 128: block_norm_kernel<H, NC, 16><<<grid, threads, 0, stream>>>(a); break;
    case 256: block_norm_kernel<H, NC, 32><<<grid, threads, 0, stream>>>(a); break;
    default: block_norm_kernel<H, NC, 0><<<grid, threads, 0, stream>>>(a);
  }
}

hipError_t block_norm(const NormArgs& a, bool fp16, hipStream_t stream) {
  if (a.cols <= 4096) fp16 ? launch_block_norm<Fp16, 1>(a, stream) : launch_block_norm<Bf16, 1>(a, stream);
  else if (a.cols <= 8192) fp16 ? launch_block_norm<Fp16, 2>(a, stream) : launch_block_norm<Bf16, 2>(a, stream);
  else fp16 ? launch_block_norm<Fp16, 4>(a, stream) : launch_block_norm<Bf16, 4>(a, stream);
  return hipGetLastError();
}

}  // namespace jv
