// Depthwise causal convolution of a ragged batch's tokens, each sequence's
// behind the inputs that its slot holds.
//
// out[t] = act(bias + sum_j w[j] x[t - W + 1 + j]) for each channel, in fp32,
// rounded once. Products and sums are apart and in the order of j, as the
// elementary operations are: what follows is a recurrence, whose states would
// show a 16-bit input that is rounded to the other side. A lane has 8 channels and a wave 512, for a run of R tokens, so
// an input row is read (R + W - 1) / R times and the weights once a run.
#include "layer.h"

namespace jv {

// The sequence that token t belongs to: the last whose start is not behind it;
// -1 if there is none. Starts do not decrease, so they are counted, 64 a step.
__device__ __forceinline__ int sequence_of(const Batch& b, int t) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b0 = 0; b0 < b.batch; b0 += 64) {
    const bool before = b0 + lane < b.batch && b.starts[min(b0 + lane, b.batch - 1)] <= t;
    const uint64_t m = __ballot(before);
    n += __popcll(m);
    if (m != ~0ull) break;
  }
  return n - 1;
}

template <class H, int W, int R>
__global__ __launch_bounds__(256) void conv_kernel(ConvArgs a, uint32_t channel_blocks) {
  const int lane = threadIdx.x & 63;
  const uint32_t task = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int t0 = (int)(task / channel_blocks) * R;
  const int c0 = (int)(task % channel_blocks) * 512 + lane * 8;
  const bool live = c0 < a.channels;
  const int c = live ? c0 : a.channels - 8;
  const Batch& b = a.b;
  if (t0 >= b.tokens) return;
  const auto row = [&](int t) {
    return *reinterpret_cast<const uint4*>(a.x + min(max(t, 0), b.tokens - 1) * a.x_ts + c);
  };
  // Inputs of the run, of the W - 1 tokens before it, and of those behind it
  // that a sequence which begins at its end still takes from the state.
  constexpr int N = R > 1 ? R + 2 * (W - 1) - 1 : 1;
  uint4 x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = row(R > 1 ? t0 + i - (W - 1) : t0);
  float w[W][8], bias[8];
#pragma unroll
  for (int i = 0; i < 2 * W; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(a.weight + (int64_t)c * W + i * 4);
    const float vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) w[(i * 4 + e) % W][(i * 4 + e) / W] = vs[e];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 v = a.bias ? *reinterpret_cast<const float4*>(a.bias + c + i * 4) : float4{0.0f, 0.0f, 0.0f, 0.0f};
    bias[i * 4] = v.x, bias[i * 4 + 1] = v.y, bias[i * 4 + 2] = v.z, bias[i * 4 + 3] = v.w;
  }

  const auto add = [&](float (&y)[8], uint4 v, int j) {
    const uint32_t p[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[2 * e] += H::lo(p[e]) * w[j][2 * e];
      y[2 * e + 1] += H::hi(p[e]) * w[j][2 * e + 1];
    }
  };
  const auto store = [&](int t, const float (&y)[8]) {
    float z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = a.activation ? silu(y[e]) : y[e];
    if (live)
      *reinterpret_cast<uint4*>(a.out + (int64_t)t * a.channels + c) =
          uint4{H::pack(z[0], z[1]), H::pack(z[2], z[3]), H::pack(z[4], z[5]), H::pack(z[6], z[7])};
  };
  // The inputs before a sequence, zeros where it has none.
  const auto old_inputs = [&](int seq, uint4 (&old)[W - 1]) {
    const int slot = uniform_at(b.from, seq);
    if (slot >= 0 && slot < b.n_slots) {
#pragma unroll
      for (int j = 0; j < W - 1; ++j)
        old[j] = *reinterpret_cast<const uint4*>(a.states + ((int64_t)slot * (W - 1) + j) * a.channels + c);
    } else {
#pragma unroll
      for (int j = 0; j < W - 1; ++j) old[j] = uint4{0, 0, 0, 0};
    }
  };
  const auto keep = [&](int seq, const uint4 (&v)[W - 1]) {
    const int slot = uniform_at(b.slots, seq);
    if (live && slot >= 0 && slot < b.n_slots)
#pragma unroll
      for (int j = 0; j < W - 1; ++j)
        *reinterpret_cast<uint4*>(a.states + ((int64_t)slot * (W - 1) + j) * a.channels + c) = v[j];
  };

  if constexpr (R == 1) {
    // One token for each sequence.
    uint4 old[W - 1];
    old_inputs(t0, old);
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = bias[e];
#pragma unroll
    for (int j = 0; j < W - 1; ++j) add(y, old[j], j);
    add(y, x[0], W - 1);
    store(t0, y);
#pragma unroll
    for (int j = 0; j + 1 < W - 1; ++j) old[j] = old[j + 1];
    old[W - 2] = x[0];
    keep(t0, old);
  } else {
    int seq = sequence_of(b, t0);
    int start = seq < 0 ? 0 : uniform_at(b.starts, seq), end = uniform_at(b.starts, seq + 1);
    uint4 old[W - 1];
    bool began = false;  // the sequence begins in this run
    // Whoever has a sequence's first token reads its state and writes it, so
    // that no other wave's read can follow the write: its first W - 1 tokens
    // are that wave's, also those past its run.
#pragma unroll
    for (int i = 0; i < R + W - 2; ++i) {
      const int t = t0 + i;
      if (t >= b.tokens) break;
      while (seq + 1 < b.batch && t >= end) {
        ++seq, began = false;
        start = end, end = uniform_at(b.starts, seq + 1);
      }
      const int place = t - start;
      if (i < R && (seq < 0 || t >= end)) {
        if (live) *reinterpret_cast<uint4*>(a.out + (int64_t)t * a.channels + c) = uint4{0, 0, 0, 0};
        continue;
      }
      if (i < R && place == 0) {
        began = true;
        old_inputs(seq, old);
        const int n = min(end, b.tokens) - start;
        uint4 last[W - 1];
#pragma unroll
        for (int j = 0; j < W - 1; ++j) last[j] = row(start + n - (W - 1) + j);
#pragma unroll
        for (int j = 0; j < W - 1; ++j)
#pragma unroll
          for (int o = 0; o < W - 1; ++o)
            if (n + j == o) last[j] = old[o];
        keep(seq, last);
      }
      // its first tokens are the wave's that has the very first
      if (place < W - 1 && !began) continue;
      if (i >= R && (place >= W - 1 || t >= end || seq < 0)) break;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = bias[e];
#pragma unroll
      for (int j = 0; j < W; ++j) {
        uint4 v = x[i + j];
        if (place < W - 1 - j) {
#pragma unroll
          for (int o = 0; o < W - 1; ++o)
            if (place + j == o) v = old[o];
        }
        add(y, v, j);
      }
      store(t, y);
    }
  }
}

template <class H, int W>
static void launch_conv(const ConvArgs& a, hipStream_t stream) {
  const uint32_t blocks = (uint32_t)(a.channels + 511) / 512;
  constexpr int R = 8;
  const uint32_t runs = a.b.starts ? (uint32_t)(a.b.tokens + R - 1) / R : (uint32_t)a.b.tokens;
  const uint32_t grid = (uint32_t)(((uint64_t)runs * blocks + 3) / 4);
  if (a.b.starts) conv_kernel<H, W, R><<<grid, 256, 0, stream>>>(a, blocks);
  else conv_kernel<H, W, 1><<<grid, 256, 0, stream>>>(a, blocks);
}

hipError_t causal_conv(const ConvArgs& a, int width, bool fp16, hipStream_t stream) {
  if (width == 2) fp16 ? launch_conv<Fp16, 2>(a, stream) : launch_conv<Bf16, 2>(a, stream);
  else if (width == 3) fp16 ? launch_conv<Fp16, 3>(a, stream) : launch_conv<Bf16, 3>(a, stream);
  else if (width == 4) fp16 ? launch_conv<Fp16, 4>(a, stream) : launch_conv<Bf16, 4>(a, stream);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

}  // namespace jv
