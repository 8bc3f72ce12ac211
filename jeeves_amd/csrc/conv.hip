// Depthwise causal convolution of a ragged batch's tokens, each sequence's
// behind the inputs that its slot holds.
//
// out[t] = act(bias + sum_j w[j] x[t - W + 1 + j]) for each channel, in fp32,
// rounded once. Products and sums are apart and in the order of j, as the
// elementary operations are: what follows is a recurrence, whose states would
// show a 16-bit input that is rounded to the other side.
//
// A lane has 4 channels and a wave 256, for a run of R tokens, so an input row
// is read (R + W - 1) / R times and the weights once a run, all of a run's rows
// under way at a time. Bound by bytes and, as near, by the sigmoids: 11417 tokens
// of 8192 channels in 84 us, 4.4 TB/s with VALU busy 88%; 96 with the exact
// division instead of a corrected reciprocal, 134 with runs of 8 tokens and 8 channels a lane.
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

constexpr int kConvChannels = 256;  // of a wave

template <class H, int W, int R>
__global__ __launch_bounds__(256) void conv_kernel(ConvArgs a, uint32_t channel_blocks) {
  const int lane = threadIdx.x & 63;
  const uint32_t task = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  const int t0 = (int)(task / channel_blocks) * R;
  const int c0 = (int)(task % channel_blocks) * kConvChannels + lane * 4;
  const bool live = c0 < a.channels;
  const int c = live ? c0 : a.channels - 4;
  const Batch& b = a.b;
  if (t0 >= b.tokens) return;
  const auto row = [&](int t) {
    return *reinterpret_cast<const uint2*>(a.x + min(max(t, 0), b.tokens - 1) * a.x_ts + c);
  };
  const auto weights = [&](float (&w)[W][4], float (&bias)[4]) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(a.weight + (int64_t)c * W + i * 4);
      const float vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) w[(i * 4 + e) % W][(i * 4 + e) / W] = vs[e];
    }
    const float4 v = a.bias ? *reinterpret_cast<const float4*>(a.bias + c) : float4{0.0f, 0.0f, 0.0f, 0.0f};
    bias[0] = v.x, bias[1] = v.y, bias[2] = v.z, bias[3] = v.w;
  };
  const auto add = [&](float (&y)[4], uint2 v, const float (&w)[4]) {
    y[0] += H::lo(v.x) * w[0], y[1] += H::hi(v.x) * w[1];
    y[2] += H::lo(v.y) * w[2], y[3] += H::hi(v.y) * w[3];
  };
  const auto store = [&](int t, const float (&y)[4]) {
    float z[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = a.activation ? silu(y[e]) : y[e];
    if (live) *reinterpret_cast<uint2*>(a.out + (int64_t)t * a.channels + c) = uint2{H::pack(z[0], z[1]), H::pack(z[2], z[3])};
  };
  // The inputs before a sequence, zeros where it has none.
  const auto old_inputs = [&](int seq, uint2 (&old)[W - 1]) {
    const int slot = uniform_at(b.from, seq);
    if (slot >= 0 && slot < b.n_slots) {
#pragma unroll
      for (int j = 0; j < W - 1; ++j)
        old[j] = *reinterpret_cast<const uint2*>(a.states + ((int64_t)slot * (W - 1) + j) * a.channels + c);
    } else {
#pragma unroll
      for (int j = 0; j < W - 1; ++j) old[j] = uint2{0, 0};
    }
  };
  const auto keep = [&](int seq, const uint2 (&v)[W - 1]) {
    const int slot = uniform_at(b.slots, seq);
    if (live && slot >= 0 && slot < b.n_slots)
#pragma unroll
      for (int j = 0; j < W - 1; ++j)
        *reinterpret_cast<uint2*>(a.states + ((int64_t)slot * (W - 1) + j) * a.channels + c) = v[j];
  };
  float w[W][4], bias[4];

  if constexpr (R == 1) {
    // One token for each sequence.
    const uint2 x = row(t0);
    uint2 old[W - 1];
    old_inputs(t0, old);
    weights(w, bias);
    float y[4] = {bias[0], bias[1], bias[2], bias[3]};
#pragma unroll
    for (int j = 0; j < W - 1; ++j) add(y, old[j], w[j]);
    add(y, x, w[W - 1]);
    store(t0, y);
#pragma unroll
    for (int j = 0; j + 1 < W - 1; ++j) old[j] = old[j + 1];
    old[W - 2] = x;
    keep(t0, old);
  } else {
    uint2 x[R + W - 1];
#pragma unroll
    for (int i = 0; i < R + W - 1; ++i) x[i] = row(t0 + i - (W - 1));
    weights(w, bias);
    int seq = sequence_of(b, t0);
    int start = seq < 0 ? 0 : uniform_at(b.starts, seq), end = uniform_at(b.starts, seq + 1);
    if (seq >= 0 && t0 - start >= W - 1 && t0 + R <= min(end, b.tokens)) {
      // inside one sequence, behind its first tokens
#pragma unroll
      for (int i = 0; i < R; ++i) {
        float y[4] = {bias[0], bias[1], bias[2], bias[3]};
#pragma unroll
        for (int j = 0; j < W; ++j) add(y, x[i + j], w[j]);
        store(t0 + i, y);
      }
      return;
    }
    uint2 old[W - 1];
    bool began = false;  // the sequence begins in this run
    // Whoever has a sequence's first token reads its state and writes it, so
    // that no other wave's read can follow the write: its first W - 1 tokens
    // are that wave's, also those past its run.
#pragma unroll 1
    for (int i = 0; i < R + W - 2; ++i) {
      const int t = t0 + i;
      if (t >= b.tokens) break;
      while (seq + 1 < b.batch && t >= end) {
        ++seq, began = false;
        start = end, end = uniform_at(b.starts, seq + 1);
      }
      const int place = t - start;
      if (i < R && (seq < 0 || t >= end)) {
        if (live) *reinterpret_cast<uint2*>(a.out + (int64_t)t * a.channels + c) = uint2{0, 0};
        continue;
      }
      if (i < R && place == 0) {
        began = true;
        old_inputs(seq, old);
        const int n = min(end, b.tokens) - start;
        uint2 last[W - 1];
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
      uint2 taps[W];
#pragma unroll
      for (int j = 0; j < W; ++j) taps[j] = row(t + j - (W - 1));
      float y[4] = {bias[0], bias[1], bias[2], bias[3]};
#pragma unroll
      for (int j = 0; j < W; ++j) {
        if (place < W - 1 - j) {
#pragma unroll
          for (int o = 0; o < W - 1; ++o)
            if (place + j == o) taps[j] = old[o];
        }
        add(y, taps[j], w[j]);
      }
      store(t, y);
    }
  }
}

template <class H, int W>
static void launch_conv(const ConvArgs& a, hipStream_t stream) {
  const uint32_t blocks = (uint32_t)(a.channels + kConvChannels - 1) / kConvChannels;
  constexpr int R = 16;
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
