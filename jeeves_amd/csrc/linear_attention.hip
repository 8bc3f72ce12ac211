// Linear attention with a state S [DK, DV] for each value head and a decay for
// each head and token, with the delta rule's correction or without:
//   S = e^g S;  u = beta (v - S^T k);  S = S + k u^T;  o = scale S^T q
// (u = v without the correction).
//
// Single tokens (step_kernel) are a read and a write of the states.
//
// Prompts go in chunks of C = 64 tokens. With G_i the sum of the log decays of
// a chunk's tokens up to i, and the state S before the chunk, the recurrence is
//   (I + A) U = beta (V - e^G K S),  A_ij = beta_i e^(G_i - G_j) k_i.k_j  (j < i)
//   O = scale (e^G Q S + M U),       M_ij = e^(G_i - G_j) q_i.k_j         (j <= i)
//   S' = e^(G_C) S + K^T (e^(G_C - G) U)
// prepare_kernel works out for all chunks at a time what does not depend on S:
// T = (I + A)^-1 by forward substitution in fp32, M, the rows' factors and K's
// transpose, all in the order in which scan_kernel's products read them.
// scan_kernel goes through a sequence's chunks with its part of S in registers.
//
// Rounding. States, sums, decays and norms are fp32 (the sums G fp64: their
// differences are what counts). The products are MFMAs of bf16: K and Q are
// exact (one bf16, or two for fp16), and what is fp32 goes in as the sum of
// three bf16 values (24 bits) towards the state, of two (16 bits) towards the
// outputs, which are rounded to 8 or 11 bits once.
#include "layer.h"

namespace jv {

constexpr int kStepCols = 32;  // columns of S that a workgroup of step_kernel has
constexpr int kCols = 32;      // and one of scan_kernel

template <class H>
__device__ __forceinline__ float gate_at(const void* p, int wide16, int64_t i) {
  return wide16 ? H::lo(reinterpret_cast<const uint16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}

// log2 of a token's decay; what is below 2^-14400 is 0 by far.
__device__ __forceinline__ double log2_decay(const LinearArgs& a, float z, int head) {
  if (a.rate) z = -a.rate[head] * softplus(z + (a.decay_bias ? a.decay_bias[head] : 0.0f));
  const double g = (double)z * 1.4426950408889634;
  return g < -14400.0 ? -14400.0 : g;
}

__device__ __forceinline__ float beta_of(const LinearArgs& a, float z) { return a.rate ? sigmoid(z) : z; }

// ---------------------------------------------------------------------------
// One token for each sequence. A workgroup has kStepCols columns of a head's
// state, a thread 4 columns of every 32nd row; S^T k and S^T q come from the
// state before the token (o = e^g S^T q + (q.k) u), so that one exchange
// between the waves serves both. Bound by the states' bytes.
// ---------------------------------------------------------------------------
template <class H, int DK>
__global__ __launch_bounds__(256) void step_kernel(LinearArgs a, int v_dim, uint32_t col_blocks) {
  constexpr int NR = DK / 32;
  __shared__ float parts[2][4][kStepCols];
  const uint32_t block = blockIdx.x, cb = block % col_blocks, rest = block / col_blocks;
  const int head = (int)(rest % (uint32_t)a.v_heads), seq = (int)(rest / (uint32_t)a.v_heads), kh = head / a.group;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, rg = tid >> 3, col = (int)cb * kStepCols + (tid & 7) * 4;
  const int from = uniform_at(a.b.from, seq), to = uniform_at(a.b.slots, seq);
  const bool have = from >= 0 && from < a.b.n_slots, keep = to >= 0 && to < a.b.n_slots;
  const int64_t slot_size = (int64_t)DK * v_dim;
  const uint16_t *q = a.q + seq * a.q_ts + kh * a.q_hs, *k = a.k + seq * a.k_ts + kh * a.k_hs;
  float4 s[NR];
  if (have) {
    const float* p = a.states + ((int64_t)from * a.v_heads + head) * slot_size + col;
#pragma unroll
    for (int i = 0; i < NR; ++i) s[i] = *reinterpret_cast<const float4*>(p + (rg + 32 * i) * v_dim);
  } else {
#pragma unroll
    for (int i = 0; i < NR; ++i) s[i] = float4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const uint2 vv = *reinterpret_cast<const uint2*>(a.v + seq * a.v_ts + head * a.v_hs + col);
  float kr[NR], qr[NR], kl[DK / 64], ql[DK / 64];
#pragma unroll
  for (int i = 0; i < NR; ++i) kr[i] = H::lo(k[rg + 32 * i]), qr[i] = H::lo(q[rg + 32 * i]);
#pragma unroll
  for (int i = 0; i < DK / 64; ++i) kl[i] = H::lo(k[lane + 64 * i]), ql[i] = H::lo(q[lane + 64 * i]);
  const float decay = __builtin_amdgcn_exp2f((float)log2_decay(a, gate_at<H>(a.decay, a.gates16, seq * a.decay_ts + head), head));
  const float beta = a.beta ? beta_of(a, gate_at<H>(a.beta, a.gates16, seq * a.beta_ts + head)) : 1.0f;
  float kk = 0.0f, qq = 0.0f, qk = 0.0f;
#pragma unroll
  for (int i = 0; i < DK / 64; ++i) {
    kk = __builtin_fmaf(kl[i], kl[i], kk), qq = __builtin_fmaf(ql[i], ql[i], qq), qk = __builtin_fmaf(ql[i], kl[i], qk);
  }
  float rk = 1.0f, rq = a.scale;
  qk = wave_sum(qk);
  if (a.norm_eps > 0.0f) rk = inv_sqrt(wave_sum(kk) + a.norm_eps), rq = a.scale * inv_sqrt(wave_sum(qq) + a.norm_eps);
  float4 pk = {0.0f, 0.0f, 0.0f, 0.0f}, pq = pk;
#pragma unroll
  for (int i = 0; i < NR; ++i) {
    pk.x = __builtin_fmaf(kr[i], s[i].x, pk.x), pk.y = __builtin_fmaf(kr[i], s[i].y, pk.y);
    pk.z = __builtin_fmaf(kr[i], s[i].z, pk.z), pk.w = __builtin_fmaf(kr[i], s[i].w, pk.w);
    pq.x = __builtin_fmaf(qr[i], s[i].x, pq.x), pq.y = __builtin_fmaf(qr[i], s[i].y, pq.y);
    pq.z = __builtin_fmaf(qr[i], s[i].z, pq.z), pq.w = __builtin_fmaf(qr[i], s[i].w, pq.w);
  }
#pragma unroll
  for (int m = 8; m < 64; m *= 2) {
    pk.x += __shfl_xor(pk.x, m), pk.y += __shfl_xor(pk.y, m), pk.z += __shfl_xor(pk.z, m), pk.w += __shfl_xor(pk.w, m);
    pq.x += __shfl_xor(pq.x, m), pq.y += __shfl_xor(pq.y, m), pq.z += __shfl_xor(pq.z, m), pq.w += __shfl_xor(pq.w, m);
  }
  const int cl = (tid & 7) * 4;
  if (lane < 8) {
    *reinterpret_cast<float4*>(&parts[0][wave][cl]) = pk;
    *reinterpret_cast<float4*>(&parts[1][wave][cl]) = pq;
  }
  __syncthreads();
  float u[4], o[4];
  const float v[4] = {H::lo(vv.x), H::hi(vv.x), H::lo(vv.y), H::hi(vv.y)};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float sk = (parts[0][0][cl + e] + parts[0][1][cl + e]) + (parts[0][2][cl + e] + parts[0][3][cl + e]);
    const float sq = (parts[1][0][cl + e] + parts[1][1][cl + e]) + (parts[1][2][cl + e] + parts[1][3][cl + e]);
    u[e] = a.beta ? beta * (v[e] - decay * rk * sk) : v[e];
    o[e] = rq * __builtin_fmaf(rk * qk, u[e], decay * sq);
  }
  if (tid < 8)
    *reinterpret_cast<uint2*>(a.out + ((int64_t)seq * a.v_heads + head) * v_dim + col) = uint2{H::pack(o[0], o[1]), H::pack(o[2], o[3])};
  if (keep) {
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const float kn = rk * kr[i];
      const float4 n = {__builtin_fmaf(kn, u[0], decay * s[i].x), __builtin_fmaf(kn, u[1], decay * s[i].y),
                        __builtin_fmaf(kn, u[2], decay * s[i].z), __builtin_fmaf(kn, u[3], decay * s[i].w)};
      *reinterpret_cast<float4*>(a.states + ((int64_t)to * a.v_heads + head) * slot_size + (rg + 32 * i) * v_dim + col) = n;
    }
  }
}

// ---------------------------------------------------------------------------
// Prompts. MFMA 16x16x32: a lane's 8 values of A are row lane % 16, k = 8
// (lane / 16) .., of B column lane % 16, the same k; its 4 results are column
// lane % 16, rows 4 (lane / 16) ...
// ---------------------------------------------------------------------------
typedef short bits8 __attribute__((ext_vector_type(8)));

// A chunk's data for a value head in the workspace, in fragments of 64 lanes
// of 16 bytes: T [row tile][32 columns][3 parts], M [row tile][32 columns]
// [2 parts], then the rows' factors.
constexpr int kFragment = 1024;
constexpr int kBytesT = 4 * 2 * 3 * kFragment, kBytesM = 4 * 2 * 2 * kFragment;
enum { kFromK, kFromQ, kBeta, kToEnd, kEnd, kFactors };  // [kFactors][64] floats; kEnd: the whole chunk's decay
constexpr int kBytesHead = kBytesT + kBytesM + kFactors * kChunk * 4;

// K's transpose for a key head: [DK / 16][32 tokens] fragments.
constexpr int bytes_kt(int k_dim) { return k_dim * kChunk * 2; }

int64_t linear_workspace(int64_t tokens, int64_t batch, int64_t k_heads, int64_t v_heads, int64_t k_dim, bool beta) {
  return linear_chunks(tokens, batch) * (v_heads * kBytesHead + k_heads * bytes_kt((int)k_dim));
}

__device__ __forceinline__ uint8_t* head_data(const LinearArgs& a, int chunk, int head) {
  return a.workspace + ((int64_t)chunk * a.v_heads + head) * kBytesHead;
}
__device__ __forceinline__ uint8_t* key_data(const LinearArgs& a, int chunk, int kh, int k_dim) {
  return a.workspace + linear_chunks(a.b.tokens, a.b.batch) * a.v_heads * kBytesHead +
         ((int64_t)chunk * a.k_heads + kh) * bytes_kt(k_dim);
}

// Two fp32 values as sums of bf16 ones: x = p0 + p1 + p2 to 24 bits.
template <int N>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&p)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = Bf16::pack(x, y);
    x -= Bf16::lo(p[i]), y -= Bf16::hi(p[i]);
  }
}

// A fragment of the tensors' type as bf16 ones whose sum it is.
template <class H>
struct Parts;
template <>
struct Parts<Bf16> {
  static constexpr int n = 1;
  static __device__ __forceinline__ void of(i32x4 v, i32x4 (&p)[1]) { p[0] = v; }
};
template <>
struct Parts<Fp16> {
  static constexpr int n = 2;
  static __device__ __forceinline__ void of(i32x4 v, i32x4 (&p)[2]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t s[2];
      split2<2>(Fp16::lo((uint32_t)v[e]), Fp16::hi((uint32_t)v[e]), s);
      p[0][e] = (int)s[0], p[1][e] = (int)s[1];
    }
  }
};

__device__ __forceinline__ int clamp_to(int v, int hi) { return min(max(v, 0), hi); }

template <class H, int DK, bool BETA>
__global__ __launch_bounds__(256) void prepare_kernel(LinearArgs a) {
  constexpr int KS = DK / 32, kRow = 68, kRow16 = 72;
  __shared__ __attribute__((aligned(16))) float tri[BETA ? kChunk * kRow : 4];
  __shared__ __attribute__((aligned(16))) uint16_t m16[2][kChunk * kRow16];
  __shared__ __attribute__((aligned(16))) uint16_t kt[DK * kRow16];
  __shared__ double sum[kChunk];
  __shared__ float rk[kChunk], rq[kChunk], betas[kChunk];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int place = (int)(blockIdx.x / (uint32_t)a.v_heads), head = (int)(blockIdx.x % (uint32_t)a.v_heads), kh = head / a.group;
  const Batch& b = a.b;

  // the sequence whose chunk this is
  int count = 0;
  for (int b0 = 0; b0 < b.batch; b0 += 64) {
    const int i = min(b0 + lane, b.batch - 1);
    const bool before = b0 + lane < b.batch && clamp_to(b.starts[i], b.tokens) / kChunk + i <= place;
    const uint64_t m = __ballot(before);
    count += __popcll(m);
    if (m != ~0ull) break;
  }
  if (count == 0) return;
  const int seq = count - 1, start = clamp_to(uniform_at(b.starts, seq), b.tokens);
  const int n = clamp_to(uniform_at(b.starts, seq + 1), b.tokens) - start;
  const int t0 = (place - start / kChunk - seq) * kChunk, rows = min(n - t0, kChunk);
  if (t0 < 0 || rows <= 0) return;
  const int first = start + t0;

  const int r16 = lane & 15, k8 = (lane >> 4) * 8;
  const auto fragment = [&](const uint16_t* p, int64_t ts, int64_t hs, int tile, int s) {
    const int i = tile * 16 + r16;
    const i32x4 v = *reinterpret_cast<const i32x4*>(p + (int64_t)(first + min(i, rows - 1)) * ts + kh * hs + s * 32 + k8);
    return v & ((i - rows) >> 31);  // 0 behind the sequence's end
  };
  i32x4 kf[KS], qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) kf[s] = fragment(a.k, a.k_ts, a.k_hs, wave, s), qf[s] = fragment(a.q, a.q_ts, a.q_hs, wave, s);
  if (wave == 0) {
    const int t = first + min(lane, rows - 1);
    const bool real = lane < rows;
    double g = real ? log2_decay(a, gate_at<H>(a.decay, a.gates16, t * a.decay_ts + head), head) : 0.0;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
      const double o = __shfl_up(g, s);
      if (lane >= s) g += o;
    }
    sum[lane] = g;
    betas[lane] = !real ? 0.0f : BETA ? beta_of(a, gate_at<H>(a.beta, a.gates16, t * a.beta_ts + head)) : 1.0f;
  }
  {
    float sk = 0.0f, sq = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float k0 = H::lo((uint32_t)kf[s][e]), k1 = H::hi((uint32_t)kf[s][e]);
        const float q0 = H::lo((uint32_t)qf[s][e]), q1 = H::hi((uint32_t)qf[s][e]);
        sk = __builtin_fmaf(k0, k0, __builtin_fmaf(k1, k1, sk)), sq = __builtin_fmaf(q0, q0, __builtin_fmaf(q1, q1, sq));
      }
    sk += __shfl_xor(sk, 16), sk += __shfl_xor(sk, 32), sq += __shfl_xor(sq, 16), sq += __shfl_xor(sq, 32);
    if (lane < 16) {
      const bool norm = a.norm_eps > 0.0f;
      rk[wave * 16 + lane] = norm ? inv_sqrt(sk + a.norm_eps) : 1.0f;
      rq[wave * 16 + lane] = a.scale * (norm ? inv_sqrt(sq + a.norm_eps) : 1.0f);
    }
  }
  if (head % a.group == 0) {
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        kt[(s * 32 + k8 + e) * kRow16 + wave * 16 + r16] = (uint16_t)((uint32_t)kf[s][e >> 1] >> (16 * (e & 1)));
  }
  __syncthreads();

  // A and M, 16 rows a wave, their column tiles up to the diagonal
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if (t > (wave | 1)) break;
    f32x4 kk = {0.0f, 0.0f, 0.0f, 0.0f}, qk = kk;
    if (t <= wave) {
      i32x4 kb[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s) kb[s] = fragment(a.k, a.k_ts, a.k_hs, t, s);
#pragma unroll
      for (int s = 0; s < KS; ++s) kk = H::mfma16(kf[s], kb[s], kk), qk = H::mfma16(qf[s], kb[s], qk);
    }
    const int j = t * 16 + r16;
    const double gj = sum[j];
    const float rkj = rk[j];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = wave * 16 + (lane >> 4) * 4 + r;
      const float e = __builtin_amdgcn_exp2f((float)(sum[i] - gj)) * rkj;
      if (BETA) tri[i * kRow + j] = j < i ? kk[r] * e * rk[i] * betas[i] : 0.0f;
      uint32_t p[2];
      split2<2>(j <= i ? qk[r] * e * rq[i] : 0.0f, 0.0f, p);
      m16[0][i * kRow16 + j] = (uint16_t)p[0], m16[1][i * kRow16 + j] = (uint16_t)p[1];
    }
  }
  uint8_t* out = head_data(a, place, head);
  if (wave == 3) {
    const double g = sum[lane], all = sum[kChunk - 1];
    const float from = __builtin_amdgcn_exp2f((float)g);
    float* f = reinterpret_cast<float*>(out + kBytesT + kBytesM);
    f[kFromK * kChunk + lane] = from * rk[lane], f[kFromQ * kChunk + lane] = from * rq[lane];
    f[kBeta * kChunk + lane] = betas[lane];
    f[kToEnd * kChunk + lane] = __builtin_amdgcn_exp2f((float)(all - g)) * rk[lane];
    f[kEnd * kChunk + lane] = __builtin_amdgcn_exp2f((float)all);
  }
  __syncthreads();

  if constexpr (BETA) {
    if (wave == 0) {
      // column `lane` of T by forward substitution
      float x[kChunk];
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        float s[4] = {lane == i ? 1.0f : 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < i; j += 4) {
          const float4 r = *reinterpret_cast<const float4*>(&tri[i * kRow + j]);
          s[0] = __builtin_fmaf(-r.x, x[j], s[0]);
          if (j + 1 < i) s[1] = __builtin_fmaf(-r.y, x[j + 1], s[1]);
          if (j + 2 < i) s[2] = __builtin_fmaf(-r.z, x[j + 2], s[2]);
          if (j + 3 < i) s[3] = __builtin_fmaf(-r.w, x[j + 3], s[3]);
        }
        x[i] = i < lane ? 0.0f : (s[0] + s[1]) + (s[2] + s[3]);
      }
#pragma unroll
      for (int i = 0; i < kChunk; ++i) tri[i * kRow + lane] = x[i];
    }
    __syncthreads();
  }
  for (int s = 0; s <= wave >> 1; ++s) {
    const int at = (wave * 16 + r16), col = s * 32 + k8;
    i32x4* m = reinterpret_cast<i32x4*>(out + kBytesT) + (wave * 2 + s) * 2 * 64 + lane;
#pragma unroll
    for (int p = 0; p < 2; ++p) m[p * 64] = *reinterpret_cast<const i32x4*>(&m16[p][at * kRow16 + col]);
    if constexpr (BETA) {
      const float4 x = *reinterpret_cast<const float4*>(&tri[at * kRow + col]), y = *reinterpret_cast<const float4*>(&tri[at * kRow + col + 4]);
      uint32_t p[4][3];
      split2<3>(x.x, x.y, p[0]), split2<3>(x.z, x.w, p[1]), split2<3>(y.x, y.y, p[2]), split2<3>(y.z, y.w, p[3]);
      i32x4* t = reinterpret_cast<i32x4*>(out) + (wave * 2 + s) * 3 * 64 + lane;
#pragma unroll
      for (int i = 0; i < 3; ++i) t[i * 64] = i32x4{(int)p[0][i], (int)p[1][i], (int)p[2][i], (int)p[3][i]};
    }
  }
  if (head % a.group == 0) {
    i32x4* dst = reinterpret_cast<i32x4*>(key_data(a, place, kh, DK)) + lane;
    for (int f = wave; f < DK / 16 * 2; f += 4)
      dst[f * 64] = *reinterpret_cast<const i32x4*>(&kt[((f >> 1) * 16 + r16) * kRow16 + (f & 1) * 32 + k8]);
  }
}

__device__ __forceinline__ f32x4 mfma_bf16(i32x4 a, i32x4 b, f32x4 c) { return Bf16::mfma16(a, b, c); }

// A sequence's chunks one after the other, kCols columns of a head's state a
// workgroup, wave w with the state's rows from w DK / 4 on and a chunk's rows
// from 16 w on. Three exchanges through LDS a chunk: the state (as the right
// operand of K S and Q S), the differences D = beta (V - e^G K S), and U.
template <class H, int DK, bool BETA>
__global__ __launch_bounds__(256) void scan_kernel(LinearArgs a, int v_dim, uint32_t col_blocks) {
  constexpr int KS = DK / 32, MT = DK / 64, NT = kCols / 16, NP = Parts<H>::n;
  constexpr int kRowS = DK + 8, kRowU = kChunk + 8;
  __shared__ __attribute__((aligned(16))) uint16_t sb[3][kCols * kRowS];
  __shared__ __attribute__((aligned(16))) uint16_t db[BETA ? 3 : 1][kCols * kRowU];
  __shared__ __attribute__((aligned(16))) uint16_t ub[5][kCols * kRowU];  // U in 2 parts, e^(G_C - G) U in 3
  __shared__ int first_d[kCols], first_us[2][kCols];  // a column's first row that is not finite; U's by turns
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t cb = blockIdx.x % col_blocks, rest = blockIdx.x / col_blocks;
  const int head = (int)(rest % (uint32_t)a.v_heads), seq = (int)(rest / (uint32_t)a.v_heads), kh = head / a.group;
  const Batch& b = a.b;
  const int start = clamp_to(uniform_at(b.starts, seq), b.tokens), n = clamp_to(uniform_at(b.starts, seq + 1), b.tokens) - start;
  if (n <= 0) return;
  const int from = uniform_at(b.from, seq), to = uniform_at(b.slots, seq);
  const int r16 = lane & 15, r4 = (lane >> 4) * 4, k8 = (lane >> 4) * 8, col0 = (int)cb * kCols + r16;
  const int64_t slot_size = (int64_t)DK * v_dim;
  const int chunk0 = start / kChunk + seq;

  f32x4 s[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < NT; ++c) s[m][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (from >= 0 && from < b.n_slots) {
    const float* p = a.states + ((int64_t)from * a.v_heads + head) * slot_size + (wave * (DK / 4) + r4) * v_dim + col0;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[m][c][r] = p[(m * 16 + r) * v_dim + c * 16];
  }
  if (tid < kCols) first_d[tid] = first_us[chunk0 & 1][tid] = kChunk;

  for (int t0 = 0; t0 < n; t0 += kChunk) {
    const int rows = min(n - t0, kChunk), first = start + t0, place = chunk0 + t0 / kChunk;
    const uint8_t* data = head_data(a, place, head);
    // this chunk's operands
    i32x4 kf[KS], qf[KS];
    {
      const int i = wave * 16 + r16;
      const int64_t t = first + min(i, rows - 1);
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        kf[x] = *reinterpret_cast<const i32x4*>(a.k + t * a.k_ts + kh * a.k_hs + x * 32 + k8);
        qf[x] = *reinterpret_cast<const i32x4*>(a.q + t * a.q_ts + kh * a.q_hs + x * 32 + k8);
      }
#pragma unroll
      for (int x = 0; x < KS; ++x) kf[x] &= (i - rows) >> 31, qf[x] &= (i - rows) >> 31;
    }
    i32x4 tf[BETA ? 2 : 1][3], mf[2][2], kt[2][MT];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if constexpr (BETA) {
#pragma unroll
        for (int i = 0; i < 3; ++i) tf[x][i] = reinterpret_cast<const i32x4*>(data)[((wave * 2 + (x & (wave >> 1))) * 3 + i) * 64 + lane];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        mf[x][i] = reinterpret_cast<const i32x4*>(data + kBytesT)[((wave * 2 + (x & (wave >> 1))) * 2 + i) * 64 + lane];
#pragma unroll
      for (int m = 0; m < MT; ++m)
        kt[x][m] = reinterpret_cast<const i32x4*>(key_data(a, place, kh, DK))[((wave * MT + m) * 2 + x) * 64 + lane];
    }
    float v[NT][4];
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = wave * 16 + r4 + r;
        const uint16_t x = a.v[(int64_t)(first + min(i, rows - 1)) * a.v_ts + head * a.v_hs + col0 + c * 16];
        v[c][r] = H::lo((uint32_t)x & (uint32_t)((i - rows) >> 31));  // 0 behind the sequence's end
      }
    const float* f = reinterpret_cast<const float*>(data + kBytesT + kBytesM) + wave * 16 + r4;
    const f32x4 from_k = *reinterpret_cast<const f32x4*>(f + kFromK * kChunk), from_q = *reinterpret_cast<const f32x4*>(f + kFromQ * kChunk);
    const f32x4 beta = *reinterpret_cast<const f32x4*>(f + kBeta * kChunk), to_end = *reinterpret_cast<const f32x4*>(f + kToEnd * kChunk);
    const float end = f[kEnd * kChunk];

    // the state in three parts, columns as rows
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        uint32_t p[2][3];
        split2<3>(s[m][c][0], s[m][c][1], p[0]), split2<3>(s[m][c][2], s[m][c][3], p[1]);
#pragma unroll
        for (int i = 0; i < 3; ++i)
          *reinterpret_cast<uint2*>(&sb[i][(c * 16 + r16) * kRowS + wave * (DK / 4) + m * 16 + r4]) = uint2{p[0][i], p[1][i]};
      }
    __syncthreads();
    int* first_u = first_us[place & 1];
    if (tid < kCols) first_us[(place + 1) & 1][tid] = kChunk;

    f32x4 pk[NT], pq[NT];
#pragma unroll
    for (int c = 0; c < NT; ++c) pk[c] = pq[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      i32x4 kp[NP], qp[NP];
      Parts<H>::of(kf[x], kp), Parts<H>::of(qf[x], qp);
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        i32x4 sp[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) sp[i] = *reinterpret_cast<const i32x4*>(&sb[i][(c * 16 + r16) * kRowS + x * 32 + k8]);
        if (BETA) {
#pragma unroll
          for (int i = 0; i < 3; ++i) pk[c] = mfma_bf16(kp[0], sp[i], pk[c]);
          if (NP > 1) pk[c] = mfma_bf16(kp[NP - 1], sp[0], mfma_bf16(kp[NP - 1], sp[1], pk[c]));
        }
        pq[c] = mfma_bf16(qp[0], sp[0], mfma_bf16(qp[0], sp[1], pq[c]));
        if (NP > 1) pq[c] = mfma_bf16(qp[NP - 1], sp[0], pq[c]);
      }
    }

    f32x4 u[NT];
    if constexpr (BETA) {
      uint32_t bad = 0;
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        float d[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          d[r] = beta[r] * (v[c][r] - from_k[r] * pk[c][r]);
          if (!(__builtin_fabsf(d[r]) < __builtin_inff())) bad |= 1u << (c * 4 + r);
        }
        uint32_t p[2][3];
        split2<3>(d[0], d[1], p[0]), split2<3>(d[2], d[3], p[1]);
#pragma unroll
        for (int i = 0; i < 3; ++i)
          *reinterpret_cast<uint2*>(&db[i][(c * 16 + r16) * kRowU + wave * 16 + r4]) = uint2{p[0][i], p[1][i]};
      }
      if (__ballot(bad != 0)) {
#pragma unroll
        for (int c = 0; c < NT; ++c)
          if ((bad >> (4 * c)) & 15) atomicMin(&first_d[c * 16 + r16], wave * 16 + r4 + __builtin_ctz((bad >> (4 * c)) & 15));
      }
      __syncthreads();
      const bool spoilt = __ballot(first_d[lane & (kCols - 1)] < kChunk) != 0;
      if (spoilt) {
        // rows behind a column's first one that is not finite must not reach those before it
        for (int i = tid; i < kCols * kChunk; i += 256)
          if ((i & (kChunk - 1)) >= first_d[i / kChunk])
            db[0][i / kChunk * kRowU + (i & (kChunk - 1))] = db[1][i / kChunk * kRowU + (i & (kChunk - 1))] =
                db[2][i / kChunk * kRowU + (i & (kChunk - 1))] = 0;
        __syncthreads();
      }
#pragma unroll
      for (int c = 0; c < NT; ++c) u[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (x > (wave >> 1)) break;
        const i32x4* t = tf[x];
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          i32x4 d[3];
#pragma unroll
          for (int i = 0; i < 3; ++i) d[i] = *reinterpret_cast<const i32x4*>(&db[i][(c * 16 + r16) * kRowU + x * 32 + k8]);
          u[c] = mfma_bf16(t[0], d[2], u[c]), u[c] = mfma_bf16(t[2], d[0], u[c]), u[c] = mfma_bf16(t[1], d[1], u[c]);
          u[c] = mfma_bf16(t[0], d[1], u[c]), u[c] = mfma_bf16(t[1], d[0], u[c]), u[c] = mfma_bf16(t[0], d[0], u[c]);
        }
      }
      if (spoilt) {
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (wave * 16 + r4 + r >= first_d[c * 16 + r16]) u[c][r] = __builtin_nanf("");
      }
    } else {
#pragma unroll
      for (int c = 0; c < NT; ++c) u[c] = f32x4{v[c][0], v[c][1], v[c][2], v[c][3]};
    }

    {
      uint32_t bad = 0;
#pragma unroll
      for (int c = 0; c < NT; ++c) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!(__builtin_fabsf(u[c][r]) < __builtin_inff())) bad |= 1u << (c * 4 + r);
        uint32_t p[2][2], w[2][3];
        split2<2>(u[c][0], u[c][1], p[0]), split2<2>(u[c][2], u[c][3], p[1]);
        split2<3>(u[c][0] * to_end[0], u[c][1] * to_end[1], w[0]), split2<3>(u[c][2] * to_end[2], u[c][3] * to_end[3], w[1]);
        const int at = (c * 16 + r16) * kRowU + wave * 16 + r4;
#pragma unroll
        for (int i = 0; i < 2; ++i) *reinterpret_cast<uint2*>(&ub[i][at]) = uint2{p[0][i], p[1][i]};
#pragma unroll
        for (int i = 0; i < 3; ++i) *reinterpret_cast<uint2*>(&ub[2 + i][at]) = uint2{w[0][i], w[1][i]};
      }
      if (__ballot(bad != 0)) {
#pragma unroll
        for (int c = 0; c < NT; ++c)
          if ((bad >> (4 * c)) & 15) atomicMin(&first_u[c * 16 + r16], wave * 16 + r4 + __builtin_ctz((bad >> (4 * c)) & 15));
      }
    }
    __syncthreads();
    const bool spoilt = __ballot(first_u[lane & (kCols - 1)] < kChunk) != 0;
    if (spoilt) {
      for (int i = tid; i < kCols * kChunk; i += 256)
        if ((i & (kChunk - 1)) >= first_u[i / kChunk])
#pragma unroll
          for (int p = 0; p < 5; ++p) ub[p][i / kChunk * kRowU + (i & (kChunk - 1))] = 0;
      __syncthreads();
    }
    if (tid < kCols) first_d[tid] = kChunk;

    // the chunk's outputs
    f32x4 o[NT];
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[c][r] = from_q[r] * pq[c][r];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (x > (wave >> 1)) break;
      const i32x4* m = mf[x];
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const i32x4 u0 = *reinterpret_cast<const i32x4*>(&ub[0][(c * 16 + r16) * kRowU + x * 32 + k8]);
        const i32x4 u1 = *reinterpret_cast<const i32x4*>(&ub[1][(c * 16 + r16) * kRowU + x * 32 + k8]);
        o[c] = mfma_bf16(m[1], u0, o[c]), o[c] = mfma_bf16(m[0], u1, o[c]), o[c] = mfma_bf16(m[0], u0, o[c]);
      }
    }
    // the state behind the chunk
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < NT; ++c) s[m][c] *= end;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        i32x4 up[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) up[i] = *reinterpret_cast<const i32x4*>(&ub[2 + i][(c * 16 + r16) * kRowU + x * 32 + k8]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          i32x4 kp[NP];
          Parts<H>::of(kt[x][m], kp);
          s[m][c] = mfma_bf16(kp[0], up[2], s[m][c]), s[m][c] = mfma_bf16(kp[0], up[1], s[m][c]);
          if (NP > 1) s[m][c] = mfma_bf16(kp[NP - 1], up[1], s[m][c]), s[m][c] = mfma_bf16(kp[NP - 1], up[0], s[m][c]);
          s[m][c] = mfma_bf16(kp[0], up[0], s[m][c]);
        }
      }
    }
    if (spoilt) {
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const int bad = first_u[c * 16 + r16];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (wave * 16 + r4 + r >= bad) o[c][r] = __builtin_nanf("");
        if (bad < kChunk)
#pragma unroll
          for (int m = 0; m < MT; ++m) s[m][c] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
      }
    }
#pragma unroll
    for (int c = 0; c < NT; ++c) {
      const uint32_t p[2] = {H::pack(o[c][0], o[c][1]), H::pack(o[c][2], o[c][3])};
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = wave * 16 + r4 + r;
        if (i < rows) a.out[((int64_t)(first + i) * a.v_heads + head) * v_dim + col0 + c * 16] = (uint16_t)(p[r >> 1] >> (16 * (r & 1)));
      }
    }
  }
  if (to >= 0 && to < b.n_slots) {
    float* p = a.states + ((int64_t)to * a.v_heads + head) * slot_size;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[(int64_t)(wave * (DK / 4) + m * 16 + r4 + r) * v_dim + col0 + c * 16] = s[m][c][r];
  }
}

// Tokens before the first sequence's and behind the last's come out as 0.
__global__ __launch_bounds__(256) void clear_kernel(LinearArgs a, int64_t row_chunks) {
  const int lo = clamp_to(a.b.starts[0], a.b.tokens), hi = clamp_to(a.b.starts[a.b.batch], a.b.tokens);
  const int64_t before = lo * row_chunks, all = before + (a.b.tokens - hi) * row_chunks, skip = (hi - lo) * row_chunks;
  uint4* out = reinterpret_cast<uint4*>(a.out);
  for (int64_t i = blockIdx.x * 256 + threadIdx.x; i < all; i += gridDim.x * 256) out[i < before ? i : i + skip] = uint4{0, 0, 0, 0};
}

template <class H>
static void launch_step(const LinearArgs& a, int k_dim, int v_dim, hipStream_t stream) {
  const uint32_t cols = (uint32_t)v_dim / kStepCols, grid = (uint32_t)a.b.tokens * (uint32_t)a.v_heads * cols;
  if (k_dim == 64) step_kernel<H, 64><<<grid, 256, 0, stream>>>(a, v_dim, cols);
  else if (k_dim == 128) step_kernel<H, 128><<<grid, 256, 0, stream>>>(a, v_dim, cols);
  else step_kernel<H, 256><<<grid, 256, 0, stream>>>(a, v_dim, cols);
}

hipError_t linear_step(const LinearArgs& a, int k_dim, int v_dim, bool fp16, hipStream_t stream) {
  fp16 ? launch_step<Fp16>(a, k_dim, v_dim, stream) : launch_step<Bf16>(a, k_dim, v_dim, stream);
  return hipGetLastError();
}

template <class H, int DK, bool BETA>
static void launch_prompt(const LinearArgs& a, int v_dim, hipStream_t stream) {
  const uint32_t cols = (uint32_t)v_dim / kCols;
  const uint32_t places = (uint32_t)linear_chunks(a.b.tokens, a.b.batch);
  prepare_kernel<H, DK, BETA><<<places * (uint32_t)a.v_heads, 256, 0, stream>>>(a);
  scan_kernel<H, DK, BETA><<<(uint32_t)a.b.batch * (uint32_t)a.v_heads * cols, 256, 0, stream>>>(a, v_dim, cols);
  const int64_t row_chunks = (int64_t)a.v_heads * v_dim / 8;
  clear_kernel<<<256, 256, 0, stream>>>(a, row_chunks);
}

template <class H>
static void pick_prompt(const LinearArgs& a, int k_dim, int v_dim, hipStream_t stream) {
  if (k_dim == 64) a.beta ? launch_prompt<H, 64, true>(a, v_dim, stream) : launch_prompt<H, 64, false>(a, v_dim, stream);
  else if (k_dim == 128) a.beta ? launch_prompt<H, 128, true>(a, v_dim, stream) : launch_prompt<H, 128, false>(a, v_dim, stream);
  else a.beta ? launch_prompt<H, 256, true>(a, v_dim, stream) : launch_prompt<H, 256, false>(a, v_dim, stream);
}

hipError_t linear_prompt(const LinearArgs& a, int k_dim, int v_dim, bool fp16, hipStream_t stream) {
  fp16 ? pick_prompt<Fp16>(a, k_dim, v_dim, stream) : pick_prompt<Bf16>(a, k_dim, v_dim, stream);
  return hipGetLastError();
}

}  // namespace jv
