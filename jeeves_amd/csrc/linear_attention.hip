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
// T = (I + A)^-1 in fp32, M, the rows' factors and K's transpose, all in the
// order in which the scans' products read them. scan_kernel and, for calls of
// few heads and sequences, scan_few_kernel go through a sequence's chunks with
// their part of S in registers.
//
// Rounding. States, sums, decays and norms are fp32 (the sums G fp64: their
// differences are what counts). The products are MFMAs of bf16: K and Q are
// exact (one bf16, or two for fp16), and what is fp32 goes in as the sum of
// three bf16 values (24 bits), towards the state and towards the outputs: with
// two values (16 bits) there, a whole call of 16384 tokens takes 612 us instead of
// 654 and one of 16 prompts 210 instead of 223, but outputs that are small
// differences lose their bits, and one in 300 (bf16) or 50 (fp16) of the others
// is rounded to the neighbouring value.
#include "layer.h"

namespace jv {

constexpr int kStepCols = 32;  // columns of S that a workgroup of step_kernel has

template <class H>
__device__ __forceinline__ float gate_at(const void* p, int wide16, int64_t i) {
  return wide16 ? H::lo(reinterpret_cast<const uint16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}

// log2 of a token's decay; what is below 2^-14400 is 0 by far.
__device__ __forceinline__ double log2_decay(float z, bool raw, float rate, float bias) {
  if (raw) z = -rate * softplus(z + bias);
  const double g = (double)z * 1.4426950408889634;
  return g < -14400.0 ? -14400.0 : g;
}

__device__ __forceinline__ float beta_of(const LinearArgs& a, float z) { return a.rate ? sigmoid(z) : z; }

// ---------------------------------------------------------------------------
// One token for each sequence. A workgroup has kStepCols columns of a head's
// state, a thread 4 columns of every 32nd row; S^T k and S^T q come from the
// state before the token (o = e^g S^T q + (q.k) u), so that one exchange
// between the waves serves both. Bound by the states' bytes: 64 sequences with
// 32 heads of 128 x 128 read and write 268 MB in 57 us, 4.7 TB/s (a large copy
// reaches 4.9). 32 columns a workgroup leave each thread 16 floats of state, all
// of whose loads are under way at a time.
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
  const float rate = a.rate ? uniform_f32(a.rate, head) : 0.0f, bias = a.decay_bias ? uniform_f32(a.decay_bias, head) : 0.0f;
  const float decay =
      __builtin_amdgcn_exp2f((float)log2_decay(gate_at<H>(a.decay, a.gates16, seq * a.decay_ts + head), a.rate != nullptr, rate, bias));
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
    // an update that is not finite makes its channel NaN, in the state as well, as a prompt's does
    if (!(__builtin_fabsf(u[e]) < __builtin_inff())) u[e] = __builtin_nanf("");
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
// of 16 bytes: T [lower fragment][3 parts], M [lower fragment][3 parts], then
// the rows' factors.
constexpr int kFragment = 1024;
constexpr int kBytesT = 6 * 3 * kFragment, kBytesM = kBytesT;
enum { kFromK, kFromQ, kBeta, kToEnd, kEnd, kFactors = 8 };  // [8][64] floats; kEnd: the whole chunk's decay
constexpr int kBytesHead = kBytesT + kBytesM + kFactors * kChunk * 4;

// K's transpose for a key head: [DK / 16][32 tokens] fragments.
constexpr int bytes_kt(int k_dim) { return k_dim * kChunk * 2; }

// Batches up to this size go through scan_kernel longest sequence first: its
// workgroups come to the compute units as these become free, and a long one that
// starts late is what the call then waits for (16 sequences of 64 to 1105 tokens
// in 512 workgroups: a sixth of that scan's time). prepare_kernel ranks the sequences, each
// against all, which past this size costs more than it can give.
constexpr int kOrdered = 1024;

int64_t linear_workspace(int64_t tokens, int64_t batch, int64_t k_heads, int64_t v_heads, int64_t k_dim) {
  return linear_chunks(tokens, batch) * (v_heads * kBytesHead + k_heads * bytes_kt((int)k_dim)) + kOrdered * (int64_t)sizeof(int32_t);
}

__device__ __forceinline__ uint8_t* head_data(const LinearArgs& a, int chunk, int head) {
  return a.workspace + ((int64_t)chunk * a.v_heads + head) * kBytesHead;
}
__device__ __forceinline__ uint8_t* key_data(const LinearArgs& a, int chunk, int kh, int k_dim) {
  return a.workspace + linear_chunks(a.b.tokens, a.b.batch) * a.v_heads * kBytesHead +
         ((int64_t)chunk * a.k_heads + kh) * bytes_kt(k_dim);
}
__device__ __forceinline__ int32_t* ordered(const LinearArgs& a, int k_dim) {
  return reinterpret_cast<int32_t*>(key_data(a, (int)linear_chunks(a.b.tokens, a.b.batch), 0, k_dim));
}

// Two fp32 values as sums of bf16 ones: x = p0 + p1 + p2 to 24 bits. What a
// rounding leaves is exact in fp32: one v_dot2_f32_bf16 with (-1, 0) or (0, -1).
// The pairs come from registers: as a constant the compiler writes the first
// one as the operand -1.0, which the instruction takes for the second.
template <int N>
__device__ __forceinline__ void split2(float x, float y, uint32_t (&p)[N]) {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  uint32_t low, high;
  asm("s_mov_b32 %0, 0xbf80" : "=s"(low));
  asm("s_mov_b32 %0, 0xbf800000" : "=s"(high));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = Bf16::pack(x, y);
    if (i + 1 < N) {
      x = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, p[i]), __builtin_bit_cast(pair, low), x, false);
      y = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair, p[i]), __builtin_bit_cast(pair, high), y, false);
    }
  }
}

// Two tiles' sums as a right operand's 32 rows.
template <int N>
__device__ __forceinline__ void split8(f32x4 x, f32x4 y, i32x4 (&f)[N]) {
  uint32_t p[4][N];
  split2<N>(x[0], x[1], p[0]), split2<N>(x[2], x[3], p[1]), split2<N>(y[0], y[1], p[2]), split2<N>(y[2], y[3], p[3]);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = i32x4{(int)p[0][i], (int)p[1][i], (int)p[2][i], (int)p[3][i]};
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

// Inclusive sums over the wave by DPP moves: row_shr 1, 2, 4, 8 within the 16
// lanes of a row (a shifted-out source adds 0), then row_bcast 15 and 31.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
  return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sums(double v) {
  v = dpp_add<0x111, 0xf>(v), v = dpp_add<0x112, 0xf>(v), v = dpp_add<0x114, 0xf>(v), v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);
  return dpp_add<0x143, 0xc>(v);
}

// The products' operands T and M go by a k order of their own: in 32 columns a
// lane's 8 are 4 g .. 4 g + 3 and 16 + 4 g .., g = lane / 16, which is what the
// four registers of two products' results hold. Row i of D and U then lies at
// place(i).
__device__ __forceinline__ int place_of(int i) { return (i & ~31) + ((i >> 2) & 3) * 8 + ((i >> 4) & 1) * 4 + (i & 3); }

// S's rows in the tiles of its sums: a tile's rows 4 g .. 4 g + 3 are the lanes'
// of group g, and two tiles hold 32 rows, 8 g .. 8 g + 7 a group, as the k of a
// product with K or Q goes.
__device__ __forceinline__ int state_row(int m, int g) { return 32 * (m >> 1) + 8 * g + 4 * (m & 1); }

// The lower triangle's fragments: of row tile t the 32 columns x, x <= t / 2.
__device__ __forceinline__ int fragment_of(int t, int x) { return x ? t + 2 : t; }

// One workgroup for a chunk of a value head; a wave has 16 of the chunk's rows.
//   A, M   K K^T and Q K^T by MFMAs (fp16 as it is), times the decays between
//          the rows, e^(G_i - G_j) of fp64 differences
//   T      A's diagonal blocks of 16 rows inverted by forward substitution, a
//          column a lane; the blocks below from those, T_ij = -T_ii (sum of
//          A_ik T_kj), as fp32 MFMAs whose results are the next one's operand
// What bounds it: its own bytes, and a workgroup's steps one after another, 25000
// cycles with four of them on a compute unit (VALU 42%). 16384 tokens of 32 heads
// (16 key heads) of 128: 109 us, 382 MB written (T and M in three bf16 parts, 38 KB a
// chunk and head, and K's transpose) and 151 fetched, 4.9 TB/s. Substitution
// over the whole 64 rows instead of blocks of 16 took 324: a chain of 64 steps.
template <class H, int DK, bool BETA>
__global__ __launch_bounds__(256) void prepare_kernel(LinearArgs a, int v_dim) {
  constexpr int KS = DK / 32, kRow = 68, kRowK = DK + 8, kRowD = 20;
  // K's rows, and in their place A once they are read: four workgroups a CU,
  // by registers, instead of three (an eighth of this kernel's time).
  constexpr int kShared = kChunk * (BETA && kRow * 4 > kRowK * 2 ? kRow * 4 : kRowK * 2);
  __shared__ __attribute__((aligned(16))) uint8_t shared[kShared];
  uint16_t* krows = reinterpret_cast<uint16_t*>(shared);
  float* tri = reinterpret_cast<float*>(shared);
  __shared__ __attribute__((aligned(16))) float diagonal[BETA ? 4 : 1][16 * kRowD];
  __shared__ __attribute__((aligned(16))) double sum[kChunk];
  __shared__ __attribute__((aligned(16))) float rk[kChunk], rq[kChunk], betas[kChunk];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Batch& b = a.b;
  // The hardware hands consecutive workgroups to the 8 XCDs in turn: the value
  // heads of one chunk and key head, which read the same rows, come to one.
  const uint32_t round_size = 8 * (uint32_t)a.group, round = blockIdx.x / round_size, within = blockIdx.x % round_size;
  const uint32_t units = min(gridDim.x / (uint32_t)a.group - round * 8, 8u), unit = round * 8 + within % units;
  const int place = (int)(unit / (uint32_t)a.k_heads), kh = (int)(unit % (uint32_t)a.k_heads), head = kh * a.group + (int)(within / units);

  // Tokens before the first sequence's and behind the last's come out as 0: of the batch's 64 from `place` x 64 on.
  {
    const int lo = clamp_to(uniform_at(b.starts, 0), b.tokens), hi = clamp_to(uniform_at(b.starts, b.batch), b.tokens);
    const int at = place * kChunk, n = rows_at(place, b.tokens);
    if (n > 0 && (at < lo || at + n > hi))
      for (int i = tid; i < n * (v_dim / 8); i += 256) {
        const int t = at + i / (v_dim / 8);
        if (t < lo || t >= hi)
          *reinterpret_cast<uint4*>(a.out + ((int64_t)t * a.v_heads + head) * v_dim + i % (v_dim / 8) * 8) = uint4{0, 0, 0, 0};
      }
  }

  // sequence `place` by its length: how many are longer, or as long and before it
  if (head == 0 && wave == 0 && b.batch <= kOrdered && place < b.batch) {
    const auto length = [&](int i) { return clamp_to(b.starts[i + 1], b.tokens) - clamp_to(b.starts[i], b.tokens); };
    const int mine = length(place);
    int rank = 0;
    for (int b0 = 0; b0 < b.batch; b0 += 64) {
      const int i = min(b0 + lane, b.batch - 1), n = length(i);
      rank += __popcll(__ballot(b0 + lane < b.batch && (n > mine || (n == mine && i < place))));
    }
    if (lane == 0) ordered(a, DK)[rank] = place;
  }

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

  const int r16 = lane & 15, g = lane >> 4, k8 = g * 8;
  float gate_d = 0.0f, gate_b = 0.0f, rate = 0.0f, bias = 0.0f;
  if (wave == 0) {
    const int64_t t = first + min(lane, rows - 1);
    if (a.rate) rate = uniform_f32(a.rate, head), bias = a.decay_bias ? uniform_f32(a.decay_bias, head) : 0.0f;
    if (a.gates16) {
      const uint16_t d = reinterpret_cast<const uint16_t*>(a.decay)[t * a.decay_ts + head];
      const uint16_t e = BETA ? reinterpret_cast<const uint16_t*>(a.beta)[t * a.beta_ts + head] : 0;
      gate_d = H::lo(d), gate_b = H::lo(e);
    } else {
      gate_d = reinterpret_cast<const float*>(a.decay)[t * a.decay_ts + head];
      if (BETA) gate_b = reinterpret_cast<const float*>(a.beta)[t * a.beta_ts + head];
    }
  }
  i32x4 kf[KS], qf[KS];
  {
    const int i = wave * 16 + r16;
    const int64_t t = first + min(i, rows - 1);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      kf[s] = *reinterpret_cast<const i32x4*>(a.k + t * a.k_ts + kh * a.k_hs + s * 32 + k8);
      qf[s] = *reinterpret_cast<const i32x4*>(a.q + t * a.q_ts + kh * a.q_hs + s * 32 + k8);
    }
    if (wave == 0) {
      const bool real = lane < rows;
      const double d = wave_sums(real ? log2_decay(gate_d, a.rate != nullptr, rate, bias) : 0.0);
      sum[lane] = d;
      betas[lane] = !real ? 0.0f : !BETA ? 1.0f : a.rate ? sigmoid(gate_b) : gate_b;
    }
    if (rows < kChunk)
#pragma unroll
      for (int s = 0; s < KS; ++s) kf[s] &= (i - rows) >> 31, qf[s] &= (i - rows) >> 31;  // 0 behind the sequence's end
    float sk = 0.0f, sq = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      *reinterpret_cast<i32x4*>(&krows[i * kRowK + s * 32 + k8]) = kf[s];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float k0 = H::lo((uint32_t)kf[s][e]), k1 = H::hi((uint32_t)kf[s][e]);
        const float q0 = H::lo((uint32_t)qf[s][e]), q1 = H::hi((uint32_t)qf[s][e]);
        sk = __builtin_fmaf(k0, k0, __builtin_fmaf(k1, k1, sk)), sq = __builtin_fmaf(q0, q0, __builtin_fmaf(q1, q1, sq));
      }
    }
    const bool norm = a.norm_eps > 0.0f;
    if (norm) {
      sk += __shfl_xor(sk, 16), sk += __shfl_xor(sk, 32), sq += __shfl_xor(sq, 16), sq += __shfl_xor(sq, 32);
      sk = inv_sqrt(sk + a.norm_eps), sq = inv_sqrt(sq + a.norm_eps);
    }
    if (lane < 16) rk[i] = norm ? sk : 1.0f, rq[i] = a.scale * (norm ? sq : 1.0f);
  }
  lds_barrier();

  // A and M transposed: a lane has row i of 16 w .. 16 w + 15 and of every
  // column tile up to the diagonal the columns 4 g .. 4 g + 3.
  uint8_t* out = head_data(a, place, head);
  const int i = wave * 16 + r16;
  const double sum_i = sum[i];
  const float rk_i = rk[i], rq_i = rq[i], beta_i = betas[i];
  uint2 mp[4][3];
  f32x4 pull[BETA ? 4 : 1];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    mp[t][0] = mp[t][1] = mp[t][2] = uint2{0u, 0u};
    if (t > wave) continue;
    f32x4 kk = {0.0f, 0.0f, 0.0f, 0.0f}, qk = kk;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const i32x4 kb = *reinterpret_cast<const i32x4*>(&krows[(t * 16 + r16) * kRowK + s * 32 + k8]);
      kk = H::mfma16(kb, kf[s], kk), qk = H::mfma16(kb, qf[s], qk);
    }
    const f32x4 rk_j = *reinterpret_cast<const f32x4*>(&rk[t * 16 + g * 4]);
    float m[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = t * 16 + g * 4 + r;
      const float e = __builtin_amdgcn_exp2f((float)(sum_i - sum[j])) * rk_j[r];
      const float x = kk[r] * e * rk_i * beta_i, y = qk[r] * e * rq_i;
      if constexpr (BETA) pull[t][r] = j < i ? x : 0.0f;
      m[r] = j <= i ? y : 0.0f;
    }
    uint32_t p[2][3];
    split2<3>(m[0], m[1], p[0]), split2<3>(m[2], m[3], p[1]);
#pragma unroll
    for (int x = 0; x < 3; ++x) mp[t][x] = uint2{p[0][x], p[1][x]};
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    if (s > wave >> 1) continue;
    uint4* m = reinterpret_cast<uint4*>(out + kBytesT) + fragment_of(wave, s) * 3 * 64 + lane;
#pragma unroll
    for (int p = 0; p < 3; ++p) m[p * 64] = uint4{mp[2 * s][p].x, mp[2 * s][p].y, mp[2 * s + 1][p].x, mp[2 * s + 1][p].y};
  }
  if (wave == 0) {
    const double d = sum[lane], all = sum[kChunk - 1];
    const float from = __builtin_amdgcn_exp2f((float)d);
    float* f = reinterpret_cast<float*>(out + kBytesT + kBytesM);
    f[kFromK * kChunk + lane] = betas[lane] * from * rk[lane], f[kFromQ * kChunk + lane] = from * rq[lane];
    f[kBeta * kChunk + lane] = betas[lane];
    f[kToEnd * kChunk + lane] = __builtin_amdgcn_exp2f((float)(all - d)) * rk[lane];
    f[kEnd * kChunk + lane] = __builtin_amdgcn_exp2f((float)all);
  }
  if (head % a.group == 0) {
    i32x4* dst = reinterpret_cast<i32x4*>(key_data(a, place, kh, DK)) + lane;
    for (int f = wave; f < DK / 16 * 2; f += 4) {
      const int row = state_row(f >> 1, r16 >> 2) + (r16 & 3);
      i32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint16_t* p = &krows[((f & 1) * 32 + (e >> 1) * 16 + g * 4 + (e & 1) * 2) * kRowK + row];
        v[e] = (int)(p[0] | (uint32_t)p[kRowK] << 16);
      }
      dst[f * 64] = v;
    }
  }

  if constexpr (BETA) {
    lds_barrier();
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (t <= wave) *reinterpret_cast<f32x4*>(&tri[i * kRow + t * 16 + g * 4]) = pull[t];
    lds_barrier();
    // T by blocks of 16 rows. Wave w inverts the diagonal block w by forward
    // substitution, a column a lane (every 16 lanes the same), then works out
    // T's block column w: T_iw = -T_ii sum_(w <= k < i) A_ik T_kw in fp32 MFMAs
    // (16x16x4: a lane's A is row lane % 16, its B column lane % 16, k = lane /
    // 16). Their k go by 4 g + s for the s-th of four, which is where a result's
    // s-th register has its rows, so that a result is the next product's B as
    // it is, and as its A the transpose: T_iw^T = -(..)^T T_ii^T has the four
    // columns of a row in a lane.
    f32x4 tb[4], tt[4];
    {
      const float* d = &tri[(wave * 16) * kRow + wave * 16];
      float x[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        float s[2] = {r16 == c ? 1.0f : 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < c; j += 4) {
          const float4 r = *reinterpret_cast<const float4*>(d + c * kRow + j);
          s[0] = __builtin_fmaf(-r.x, x[j], s[0]);
          if (j + 1 < c) s[1] = __builtin_fmaf(-r.y, x[j + 1], s[1]);
          if (j + 2 < c) s[0] = __builtin_fmaf(-r.z, x[j + 2], s[0]);
          if (j + 3 < c) s[1] = __builtin_fmaf(-r.w, x[j + 3], s[1]);
        }
        x[c] = c < r16 ? 0.0f : s[0] + s[1];
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        tb[0][r] = g == 0 ? x[r] : g == 1 ? x[4 + r] : g == 2 ? x[8 + r] : x[12 + r];
        diagonal[wave][(g * 4 + r) * kRowD + r16] = tb[0][r];
      }
    }
    lds_barrier();
    tt[0] = *reinterpret_cast<const f32x4*>(&diagonal[wave][r16 * kRowD + g * 4]);
#pragma unroll
    for (int c = 1; c < 4; ++c) {
      if (wave + c > 3) break;
      f32x4 sums = {0.0f, 0.0f, 0.0f, 0.0f}, next = sums, turned = sums;
#pragma unroll
      for (int k = 0; k < c; ++k) {
        const f32x4 l = *reinterpret_cast<const f32x4*>(&tri[((wave + c) * 16 + r16) * kRow + (wave + k) * 16 + g * 4]);
#pragma unroll
        for (int s = 0; s < 4; ++s) sums = __builtin_amdgcn_mfma_f32_16x16x4f32(l[s], tb[k][s], sums, 0, 0, 0);
      }
      // rows behind a column's first one that is not finite must not reach those before it
      int bad = 16;
#pragma unroll
      for (int r = 3; r >= 0; --r)
        if (!(__builtin_fabsf(sums[r]) < __builtin_inff())) bad = g * 4 + r;
      const bool spoilt = __ballot(bad < 16) != 0;
      if (spoilt) {
        bad = min(bad, __shfl_xor(bad, 16));
        bad = min(bad, __shfl_xor(bad, 32));
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (g * 4 + r >= bad) sums[r] = 0.0f;
      }
      const f32x4 l = *reinterpret_cast<const f32x4*>(&diagonal[wave + c][r16 * kRowD + g * 4]);
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        next = __builtin_amdgcn_mfma_f32_16x16x4f32(l[s], sums[s], next, 0, 0, 0);
        turned = __builtin_amdgcn_mfma_f32_16x16x4f32(sums[s], l[s], turned, 0, 0, 0);
      }
      tb[c] = -next, tt[c] = -turned;
      if (spoilt) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (g * 4 + r >= bad) tb[c][r] = __builtin_nanf("");
          if (r16 >= __shfl(bad, g * 4 + r)) tt[c][r] = __builtin_nanf("");
        }
      }
    }
    // half of each fragment: the wave's 16 columns
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int tile = wave + c;
      if (tile > 3) break;
      uint32_t p[2][3];
      split2<3>(tt[c][0], tt[c][1], p[0]), split2<3>(tt[c][2], tt[c][3], p[1]);
#pragma unroll
      for (int x = 0; x < 3; ++x)
        *reinterpret_cast<uint2*>(out + (fragment_of(tile, wave >> 1) * 3 + x) * kFragment + lane * 16 + (wave & 1) * 8) = uint2{p[0][x], p[1][x]};
    }
    if (wave & 1) {
#pragma unroll
      for (int x = 0; x < 3; ++x)
        *reinterpret_cast<uint2*>(out + (fragment_of(wave - 1, wave >> 1) * 3 + x) * kFragment + lane * 16 + 8) = uint2{0u, 0u};
    }
  }
}

__device__ __forceinline__ f32x4 mfma_bf16(i32x4 a, i32x4 b, f32x4 c) { return Bf16::mfma16(a, b, c); }

// Waits out 16x16 MFMAs' results, which other instructions may not read for up
// to 11 issue slots: ahead of a wave-uniform branch the compiler has left the
// wait out (the listing's test follows every path).
template <int N>
__device__ __forceinline__ void settle(f32x4 (&r)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(r[i]));
  asm volatile("s_nop 7\n\ts_nop 2" : "+v"(r[N - 1]));
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(r[i]));
}

// A sequence's chunks one after the other, kCols columns of a head's state a
// workgroup, 16 a wave: a wave's columns of S, D and U are no other wave's, so
// that what a product leaves in registers is the next one's right operand as
// it lies there (the left operands have their k in that order), in two or three
// bf16 parts. The left operands K, Q, T, M and K^T are the same for all waves:
// they go through LDS, K and Q of the next chunk once this one's are read, the
// others at its end. A wave has loaded its share of them into registers a
// chunk's time before (copies straight into LDS are not used: the compiler
// waits for all of those in flight at any read of LDS).
//
// What bounds it: a chunk's steps one after another, two waves a SIMD to fill
// each other's gaps. 6.8 us a chunk (DK 128); of a call's time MFMA is busy 34%,
// LDS, where every wave reads all of the left operands, 25%, VALU 24%. A call takes as long
// as the chunks of its longest sequence, or all chunks over the compute units. 16
// sequences of 64 to 1105 tokens (149 chunks), 32 heads of 128 x 128: 166 to 174
// us. 32 columns a wave, which would halve the reads, took a quarter more: their
// sums no longer fit the registers without moves to and from the accumulators.
//
// A chunk whose U is not finite is gone through again: what lies behind a
// column's first row that is not finite is left out, where it would reach the
// rows before it as 0 times infinity, and comes out as NaN.
template <class H, int DK, int NW, bool BETA>
__global__ __launch_bounds__(64 * NW, DK == 64 ? 2 : NW / 4) void scan_kernel(LinearArgs a, int v_dim, uint32_t col_blocks) {
  constexpr int kCols = 16 * NW, kRowO = kCols + 8;
  constexpr int KS = DK / 32, MT = DK / 16, NP = Parts<H>::n, NU = BETA ? 3 : NP;  // parts of U: without beta it is V
  // fragments of 1 KB: what the first half of a chunk reads, and the second
  constexpr int kK = 0, kQ = BETA ? 4 * KS : 0, kKt = kQ + 4 * KS, kM = kKt + 2 * MT, kT = kM + 18, kF = kT + (BETA ? 18 : 0), kV = kF + 2;
  constexpr int kVs = 2 * NW;  // V's fragments
  __shared__ __attribute__((aligned(1024))) uint8_t lds[(kV + kVs) * kFragment];
  __shared__ __attribute__((aligned(16))) uint16_t ob[kChunk * kRowO];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // The hardware hands consecutive workgroups to the 8 XCDs in turn: those of
  // one sequence and key head, which read the same operands, come to one.
  const Batch& b = a.b;
  const uint32_t unit_size = (uint32_t)a.group * col_blocks, round = blockIdx.x / (8 * unit_size), within = blockIdx.x % (8 * unit_size);
  const uint32_t units = min((uint32_t)(b.batch * a.k_heads) - round * 8, 8u);
  const uint32_t unit = round * 8 + within % units, inner = within / units, cb = inner % col_blocks;
  const int kh = (int)(unit % (uint32_t)a.k_heads), rank = (int)(unit / (uint32_t)a.k_heads), head = kh * a.group + (int)(inner / col_blocks);
  const int seq = b.batch <= kOrdered ? __builtin_amdgcn_readfirstlane(uniform_at(ordered(a, DK), rank)) : rank;
  const int start = clamp_to(uniform_at(b.starts, seq), b.tokens), n = clamp_to(uniform_at(b.starts, seq + 1), b.tokens) - start;
  if (n <= 0) return;
  const int from = uniform_at(b.from, seq), to = uniform_at(b.slots, seq);
  const int r16 = lane & 15, g = lane >> 4, r4 = g * 4, k8 = g * 8;
  const int last = (n - 1) / kChunk, chunk0 = start / kChunk + seq;
  const int64_t slot_size = (int64_t)DK * v_dim;
  const int col = (int)cb * kCols + wave * 16 + r16;

  // Chunk c's rows of K and Q as fragments [row tile][32 columns]; rows behind the end: the last one's. The wave's share is
  // every (NW / 4)-th of a row tile's.
  constexpr int kShare = 4 * KS / NW;
  const int tile = wave & 3, x0 = wave >> 2;
  i32x4 kq[2][kShare];
  const auto load_kq = [&](int c) {
    const int64_t t = start + c * kChunk + min(tile * 16 + r16, n - c * kChunk - 1);
    const uint16_t *k = a.k + t * a.k_ts + kh * a.k_hs + x0 * 32 + k8, *q = a.q + t * a.q_ts + kh * a.q_hs + x0 * 32 + k8;
#pragma unroll
    for (int x = 0; x < kShare; ++x) {
      if (BETA) kq[0][x] = *reinterpret_cast<const i32x4*>(k + x * (NW / 4) * 32);
      kq[1][x] = *reinterpret_cast<const i32x4*>(q + x * (NW / 4) * 32);
    }
  };
  const auto put = [&](int i, i32x4 v) { *reinterpret_cast<i32x4*>(lds + i * kFragment + lane * 16) = v; };
  const auto put_kq = [&]() {
#pragma unroll
    for (int x = 0; x < kShare; ++x) {
      if (BETA) put(kK + tile * KS + x * (NW / 4) + x0, kq[0][x]);
      put(kQ + tile * KS + x * (NW / 4) + x0, kq[1][x]);
    }
  };
  // Its other operands, every NW-th fragment of each kind a wave's (a kind's
  // last one again where it has none), and V's rows [64][kCols].
  constexpr int kKts = 2 * MT, kMs = 18, kTs = BETA ? 20 : 2;  // T's 18 and the factors' 2, in the order of LDS
  constexpr int kNKt = (kKts + NW - 1) / NW, kNM = (kMs + NW - 1) / NW, kNT = (kTs + NW - 1) / NW;
  i32x4 kt[kNKt], mt[kNM], tail[kNT], v8[2];
  const auto load_rest = [&](int c) {
    const i32x4* d = reinterpret_cast<const i32x4*>(head_data(a, chunk0 + c, head)) + lane;
    const i32x4* k = reinterpret_cast<const i32x4*>(key_data(a, chunk0 + c, kh, DK)) + lane;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = ((i * NW + wave) * 64 + lane) * 8, row = at / kCols;
      const int64_t t = start + c * kChunk + min(row, n - c * kChunk - 1);
      v8[i] = *reinterpret_cast<const i32x4*>(a.v + t * a.v_ts + head * a.v_hs + cb * kCols + at % kCols);
    }
#pragma unroll
    for (int i = 0; i < kNT; ++i) {
      const int f = min(i * NW + wave, kTs - 1);
      tail[i] = d[(f < kTs - 2 ? f : f - (kTs - 2) + (kBytesT + kBytesM) / kFragment) * 64];
    }
#pragma unroll
    for (int i = 0; i < kNM; ++i) mt[i] = d[(kBytesT / kFragment + min(i * NW + wave, kMs - 1)) * 64];
#pragma unroll
    for (int i = 0; i < kNKt; ++i) kt[i] = k[min(i * NW + wave, kKts - 1) * 64];
  };
  const auto put_rest = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i) put(kV + i * NW + wave, v8[i]);
#pragma unroll
    for (int i = 0; i < kNT; ++i) put(kT + min(i * NW + wave, kTs - 1), tail[i]);
#pragma unroll
    for (int i = 0; i < kNM; ++i) put(kM + min(i * NW + wave, kMs - 1), mt[i]);
#pragma unroll
    for (int i = 0; i < kNKt; ++i) put(kKt + min(i * NW + wave, kKts - 1), kt[i]);
  };
  const auto fragment = [&](int i) { return *reinterpret_cast<const i32x4*>(lds + i * kFragment + lane * 16); };
  const auto factor = [&](int which, int t) {
    return *reinterpret_cast<const f32x4*>(lds + kF * kFragment + (which * kChunk + t * 16 + r4) * 4);
  };

  load_kq(0);
  __builtin_amdgcn_sched_barrier(0);
  load_rest(0);
  __builtin_amdgcn_sched_barrier(0);
  // S's row state_row(m, g) + r is tile m's row 4 g + r.
  f32x4 s[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) s[m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (from >= 0 && from < b.n_slots) {
    const float* p = a.states + ((int64_t)from * a.v_heads + head) * slot_size + col;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[m][r] = p[(state_row(m, g) + r) * v_dim];
  }

  put_kq();
  for (int chunk = 0; chunk <= last; ++chunk) {
    const int rows = min(n - chunk * kChunk, kChunk);
    lds_barrier();
    put_rest();
    load_kq(min(chunk + 1, last));
    if (chunk) {
      // the outputs of the chunk before, which is a whole one
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = ((i * NW + wave) * 64 + lane) * 8, row = at / kCols;
        const int64_t t = start + (chunk - 1) * kChunk + row;
        *reinterpret_cast<uint4*>(a.out + (t * a.v_heads + head) * v_dim + cb * kCols + at % kCols) =
            *reinterpret_cast<const uint4*>(&ob[row * kRowO + at % kCols]);
      }
    }
    // K S and Q S, 16 rows a tile
    f32x4 pk[4], pq[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) pk[t] = pq[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      i32x4 sp[3];
      split8(s[2 * x], s[2 * x + 1], sp);
#pragma unroll
      for (int i = BETA ? 0 : 1; i < 2; ++i) {
        i32x4 rp[4][NP];
#pragma unroll
        for (int t = 0; t < 4; ++t) Parts<H>::of(fragment((i ? kQ : kK) + t * KS + x), rp[t]);
#pragma unroll
        for (int j = 2; j >= 0; --j)
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            f32x4& p = i ? pq[t] : pk[t];
            if (NP > 1 && j < 2) p = mfma_bf16(rp[t][NP - 1], sp[j], p);
            p = mfma_bf16(rp[t][0], sp[j], p);
          }
      }
    }
    settle(pq);
    lds_barrier();
    put_kq();

    f32x4 d[4], u[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t v = *reinterpret_cast<const uint16_t*>(lds + kV * kFragment + ((t * 16 + r4 + r) * kCols + wave * 16 + r16) * 2);
        d[t][r] = H::lo(v);
      }
      if constexpr (BETA) {
        const f32x4 from_k = factor(kFromK, t), beta = factor(kBeta, t);
#pragma unroll
        for (int r = 0; r < 4; ++r) d[t][r] = __builtin_fmaf(-from_k[r], pk[t][r], beta[r] * d[t][r]);
      }
      // rows behind the sequence's end, whose K, Q and V are its last row's, count nothing
      if (rows < kChunk)
#pragma unroll
        for (int r = 0; r < 4; ++r) d[t][r] = t * 16 + r4 + r < rows ? d[t][r] : 0.0f;
    }
    const auto solve = [&]() {
      if constexpr (BETA) {
        i32x4 dp[2][3];
#pragma unroll
        for (int x = 0; x < 2; ++x) split8(d[2 * x], d[2 * x + 1], dp[x]);
#pragma unroll
        for (int t = 0; t < 4; ++t) u[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int i = 2; i >= 0; --i) {
            i32x4 tf[4];
#pragma unroll
            for (int t = 2 * x; t < 4; ++t) tf[t] = fragment(kT + fragment_of(t, x) * 3 + i);
#pragma unroll
            for (int j = 2 - i; j >= 0; --j)
#pragma unroll
              for (int t = 2 * x; t < 4; ++t) u[t] = mfma_bf16(tf[t], dp[x][j], u[t]);
          }
        }
        settle(u);
      } else {
#pragma unroll
        for (int t = 0; t < 4; ++t) u[t] = d[t];
      }
    };
    // a column's first row of x that is not finite
    const auto first_bad = [&](const f32x4(&x)[4]) {
      int first = kChunk;
#pragma unroll
      for (int t = 3; t >= 0; --t)
#pragma unroll
        for (int r = 3; r >= 0; --r)
          if (!(__builtin_fabsf(x[t][r]) < __builtin_inff())) first = t * 16 + r4 + r;
      first = min(first, __shfl_xor(first, 16));
      return min(first, __shfl_xor(first, 32));
    };
    solve();
    int bad = kChunk;
    {
      float z = 0.0f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) z = __builtin_fmaf(u[t][r], 0.0f, z);
      if (__ballot(z != z)) {
        bad = first_bad(d);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (t * 16 + r4 + r >= bad) d[t][r] = 0.0f;
        solve();
        bad = min(bad, first_bad(u));
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (t * 16 + r4 + r >= bad) u[t][r] = 0.0f;
      }
    }

    load_rest(min(chunk + 1, last));

    // the chunk's outputs
    f32x4 o[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) o[t] = factor(kFromQ, t) * pq[t];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      i32x4 up[NU];
      split8(u[2 * x], u[2 * x + 1], up);
#pragma unroll
      for (int i = 2; i >= 0; --i) {
        i32x4 mf[4];
#pragma unroll
        for (int t = 2 * x; t < 4; ++t) mf[t] = fragment(kM + fragment_of(t, x) * 3 + i);
#pragma unroll
        for (int j = min(2 - i, NU - 1); j >= 0; --j)
#pragma unroll
          for (int t = 2 * x; t < 4; ++t) o[t] = mfma_bf16(mf[t], up[j], o[t]);
      }
    }
    // the state behind the chunk
    const float end = *reinterpret_cast<const float*>(lds + kF * kFragment + kEnd * kChunk * 4);
#pragma unroll
    for (int t = 0; t < 4; ++t) u[t] *= factor(kToEnd, t);
#pragma unroll
    for (int m = 0; m < MT; ++m) s[m] *= end;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      i32x4 up[3];
      split8(u[2 * x], u[2 * x + 1], up);
#pragma unroll
      for (int m0 = 0; m0 < MT; m0 += 4) {
        i32x4 kp[4][NP];
#pragma unroll
        for (int m = 0; m < 4; ++m) Parts<H>::of(fragment(kKt + (m0 + m) * 2 + x), kp[m]);
#pragma unroll
        for (int i = 2; i >= 0; --i)
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            if (NP > 1 && i < 2) s[m0 + m] = mfma_bf16(kp[m][NP - 1], up[i], s[m0 + m]);
            s[m0 + m] = mfma_bf16(kp[m][0], up[i], s[m0 + m]);
          }
      }
    }
    settle(o);
    settle(s);
    if (__ballot(bad < kChunk)) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (t * 16 + r4 + r >= bad) o[t][r] = __builtin_nanf("");
#pragma unroll
      for (int m = 0; m < MT; ++m)
        if (bad < kChunk) s[m] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; r += 2) {
        const uint32_t p = H::pack(o[t][r], o[t][r + 1]);
        ob[(t * 16 + r4 + r) * kRowO + wave * 16 + r16] = (uint16_t)p;
        ob[(t * 16 + r4 + r + 1) * kRowO + wave * 16 + r16] = (uint16_t)(p >> 16);
      }
  }
  lds_barrier();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = ((i * NW + wave) * 64 + lane) * 8, row = at / kCols;
    const int64_t t = start + last * kChunk + row;
    if (t < start + n)
      *reinterpret_cast<uint4*>(a.out + (t * a.v_heads + head) * v_dim + cb * kCols + at % kCols) =
          *reinterpret_cast<const uint4*>(&ob[row * kRowO + at % kCols]);
  }
  if (to >= 0 && to < b.n_slots) {
    float* p = a.states + ((int64_t)to * a.v_heads + head) * slot_size + col;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) p[(state_row(m, g) + r) * v_dim] = s[m][r];
  }
}

// The same with 16 or 32 columns a workgroup, for calls of few heads and
// sequences, where scan_kernel would leave compute units without one: a chunk's
// work is spread over eight waves, in three steps with an exchange through LDS behind each:
//   the state in three parts                               -> sb, as the right operand of K S and Q S
//   D = beta (V - e^G K S) in three parts                  -> db, as that of T D
//   U = T D and e^(G_C - G) U, each in three parts         -> ub, as that of M U and of K^T U, which gives the state
// Waves 0 to 3 go through them, wave w with a chunk's rows from 16 w on and the
// state's from w DK / 4 on. Waves 4 to 7 have the rows' outputs e^G Q S + M U,
// which no later chunk waits for, and bring the factors and V to LDS (a load's
// issue is a wait of 16 to 32 cycles). An operand is loaded for the next chunk once
// this one has used it, so that a load has most of a chunk's time and no
// register of its own.
//
// What bounds it: the chain of a chunk, 4850 cycles; taken apart when U went to the
// outputs in two parts and it was 4600: the split of S 450, K S 750, D 500, T D 360,
// U 590, K^T U 720, and the exchanges between them. One sequence of 16384 tokens, 32
// heads (16 key heads) of 128 x 128: 256 chunks in 553 to 563 us. For the 525 of
// those two parts it was 690 with waves 4 to 7 left out, 600 with K S as partial sums
// of the waves, exchanged instead of the state's parts, and 1290 with 16 columns a
// wave for all 64 rows.
template <class H, int DK, int kCols, bool BETA>
__global__ __launch_bounds__(512, 1) void scan_few_kernel(LinearArgs a, int v_dim, uint32_t col_blocks) {
  constexpr int KS = DK / 32, MT = DK / 64, NT = kCols / 16, NP = Parts<H>::n, NU = BETA ? 3 : NP;  // parts of U: without beta it is V
  constexpr int kRowS = DK + 8, kRowU = kChunk + 8;
  __shared__ __attribute__((aligned(16))) uint16_t sb[3][kCols * kRowS];
  __shared__ __attribute__((aligned(16))) uint16_t db[BETA ? 3 : 1][kCols * kRowU];
  __shared__ __attribute__((aligned(16))) uint16_t ub[NU + 3][kCols * kRowU];
  __shared__ __attribute__((aligned(16))) float fb[2][5 * kChunk];            // the rows' factors, by turns
  __shared__ __attribute__((aligned(16))) uint16_t vb[2][kChunk * kCols];     // and V's rows
  __shared__ int first_d[kCols], first_us[2][kCols];  // a column's first row that is not finite; U's by turns
  const int tid = threadIdx.x, lane = tid & 63, all_wave = __builtin_amdgcn_readfirstlane(tid >> 6), wave = all_wave & 3;
  // The hardware hands consecutive workgroups to the 8 XCDs in turn: those of
  // one sequence and key head, which read the same operands, come to one.
  const Batch& b = a.b;
  const uint32_t unit_size = (uint32_t)a.group * col_blocks, round = blockIdx.x / (8 * unit_size), within = blockIdx.x % (8 * unit_size);
  const uint32_t units = min((uint32_t)(b.batch * a.k_heads) - round * 8, 8u);
  const uint32_t unit = round * 8 + within % units, inner = within / units, cb = inner % col_blocks;
  const int kh = (int)(unit % (uint32_t)a.k_heads), seq = (int)(unit / (uint32_t)a.k_heads), head = kh * a.group + (int)(inner / col_blocks);
  const int start = clamp_to(uniform_at(b.starts, seq), b.tokens), n = clamp_to(uniform_at(b.starts, seq + 1), b.tokens) - start;
  if (n <= 0) return;
  const int r16 = lane & 15, r4 = (lane >> 4) * 4, k8 = (lane >> 4) * 8, col0 = (int)cb * kCols + r16, row16 = wave * 16 + r16;
  const int last = (n - 1) / kChunk, chunk0 = start / kChunk + seq;
  const uint8_t* data = head_data(a, chunk0, head);
  const int64_t data_step = (int64_t)a.v_heads * kBytesHead;
  if (tid < kCols) first_d[tid] = first_us[chunk0 & 1][tid] = kChunk;

  if (all_wave >= 4) {
    i32x4 qf[KS], mf[2][3];
    const uint16_t* q_next = a.q + (int64_t)(start + row16) * a.q_ts + kh * a.q_hs + k8;
    const auto load_q = [&](int c) {
      const int rows = n - c * kChunk;
      const uint16_t* p = rows >= kChunk ? q_next : a.q + (int64_t)(start + c * kChunk + min(row16, rows - 1)) * a.q_ts + kh * a.q_hs + k8;
#pragma unroll
      for (int x = 0; x < KS; ++x) qf[x] = *reinterpret_cast<const i32x4*>(p + x * 32);
      q_next += c < last ? kChunk * a.q_ts : 0;  // never past the last chunk, which is loaded again
    };
    const auto load_m = [&](const uint8_t* d) {
      const i32x4* p = reinterpret_cast<const i32x4*>(d + kBytesT) + lane;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (x > (wave >> 1)) break;
#pragma unroll
        for (int i = 0; i < 3; ++i) mf[x][i] = p[(fragment_of(wave, x) * 3 + i) * 64];
      }
    };
    // 80 times 16 bytes of factors and kCols / 8 of each row of V
    constexpr int kItems = 80 + kChunk * kCols / 8, kMine = (kItems + 255) / 256;
    const int item = (all_wave - 4) * 64 + lane;
    i32x4 held[kMine];
    const auto load_held = [&](int c) {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int at = min(item + i * 256, kItems - 1), v_at = max(at - 80, 0) * 8, row = min(v_at / kCols, n - c * kChunk - 1);
        const uint16_t* v = a.v + (int64_t)(start + c * kChunk + row) * a.v_ts + head * a.v_hs + cb * kCols + v_at % kCols;
        const uint8_t* f = head_data(a, chunk0 + c, head) + kBytesT + kBytesM + at * 16;
        held[i] = *reinterpret_cast<const i32x4*>(at < 80 ? f : reinterpret_cast<const uint8_t*>(v));
      }
    };
    const auto put_held = [&](int c) {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        const int at = item + i * 256;
        if (at < 80) *reinterpret_cast<i32x4*>(&fb[c & 1][at * 4]) = held[i];
        else if (at < kItems) *reinterpret_cast<i32x4*>(&vb[c & 1][(at - 80) * 8]) = held[i];
      }
    };
    load_held(0);
    __builtin_amdgcn_sched_barrier(0);
    load_q(0);
    __builtin_amdgcn_sched_barrier(0);
    load_m(data);
    __builtin_amdgcn_sched_barrier(0);
    put_held(0);
    load_held(min(1, last));
    uint16_t* out = a.out + ((int64_t)(start + wave * 16 + r4) * a.v_heads + head) * v_dim + col0;
    const int64_t out_ts = (int64_t)a.v_heads * v_dim;
    for (int chunk = 0; chunk <= last; ++chunk) {
      const int rows = n - chunk * kChunk;
      lds_barrier();
      f32x4 pq[NT][2];
#pragma unroll
      for (int c = 0; c < NT; ++c) pq[c][0] = pq[c][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        i32x4 qp[NP];
        Parts<H>::of(qf[x], qp);
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          i32x4 sp[3];
#pragma unroll
          for (int i = 0; i < 3; ++i) sp[i] = *reinterpret_cast<const i32x4*>(&sb[i][(c * 16 + r16) * kRowS + x * 32 + k8]);
          pq[c][1] = mfma_bf16(qp[0], sp[2], pq[c][1]), pq[c][0] = mfma_bf16(qp[0], sp[0], pq[c][0]);
          pq[c][1] = mfma_bf16(qp[0], sp[1], pq[c][1]);
          if (NP > 1) pq[c][1] = mfma_bf16(qp[NP - 1], sp[1], pq[c][1]), pq[c][1] = mfma_bf16(qp[NP - 1], sp[0], pq[c][1]);
        }
      }
      load_q(min(chunk + 1, last));
      const f32x4 from_q = *reinterpret_cast<const f32x4*>(&fb[chunk & 1][kFromQ * kChunk + wave * 16 + r4]);
      put_held(chunk + 1);
      load_held(min(chunk + 2, last));
      if constexpr (BETA) {
        lds_barrier();
        if (__ballot(first_d[lane & (kCols - 1)] < kChunk)) lds_barrier();
      }
      lds_barrier();
      const int* first_u = first_us[(chunk0 + chunk) & 1];
      const bool spoilt = __ballot(first_u[lane & (kCols - 1)] < kChunk) != 0;
      if (spoilt) lds_barrier();
      f32x4 o[NT][2];
#pragma unroll
      for (int c = 0; c < NT; ++c) o[c][0] = o[c][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (x > (wave >> 1)) break;
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          i32x4 up[NU];
#pragma unroll
          for (int i = 0; i < NU; ++i) up[i] = *reinterpret_cast<const i32x4*>(&ub[i][(c * 16 + r16) * kRowU + x * 32 + k8]);
#pragma unroll
          for (int i = 2; i >= 0; --i)
#pragma unroll
            for (int j = min(2 - i, NU - 1); j >= 0; --j) {
              f32x4& sum = o[c][i + j > 0];
              sum = mfma_bf16(mf[x][i], up[j], sum);
            }
        }
      }
#pragma unroll
      for (int c = 0; c < NT; ++c) {
#pragma unroll
        for (int r = 0; r < 4; ++r) o[c][0][r] = __builtin_fmaf(from_q[r], pq[c][0][r] + pq[c][1][r], o[c][0][r] + o[c][1][r]);
        if (spoilt) {
          const int bad = first_u[c * 16 + r16];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (wave * 16 + r4 + r >= bad) o[c][0][r] = __builtin_nanf("");
        }
      }
      data += chunk < last ? data_step : 0;
      load_m(data);
      const int mine = rows - wave * 16 - r4;  // this lane's rows that are the sequence's
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const uint32_t p[2] = {H::pack(o[c][0][0], o[c][0][1]), H::pack(o[c][0][2], o[c][0][3])};
        const uint16_t p16[4] = {(uint16_t)p[0], (uint16_t)(p[0] >> 16), (uint16_t)p[1], (uint16_t)(p[1] >> 16)};
        if (rows >= kChunk) {
#pragma unroll
          for (int r = 0; r < 4; ++r) out[r * out_ts + c * 16] = p16[r];
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r < mine) out[r * out_ts + c * 16] = p16[r];
        }
      }
      out += kChunk * out_ts;
    }
    return;
  }

  const int from = uniform_at(b.from, seq), to = uniform_at(b.slots, seq);
  const int place4 = place_of(wave * 16 + r4);
  const int64_t slot_size = (int64_t)DK * v_dim;
  f32x4 s[MT][NT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int c = 0; c < NT; ++c) s[m][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (from >= 0 && from < b.n_slots) {
    const float* p = a.states + ((int64_t)from * a.v_heads + head) * slot_size + col0;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[m][c][r] = p[(state_row(wave * MT + m, lane >> 4) + r) * v_dim + c * 16];
  }
  i32x4 kf[KS], tf[BETA ? 2 : 1][3], kt[2][MT];
  const uint16_t* k_next = a.k + (int64_t)(start + row16) * a.k_ts + kh * a.k_hs + k8;
  const auto load_k = [&](int c) {
    if constexpr (BETA) {
      const int rows = n - c * kChunk;
      const uint16_t* p = rows >= kChunk ? k_next : a.k + (int64_t)(start + c * kChunk + min(row16, rows - 1)) * a.k_ts + kh * a.k_hs + k8;
#pragma unroll
      for (int x = 0; x < KS; ++x) kf[x] = *reinterpret_cast<const i32x4*>(p + x * 32);
      k_next += c < last ? kChunk * a.k_ts : 0;  // never past the last chunk, which is loaded again
    }
  };
  const auto load_t = [&](const uint8_t* d) {
    if constexpr (BETA) {
      const i32x4* p = reinterpret_cast<const i32x4*>(d) + lane;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (x > (wave >> 1)) break;
#pragma unroll
        for (int i = 0; i < 3; ++i) tf[x][i] = p[(fragment_of(wave, x) * 3 + i) * 64];
      }
    }
  };
  const uint8_t* keys = key_data(a, chunk0, kh, DK);
  const int64_t keys_step = (int64_t)a.k_heads * bytes_kt(DK);
  const auto load_kt = [&]() {
    const i32x4* p = reinterpret_cast<const i32x4*>(keys) + wave * MT * 2 * 64 + lane;
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int m = 0; m < MT; ++m) kt[x][m] = p[(m * 2 + x) * 64];
  };
  // what of a lane's rows is not finite
  const auto mark = [&](int* first, const auto& x) {
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (!(__builtin_fabsf(x[c][r]) < __builtin_inff())) atomicMin(&first[c * 16 + r16], wave * 16 + r4 + r);
  };
  // in the order of the loop, whose waits count the loads behind the one that is waited for
  load_k(0);
  __builtin_amdgcn_sched_barrier(0);
  load_t(data);
  __builtin_amdgcn_sched_barrier(0);
  load_kt();
  __builtin_amdgcn_sched_barrier(0);

  for (int chunk = 0; chunk <= last; ++chunk) {
    const int rows = n - chunk * kChunk, place = chunk0 + chunk, next = min(chunk + 1, last);
    int* first_u = first_us[place & 1];
    // the state in three parts, columns as rows
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        uint32_t p[2][3];
        split2<3>(s[m][c][0], s[m][c][1], p[0]), split2<3>(s[m][c][2], s[m][c][3], p[1]);
#pragma unroll
        for (int i = 0; i < 3; ++i)
          *reinterpret_cast<uint2*>(&sb[i][(c * 16 + r16) * kRowS + state_row(wave * MT + m, lane >> 4)]) = uint2{p[0][i], p[1][i]};
      }
    lds_barrier();
    if (tid < kCols) first_us[(place + 1) & 1][tid] = kChunk;
    f32x4 u[NT], pk[NT][2];
    if constexpr (BETA) {
      if (rows < kChunk)
#pragma unroll
        for (int x = 0; x < KS; ++x) kf[x] &= (row16 - rows) >> 31;
#pragma unroll
      for (int c = 0; c < NT; ++c) pk[c][0] = pk[c][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int x = 0; x < KS; ++x) {
        i32x4 kp[NP];
        Parts<H>::of(kf[x], kp);
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          i32x4 sp[3];
#pragma unroll
          for (int i = 0; i < 3; ++i) sp[i] = *reinterpret_cast<const i32x4*>(&sb[i][(c * 16 + r16) * kRowS + x * 32 + k8]);
          pk[c][1] = mfma_bf16(kp[0], sp[2], pk[c][1]), pk[c][0] = mfma_bf16(kp[0], sp[0], pk[c][0]);
          pk[c][1] = mfma_bf16(kp[0], sp[1], pk[c][1]);
          if (NP > 1) pk[c][1] = mfma_bf16(kp[NP - 1], sp[1], pk[c][1]), pk[c][1] = mfma_bf16(kp[NP - 1], sp[0], pk[c][1]);
        }
      }
      load_k(next);
    }
    float v[NT][4];
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t x = vb[chunk & 1][(wave * 16 + r4 + r) * kCols + c * 16 + r16];
        v[c][r] = H::lo(x & (uint32_t)((wave * 16 + r4 + r - rows) >> 31));  // 0 behind the end
      }
    const auto factor = [&](int which) { return *reinterpret_cast<const f32x4*>(&fb[chunk & 1][which * kChunk + wave * 16 + r4]); };
    const f32x4 from_k = factor(kFromK), beta = factor(kBeta), to_end = factor(kToEnd);
    const float end = fb[chunk & 1][kEnd * kChunk];

    if constexpr (BETA) {
      float d[NT][4], z = 0.0f;
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          d[c][r] = __builtin_fmaf(-from_k[r], pk[c][0][r] + pk[c][1][r], beta[r] * v[c][r]);
          z = __builtin_fmaf(d[c][r], 0.0f, z);
        }
      const auto hand_over_d = [&]() {
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          uint32_t p[2][3];
          split2<3>(d[c][0], d[c][1], p[0]), split2<3>(d[c][2], d[c][3], p[1]);
#pragma unroll
          for (int i = 0; i < 3; ++i) *reinterpret_cast<uint2*>(&db[i][(c * 16 + r16) * kRowU + place4]) = uint2{p[0][i], p[1][i]};
        }
      };
      hand_over_d();
      if (__ballot(z != z)) mark(first_d, d);
      lds_barrier();
      const bool spoilt = __ballot(first_d[lane & (kCols - 1)] < kChunk) != 0;
      if (spoilt) {
        // rows behind a column's first one that is not finite must not reach those before it
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (wave * 16 + r4 + r >= first_d[c * 16 + r16]) d[c][r] = 0.0f;
        hand_over_d();
        lds_barrier();
      }
      f32x4 td[NT][3];
#pragma unroll
      for (int c = 0; c < NT; ++c) td[c][0] = td[c][1] = td[c][2] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (x > (wave >> 1)) break;
        const i32x4* t = tf[x];
#pragma unroll
        for (int c = 0; c < NT; ++c) {
          i32x4 d[3];
#pragma unroll
          for (int i = 0; i < 3; ++i) d[i] = *reinterpret_cast<const i32x4*>(&db[i][(c * 16 + r16) * kRowU + x * 32 + k8]);
          td[c][2] = mfma_bf16(t[0], d[2], td[c][2]), td[c][1] = mfma_bf16(t[0], d[1], td[c][1]);
          td[c][0] = mfma_bf16(t[0], d[0], td[c][0]), td[c][2] = mfma_bf16(t[1], d[1], td[c][2]);
          td[c][1] = mfma_bf16(t[1], d[0], td[c][1]), td[c][2] = mfma_bf16(t[2], d[0], td[c][2]);
        }
      }
#pragma unroll
      for (int c = 0; c < NT; ++c) u[c] = td[c][0] + (td[c][1] + td[c][2]);
      load_t(data + (chunk < last ? data_step : 0));
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

    const auto hand_over = [&]() {
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        uint32_t p[2][NU], w[2][3];
        split2<NU>(u[c][0], u[c][1], p[0]), split2<NU>(u[c][2], u[c][3], p[1]);
        split2<3>(u[c][0] * to_end[0], u[c][1] * to_end[1], w[0]), split2<3>(u[c][2] * to_end[2], u[c][3] * to_end[3], w[1]);
        const int at = (c * 16 + r16) * kRowU + place4;
#pragma unroll
        for (int i = 0; i < NU; ++i) *reinterpret_cast<uint2*>(&ub[i][at]) = uint2{p[0][i], p[1][i]};
#pragma unroll
        for (int i = 0; i < 3; ++i) *reinterpret_cast<uint2*>(&ub[NU + i][at]) = uint2{w[0][i], w[1][i]};
      }
    };
    {
      float z = 0.0f;
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) z = __builtin_fmaf(u[c][r], 0.0f, z);
      hand_over();
      if (__ballot(z != z)) mark(first_u, u);
    }
    lds_barrier();
    const bool spoilt = __ballot(first_u[lane & (kCols - 1)] < kChunk) != 0;
    if (spoilt) {
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (wave * 16 + r4 + r >= first_u[c * 16 + r16]) u[c][r] = 0.0f;
      hand_over();
      lds_barrier();
    }
    if (tid < kCols) first_d[tid] = kChunk;

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
        for (int i = 0; i < 3; ++i) up[i] = *reinterpret_cast<const i32x4*>(&ub[NU + i][(c * 16 + r16) * kRowU + x * 32 + k8]);
        i32x4 kp[MT][NP];
#pragma unroll
        for (int m = 0; m < MT; ++m) Parts<H>::of(kt[x][m], kp[m]);
#pragma unroll
        for (int i = 2; i >= 0; --i)
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if (NP > 1 && i < 2) s[m][c] = mfma_bf16(kp[m][NP - 1], up[i], s[m][c]);
            s[m][c] = mfma_bf16(kp[m][0], up[i], s[m][c]);
          }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) settle(s[m]);
    data += chunk < last ? data_step : 0, keys += chunk < last ? keys_step : 0;
    load_kt();
    if (spoilt) {
#pragma unroll
      for (int c = 0; c < NT; ++c)
        if (first_u[c * 16 + r16] < kChunk)
#pragma unroll
          for (int m = 0; m < MT; ++m) s[m][c] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
    }
  }
  if (to >= 0 && to < b.n_slots) {
    float* p = a.states + ((int64_t)to * a.v_heads + head) * slot_size + col0;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[(state_row(wave * MT + m, lane >> 4) + r) * v_dim + c * 16] = s[m][c][r];
  }
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
  const uint32_t places = (uint32_t)linear_chunks(a.b.tokens, a.b.batch);
  prepare_kernel<H, DK, BETA><<<places * (uint32_t)a.v_heads, 256, 0, stream>>>(a, v_dim);
  const uint32_t heads = (uint32_t)a.b.batch * (uint32_t)a.v_heads, cols = (uint32_t)v_dim, w16 = heads * (cols / 16);
  const uint32_t cus = (uint32_t)max(cu_count_of(-1), 1);
  // Which scan: few columns a workgroup as long as that gives each compute unit
  // one (two, where the state's parts in LDS are small or the wide one's workgroups
  // few). Whole calls of 1024 tokens a sequence in us, 16 / 32 columns / scan_kernel:
  //   16 key and 32 value heads of 128 x 128   1 sequence 50 / 63 / 120, 2 82 / 69 / 126, 3 116 / 121 / 133,
  //                                            4 145 / 127 / 138, 8 313 / 271 / 194, 16 612 / 528 / 388
  //   14 heads of 64 x 64                      up to 4 39-45 / - / 68-74, 8 69 / - / 82, 12 94 / - / 92, 16 137 / - / 119
  //   5 heads of 256 x 256                     up to 3 71-76 / - / 150, 6 132 / - / 154, 8 188 / - / 158
  // All sequences here are of one length; a long one among short ones goes by their number all the same.
  if (w16 <= (DK == 128 ? cus : 2 * cus))
    scan_few_kernel<H, DK, 16, BETA><<<w16, 512, 0, stream>>>(a, v_dim, cols / 16);
  else if (DK == 128 && w16 / 2 <= cus)
    scan_few_kernel<H, 128, 32, BETA><<<w16 / 2, 512, 0, stream>>>(a, v_dim, cols / 32);
  else if (DK == 256 || v_dim == 64)
    scan_kernel<H, DK, 4, BETA><<<heads * (cols / 64), 256, 0, stream>>>(a, v_dim, cols / 64);
  else
    scan_kernel<H, DK < 256 ? DK : 128, 8, BETA><<<heads * (cols / 128), 512, 0, stream>>>(a, v_dim, cols / 128);
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
