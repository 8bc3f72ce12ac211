/*
 * jeeves_linear_attention.h -- C ABI of what lies between the projections of a
 * layer whose attention is linear (libjeeves_fp8.so, MI355X / gfx950): the
 * short causal convolution of q, k and v, and the linear attention with a decay
 * for each head, with the delta rule's correction or without.
 *
 * Conventions are those of jeeves_fp8.h: device pointers, a hipStream_t, a
 * JV_* status with jv_fp8_last_error(), launches only (no allocation, no host
 * synchronisation), so that every call may be captured into a HIP graph.
 *
 * Tensors are bf16 (fp16 = 0) or fp16 (fp16 = 1). A batch's sequence b has the
 * tokens starts[b] .. starts[b + 1] - 1 (starts: int32 [batch + 1], not
 * decreasing, from 0 to tokens; NULL: one token each, tokens = batch). What a
 * sequence carries on from its last call lies in a slot: from_slots[b] is read
 * (int32; NULL: slots; below 0 or past n_slots: the sequence starts from
 * zeros), slots[b] written (below 0 or past n_slots: nothing is kept). Several
 * sequences may start from one slot. A slot that two sequences write, or that
 * one reads and another writes, holds or gives either's, value by value. A sequence without
 * tokens reads and writes nothing. Tokens of no sequence come out as 0.
 */
#ifndef JEEVES_LINEAR_ATTENTION_H
#define JEEVES_LINEAR_ATTENTION_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Depthwise causal convolution over a sequence's tokens and the width - 1
 * inputs before them: out[t] = act(bias + sum_j weight[:, j] x[t - width + 1 + j]),
 * in fp32, rounded once; act: JV_CONV_PLAIN or JV_CONV_SILU.
 * x [tokens, channels] with row stride x_ts, rows 16-byte aligned, channels a
 * multiple of 8; weight float32 [channels, width], 16-byte aligned, width 2 to
 * 4; bias float32 [channels], 16-byte aligned, or NULL; states [n_slots,
 * width - 1, channels], a sequence's last inputs, oldest first; out [tokens,
 * channels], contiguous. tokens below 2^24, channels up to 65536. The role of
 * _conv_step (model/triton_kernels.py:267) and of the convolution of prompts.
 */
#define JV_CONV_PLAIN 0
#define JV_CONV_SILU 1
int jv_causal_conv(const void* x, int64_t x_ts, const float* weight, const float* bias, int64_t width, int activation,
                   void* states, int64_t n_slots, const int32_t* slots, const int32_t* from_slots, const int32_t* starts,
                   int64_t batch, void* out, int64_t tokens, int64_t channels, int fp16, void* stream);

/* Bytes of workspace jv_linear_attention needs for these sizes (0: none); -1 if
 * the sizes are refused. ragged: whether starts are given. For every 64 tokens, and
 * for every sequence, 38 KB a value head and 128 k_dim bytes a key head: 386 MB for
 * 16384 tokens of 32 value and 16 key heads of 128. */
int64_t jv_linear_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t k_heads, int64_t v_heads, int64_t k_dim,
                                            int64_t v_dim, int ragged);

/*
 * Linear attention with a state S [k_dim, v_dim] for each value head: token by
 * token of a sequence
 *   S = e^g S;  u = beta (v - S^T k)  (u = v where beta is NULL);  S = S + k u^T;  out = scale S^T q
 * in fp32, out rounded once. Value head h reads query and key head
 * h / (v_heads / k_heads). With norm_eps > 0 (a normal float32) q and k are
 * divided by sqrt(sum(x^2) + norm_eps) first.
 * g and beta of a token and value head: decay and beta [tokens, v_heads] with
 * row strides, float32 (gates16 = 0) or of the tensors' 16-bit type (gates16 =
 * 1); with rate (float32 [v_heads]; NULL: none) g = -rate softplus(decay +
 * decay_bias) and beta = sigmoid(beta) (decay_bias float32 [v_heads] or NULL),
 * else g = decay (at most 0 for a state that does not grow) and beta as it is.
 * q, k [tokens, k_heads, k_dim], v [tokens, v_heads, v_dim], strides in
 * elements for tokens (`ts`) and heads (`hs`), 16-byte aligned rows; k_dim and
 * v_dim 64, 128 or 256. states: float32 [n_slots, v_heads, k_dim, v_dim],
 * 16-byte aligned. out [tokens, v_heads, v_dim], contiguous. workspace:
 * 256-byte aligned. A token has no effect on those before it. Values that are
 * not finite stay visible: from the first token on that gives a non-finite update
 * u of a value channel, in a prompt or by itself, that channel is NaN until the
 * sequence's end and in its state. The role of the gated delta rule and of its
 * in-place step (model/fla_inplace.py:17-60) with their gates (_delta_gates,
 * model/triton_kernels.py:78).
 */
int jv_linear_attention(const void* q, int64_t q_ts, int64_t q_hs, const void* k, int64_t k_ts, int64_t k_hs, const void* v,
                        int64_t v_ts, int64_t v_hs, const void* decay, int64_t decay_ts, const void* beta, int64_t beta_ts,
                        int gates16, const float* rate, const float* decay_bias, float norm_eps, float* states,
                        int64_t n_slots, const int32_t* slots, const int32_t* from_slots, const int32_t* starts,
                        int64_t batch, float scale, void* out, int64_t tokens, int64_t k_heads, int64_t v_heads,
                        int64_t k_dim, int64_t v_dim, int fp16, void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* JEEVES_LINEAR_ATTENTION_H */
