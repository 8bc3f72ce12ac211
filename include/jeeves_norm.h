/*
 * jeeves_norm.h -- C ABI of the norms around a block of a served model, fused
 * with its gate, its residual and the quantizer of the next FP8 projection
 * (libjeeves_fp8.so, MI355X / gfx950).
 *
 * Conventions are those of jeeves_fp8.h: device pointers, a hipStream_t, a
 * JV_* status with jv_fp8_last_error(), launches only (no allocation, no host
 * synchronisation), so that every call may be captured into a HIP graph.
 */
#ifndef JEEVES_NORM_H
#define JEEVES_NORM_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define JV_GATE_PLAIN 0   /* the gate as it is */
#define JV_GATE_SIGMOID 1
#define JV_GATE_SILU 2

/*
 * For each token's row x of heads * dim channels, in fp32:
 *   b = x post_weight / sqrt(mean(x^2) + eps)  over each head's dim channels (b = x where post_weight is NULL)
 *   b = b act(gate)                            (gate NULL: none)
 *   h = residual + scale b                     (residual NULL: scale b)
 *   y = h weight / sqrt(mean(h^2) + eps)       over the whole row (y = h where weight is NULL)
 * h_out and y_out [tokens, heads * dim] (contiguous, either may be NULL) are
 * rounded once, y from the h before its rounding; codes and scales (both or
 * neither) are quantize_rows (inference/fp8_weights.py:16-19) of the y before
 * its rounding: ldc the codes' row stride, a multiple of 8, or 0 for the packed
 * order of jv_fp8_gemm in jv_fp8_packed_codes_bytes(tokens, heads * dim) bytes.
 *
 * x, residual, gate: bf16 (fp16 = 0) or fp16 (fp16 = 1), strides in elements
 * for tokens (`ts`) and heads (`hs`; residual is one row a token), 16-byte
 * aligned rows. post_weight: float32 [dim], weight: float32 [heads * dim], both
 * 16-byte aligned. A row has a multiple of 8 channels up to 16384; more than
 * one head: of 64, 128 or 256 channels. tokens below 2^22. eps at least 0.
 */
int jv_block_norm(const void* x, int64_t x_ts, int64_t x_hs, const void* residual, int64_t residual_ts, const void* gate,
                  int64_t gate_ts, int64_t gate_hs, int activation, const float* post_weight, float scale, const float* weight,
                  float eps, void* h_out, void* y_out, uint8_t* codes, int64_t ldc, float* scales, int64_t tokens,
                  int64_t heads, int64_t dim, int fp16, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* JEEVES_NORM_H */
