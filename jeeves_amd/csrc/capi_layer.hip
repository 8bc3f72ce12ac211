// C ABI of the norms around a block, the short convolution and the linear
// attention (declared in include/jeeves_norm.h and
// include/jeeves_linear_attention.h): argument validation and launches only.
#include <cfloat>
#include <cmath>

#include "../../include/jeeves_fp8.h"
#include "../../include/jeeves_linear_attention.h"
#include "../../include/jeeves_norm.h"
#include "layer.h"

namespace {

using jv::fail;
using jv::hip_status;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Workgroups of 256 threads of a launch.
constexpr int64_t kMaxGrid = (int64_t(1) << 24) - 1;

int check_rows(const char* name, const void* p, int64_t ts, int64_t hs) {
  if (!p) return fail(JV_ERR_VALUE, "%s is missing", name);
  if (!aligned16(p) || ts % 8 || hs % 8) return fail(JV_ERR_VALUE, "%s needs 16-byte aligned rows", name);
  return JV_OK;
}

int check_weights(const char* name, const float* p) {
  return aligned16(p) ? JV_OK : fail(JV_ERR_VALUE, "%s needs a 16-byte aligned address", name);
}

int check_batch(int64_t tokens, int64_t batch, const int32_t* starts, const int32_t* slots, int64_t n_slots, const void* states) {
  if (tokens < 0 || tokens >= (1 << 24) || batch < 0 || batch > (1 << 20))
    return fail(JV_ERR_VALUE, "bad sizes: %lld tokens, batch %lld", (long long)tokens, (long long)batch);
  if (!starts && tokens != batch)
    return fail(JV_ERR_VALUE, "without query starts each of the %lld sequences has one token, got %lld", (long long)batch, (long long)tokens);
  if (tokens == 0) return JV_OK;
  if (batch == 0) return fail(JV_ERR_VALUE, "%lld tokens of no sequence", (long long)tokens);
  if (!slots) return fail(JV_ERR_VALUE, "the sequences' slots are missing");
  if (n_slots < 0 || n_slots > INT32_MAX || (n_slots && (!states || !aligned16(states))))
    return fail(JV_ERR_VALUE, "the states need a 16-byte aligned address and at most 2^31 - 1 slots");
  return JV_OK;
}

int check_dims(int64_t tokens, int64_t batch, int64_t k_heads, int64_t v_heads, int64_t k_dim, int64_t v_dim) {
  for (int64_t d : {k_dim, v_dim})
    if (d != 64 && d != 128 && d != 256) return fail(JV_ERR_VALUE, "heads of 64, 128 or 256 channels, got %lld", (long long)d);
  if (k_heads <= 0 || v_heads <= 0 || v_heads > 65536 || v_heads % k_heads)
    return fail(JV_ERR_VALUE, "%lld value heads are no multiple of %lld key heads", (long long)v_heads, (long long)k_heads);
  if (tokens < 0 || batch < 0 || tokens >= (1 << 24) || batch > (1 << 20) || tokens * v_heads >= (1 << 28) ||
      (jv::linear_chunks(tokens, batch) + tokens) * v_heads > kMaxGrid * 8 || jv::linear_chunks(tokens, batch) * v_heads > kMaxGrid ||
      batch * v_heads * (v_dim / 32) > kMaxGrid)
    return fail(JV_ERR_VALUE, "too many rows for one call: %lld tokens, batch %lld, %lld heads", (long long)tokens, (long long)batch,
                (long long)v_heads);
  return JV_OK;
}

}  // namespace

extern "C" {

int jv_block_norm(const void* x, int64_t x_ts, int64_t x_hs, const void* residual, int64_t residual_ts, const void* gate,
                  int64_t gate_ts, int64_t gate_hs, int activation, const float* post_weight, float scale, const float* weight,
                  float eps, void* h_out, void* y_out, uint8_t* codes, int64_t ldc, float* scales, int64_t tokens, int64_t heads,
                  int64_t dim, int fp16, void* stream) {
  if (heads <= 0 || dim <= 0 || heads > 16384 || dim > 16384 || heads * dim > 16384 || dim % 8)
    return fail(JV_ERR_VALUE, "a row has a multiple of 8 channels up to 16384, got %lld heads of %lld", (long long)heads, (long long)dim);
  if (heads > 1 && dim != 64 && dim != 128 && dim != 256)
    return fail(JV_ERR_VALUE, "heads of 64, 128 or 256 channels, got %lld", (long long)dim);
  if (tokens < 0 || tokens >= (1 << 22)) return fail(JV_ERR_VALUE, "bad sizes: %lld tokens", (long long)tokens);
  if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(JV_ERR_VALUE, "eps is finite and at least 0, got %g", eps);
  if (activation < JV_GATE_PLAIN || activation > JV_GATE_SILU) return fail(JV_ERR_VALUE, "unknown activation %d", activation);
  if (!codes != !scales) return fail(JV_ERR_VALUE, "codes and their scales come together");
  const int64_t cols = heads * dim;
  if (codes && (ldc == 0 ? cols % JV_FP8_BLOCK_K != 0 : ldc < cols || ldc % 8))
    return fail(JV_ERR_VALUE, "codes of %lld channels need a row stride of a multiple of 8, or whole steps of %d to be packed",
                (long long)cols, JV_FP8_BLOCK_K);
  if (tokens == 0) return JV_OK;
  if (int rc = check_rows("x", x, x_ts, heads > 1 ? x_hs : 0)) return rc;
  if (residual)
    if (int rc = check_rows("the residual", residual, residual_ts, 0)) return rc;
  if (gate)
    if (int rc = check_rows("the gate", gate, gate_ts, heads > 1 ? gate_hs : 0)) return rc;
  if (int rc = check_weights("the weight", post_weight)) return rc;
  if (int rc = check_weights("the weight", weight)) return rc;
  if (!aligned16(h_out) || !aligned16(y_out) || (reinterpret_cast<uintptr_t>(codes) & 15))
    return fail(JV_ERR_VALUE, "the outputs need 16-byte aligned addresses");
  jv::NormArgs a{};
  a.x = (const uint16_t*)x, a.residual = (const uint16_t*)residual, a.gate = (const uint16_t*)gate;
  a.x_ts = x_ts, a.x_hs = x_hs, a.residual_ts = residual_ts, a.gate_ts = gate_ts, a.gate_hs = gate_hs;
  a.activation = activation, a.post_weight = post_weight, a.weight = weight, a.scale = scale, a.eps = eps;
  a.h_out = (uint16_t*)h_out, a.y_out = (uint16_t*)y_out, a.codes = codes, a.ldc = ldc, a.scales = scales;
  a.tokens = (int)tokens, a.heads = (int)heads, a.dim = (int)dim, a.cols = (int)cols;
  return hip_status(jv::block_norm(a, fp16 != 0, (hipStream_t)stream), "norm launch");
}

int jv_causal_conv(const void* x, int64_t x_ts, const float* weight, const float* bias, int64_t width, int activation,
                   void* states, int64_t n_slots, const int32_t* slots, const int32_t* from_slots, const int32_t* starts,
                   int64_t batch, void* out, int64_t tokens, int64_t channels, int fp16, void* stream) {
  if (width < 2 || width > 4) return fail(JV_ERR_VALUE, "the convolution takes 2 to 4 inputs, got %lld", (long long)width);
  if (channels <= 0 || channels > 65536 || channels % 8)
    return fail(JV_ERR_VALUE, "the convolution takes a multiple of 8 channels up to 65536, got %lld", (long long)channels);
  if (activation != JV_CONV_PLAIN && activation != JV_CONV_SILU) return fail(JV_ERR_VALUE, "unknown activation %d", activation);
  if (int rc = check_batch(tokens, batch, starts, slots, n_slots, states)) return rc;
  if ((tokens + 1) * ((channels + 255) / 256) / 4 >= kMaxGrid)
    return fail(JV_ERR_VALUE, "too many rows for one call: %lld tokens of %lld channels", (long long)tokens, (long long)channels);
  if (tokens == 0) return JV_OK;
  if (int rc = check_rows("x", x, x_ts, 0)) return rc;
  if (int rc = check_rows("the output", out, 0, 0)) return rc;
  if (!weight) return fail(JV_ERR_VALUE, "the weight is missing");
  if (int rc = check_weights("the weight", weight)) return rc;
  if (int rc = check_weights("the bias", bias)) return rc;
  jv::ConvArgs a{};
  a.x = (const uint16_t*)x, a.x_ts = x_ts, a.weight = weight, a.bias = bias, a.activation = activation;
  a.states = (uint16_t*)states;
  a.b = {starts, slots, from_slots ? from_slots : slots, n_slots, (int)tokens, (int)batch};
  a.out = (uint16_t*)out, a.channels = (int)channels;
  return hip_status(jv::causal_conv(a, (int)width, fp16 != 0, (hipStream_t)stream), "convolution launch");
}

int64_t jv_linear_attention_workspace_bytes(int64_t tokens, int64_t batch, int64_t k_heads, int64_t v_heads, int64_t k_dim,
                                            int64_t v_dim, int ragged) {
  if (check_dims(tokens, batch, k_heads, v_heads, k_dim, v_dim)) return -1;
  return ragged && tokens && batch ? jv::linear_workspace(tokens, batch, k_heads, v_heads, k_dim) : 0;
}

int jv_linear_attention(const void* q, int64_t q_ts, int64_t q_hs, const void* k, int64_t k_ts, int64_t k_hs, const void* v,
                        int64_t v_ts, int64_t v_hs, const void* decay, int64_t decay_ts, const void* beta, int64_t beta_ts,
                        int gates16, const float* rate, const float* decay_bias, float norm_eps, float* states, int64_t n_slots,
                        const int32_t* slots, const int32_t* from_slots, const int32_t* starts, int64_t batch, float scale,
                        void* out, int64_t tokens, int64_t k_heads, int64_t v_heads, int64_t k_dim, int64_t v_dim, int fp16,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_dims(tokens, batch, k_heads, v_heads, k_dim, v_dim)) return rc;
  if (int rc = check_batch(tokens, batch, starts, slots, n_slots, states)) return rc;
  if (!std::isfinite(scale)) return fail(JV_ERR_VALUE, "the scale must be finite, got %g", scale);
  if (norm_eps != 0.0f && !(norm_eps >= FLT_MIN && std::isfinite(norm_eps)))
    return fail(JV_ERR_VALUE, "norm_eps is 0 or a normal float32, got %g", norm_eps);
  if (decay_bias && !rate) return fail(JV_ERR_VALUE, "a decay bias goes with the heads' rates");
  if (tokens == 0) return JV_OK;
  if (int rc = check_rows("q", q, q_ts, q_hs)) return rc;
  if (int rc = check_rows("k", k, k_ts, k_hs)) return rc;
  if (int rc = check_rows("v", v, v_ts, v_hs)) return rc;
  if (int rc = check_rows("the output", out, 0, 0)) return rc;
  if (!decay) return fail(JV_ERR_VALUE, "the decays are missing");
  const int64_t need = starts ? jv::linear_workspace(tokens, batch, k_heads, v_heads, k_dim) : 0;
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255)))
    return fail(JV_ERR_VALUE, "workspace needs %lld bytes, 256-byte aligned", (long long)need);
  jv::LinearArgs a{};
  a.q = (const uint16_t*)q, a.k = (const uint16_t*)k, a.v = (const uint16_t*)v;
  a.q_ts = q_ts, a.q_hs = q_hs, a.k_ts = k_ts, a.k_hs = k_hs, a.v_ts = v_ts, a.v_hs = v_hs;
  a.decay = decay, a.beta = beta, a.decay_ts = decay_ts, a.beta_ts = beta_ts, a.gates16 = gates16;
  a.rate = rate, a.decay_bias = decay_bias, a.norm_eps = norm_eps;
  a.states = states;
  a.b = {starts, slots, from_slots ? from_slots : slots, n_slots, (int)tokens, (int)batch};
  a.scale = scale, a.out = (uint16_t*)out;
  a.k_heads = (int)k_heads, a.v_heads = (int)v_heads, a.group = (int)(v_heads / k_heads);
  a.workspace = (uint8_t*)workspace;
  const auto run = starts ? jv::linear_prompt : jv::linear_step;
  return hip_status(run(a, (int)k_dim, (int)v_dim, fp16 != 0, (hipStream_t)stream), "linear attention launch");
}

}  // extern "C"
