// C ABI of the serving operators (include/moe_serve.h): checks, workspace, and the order of launches.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "../../include/moe_serve.h"
#include "call.hpp"
#include "serve.hpp"

using namespace moe;

namespace {

constexpr size_t kMaxRows = (size_t)1 << 24;     // of a matrix
// tokens of a product at once, and values of theirs: 19 GB as terms of f32 rows at most, within 2^25 wavefronts' steps and 32-bit offsets
// in 16 tiles
constexpr size_t kMatmulTokens = 65536, kMatmulValues = (size_t)1 << 32;

int check_cols(size_t cols) {
  if (!cols || cols % 32 || cols > kMaxInter) return fail(MOE_ERR_INVALID, "cols %zu must be a positive multiple of 32, at most %zu", cols, kMaxInter);
  return MOE_OK;
}

int check_rule(const moe_routing *r, size_t T, size_t E) {
  if (!r) return fail(MOE_ERR_INVALID, "null rule");
  RETURN_IF(check_tokens(T));
  if (!E || E > 1024) return fail(MOE_ERR_INVALID, "n_experts %zu outside [1, 1024]", E);
  if (r->score != MOE_SCORE_SOFTMAX && r->score != MOE_SCORE_SIGMOID) return fail(MOE_ERR_INVALID, "score %d is neither MOE_SCORE_SOFTMAX nor MOE_SCORE_SIGMOID", r->score);
  if (!std::isfinite(r->scale)) return fail(MOE_ERR_INVALID, "scale is not finite");
  size_t most = E;
  if (r->n_groups > 1) {
    if (r->n_groups > 64 || E % r->n_groups) return fail(MOE_ERR_INVALID, "n_groups %zu must divide the %zu experts and be at most 64", r->n_groups, E);
    if (!r->top_groups || r->top_groups > r->n_groups) return fail(MOE_ERR_INVALID, "top_groups %zu outside [1, %zu]", r->top_groups, r->n_groups);
    if (r->group_score != MOE_GROUP_MAX && r->group_score != MOE_GROUP_TOP2) return fail(MOE_ERR_INVALID, "group_score %d is neither MOE_GROUP_MAX nor MOE_GROUP_TOP2", r->group_score);
    most = E / r->n_groups * r->top_groups;
  }
  if (!r->top_k || r->top_k > 32 || r->top_k > most) return fail(MOE_ERR_INVALID, "top_k %zu outside [1, min(32, %zu)]", r->top_k, most);
  return check_aligned({r->bias}, 4);
}

RouteRule rule_of(const moe_routing &r) {
  return RouteRule{r.score, r.normalize != 0, (int)r.top_k, r.n_groups > 1 ? (int)r.n_groups : 1, (int)r.top_groups,
                   r.group_score == MOE_GROUP_TOP2, r.scale, r.bias};
}

}  // namespace

extern "C" {

int moe_mxfp4_quantize_device(moe_ctx *ctx, const void *x, int dtype, size_t n, size_t cols, uint8_t *blocks, uint8_t *scales,
                              void *stream) {
  DenseCtx c;
  RETURN_IF(dense_ctx(ctx, &c));
  RETURN_IF(check_dtype(dtype));
  RETURN_IF(check_cols(cols));
  if (n > kMaxRows) return fail(MOE_ERR_INVALID, "n_rows %zu above %zu", n, kMaxRows);
  if (!n) return MOE_OK;
  if (!x || !blocks || !scales) return fail(MOE_ERR_INVALID, "null argument");
  RETURN_IF(check_aligned({x, blocks}));
  RETURN_IF(check_distinct({blocks, scales}, {x}));
  HIP_TRY(launch_mx4_quantize(x, dtype == MOE_BF16, n, cols, blocks, scales, stream ? (hipStream_t)stream : c.stream));
  return MOE_OK;
}

int moe_mxfp4_matmul_device(moe_ctx *ctx, const uint8_t *packed, size_t rows, size_t cols, const float *bias, const void *x, int x_type,
                            const uint8_t *x_scales, size_t T, void *y, int dtype, void *stream) {
  DenseCtx c;
  RETURN_IF(dense_ctx(ctx, &c));
  RETURN_IF(check_dtype(dtype));
  if (x_type < MOE_F32 || x_type > MOE_MXFP4) return fail(MOE_ERR_INVALID, "x_type %d is none of MOE_F32, MOE_BF16, MOE_MXFP8, MOE_MXFP4", x_type);
  RETURN_IF(check_cols(cols));
  if (!rows || rows % 16 || rows > kMaxRows) return fail(MOE_ERR_INVALID, "rows %zu must be a positive multiple of 16, at most %zu", rows, kMaxRows);
  RETURN_IF(check_tokens(T));
  if (!T) return MOE_OK;
  if (!packed || !x || !y) return fail(MOE_ERR_INVALID, "null packed, x or y");
  if (x_type == MOE_MXFP4 && !x_scales) return fail(MOE_ERR_INVALID, "rows of MOE_MXFP4 need x_scales");
  if (x_type == MOE_MXFP8 && !x_scales) x_scales = (const uint8_t *)x + T * cols;
  RETURN_IF(check_aligned({packed, x, y, bias}));
  RETURN_IF(check_distinct({y}, {packed, x, bias, x_scales}));
  const hipStream_t s = stream ? (hipStream_t)stream : c.stream;
  const size_t el = dtype == MOE_F32 ? 4 : 2;
  // bytes of a row of x
  const size_t xb = x_type == MOE_F32 ? 4 * cols : x_type == MOE_BF16 ? 2 * cols : x_type == MOE_MXFP8 ? cols : cols / 2;
  const size_t Tc = std::min({T, kMatmulTokens, kMatmulValues / cols / 16 * 16});
  MxGemmArgs a{};
  a.w = packed;
  a.d = pack_dims(rows, cols);
  a.bias = bias;
  a.bf16 = dtype == MOE_BF16;
  if (mx_one_takes(x_type, T, cols)) {
    a.r = mx_rows(x_type, T, cols);
    a.out = y;
    HIP_TRY(launch_mx_one(a, x, s));
    return MOE_OK;
  }
  Carve w;
  uint8_t *codes = nullptr;
  uint32_t *scales = nullptr;
  for (int placed = 0; placed < 2; placed++) {
    a.r = mx_rows(x_type, Tc, cols);
    codes = w.take<uint8_t>(mx_rows_code_bytes(a.r));
    scales = w.take<uint32_t>(mx_rows_scale_bytes(a.r) / 4);
    if (!placed) {
      RETURN_IF(ensure(c, w.off, s));
      w = Carve{(char *)c.work->p};
    }
  }
  for (size_t t0 = 0; t0 < T; t0 += Tc) {
    a.r = mx_rows(x_type, std::min(Tc, T - t0), cols);
    a.codes = codes;
    a.scales = scales;
    a.out = (char *)y + t0 * rows * el;
    HIP_TRY(launch_mx_rows(a.r, (const char *)x + t0 * xb, x_scales ? x_scales + t0 * (cols / 32) : nullptr, codes, scales, s));
    HIP_TRY(launch_mx_gemm(a, s));
  }
  return MOE_OK;
}

int moe_route_device(moe_ctx *ctx, const moe_routing *rule, const float *logits, size_t T, size_t E, int32_t *idx, float *weights,
                     int32_t *counts, void *stream) {
  DenseCtx c;
  RETURN_IF(dense_ctx(ctx, &c));
  RETURN_IF(check_rule(rule, T, E));
  if (T && (!logits || !idx || !weights)) return fail(MOE_ERR_INVALID, "null logits, idx or weights");
  RETURN_IF(check_aligned({logits, idx, weights, counts}, 4));
  RETURN_IF(check_distinct({idx, weights, counts}, {logits, rule->bias}));
  if (T || counts)
    HIP_TRY(launch_route_rule(rule_of(*rule), logits, T, (int)E, idx, weights, counts, stream ? (hipStream_t)stream : c.stream));
  return MOE_OK;
}

int moe_route_backward_device(moe_ctx *ctx, const moe_routing *rule, const float *logits, const int32_t *idx, const float *dweights, size_t T,
                              size_t E, float *dlogits, void *stream) {
  DenseCtx c;
  RETURN_IF(dense_ctx(ctx, &c));
  RETURN_IF(check_rule(rule, T, E));
  if (!T) return MOE_OK;
  if (!logits || !idx || !dweights || !dlogits) return fail(MOE_ERR_INVALID, "null argument");
  RETURN_IF(check_aligned({logits, idx, dweights, dlogits}, 4));
  RETURN_IF(check_distinct({dlogits}, {logits, idx, dweights}));
  HIP_TRY(launch_route_rule_backward(rule_of(*rule), logits, idx, dweights, T, (int)E, dlogits, stream ? (hipStream_t)stream : c.stream));
  return MOE_OK;
}

int moe_sample_device(moe_ctx *ctx, const moe_sampling *rule, const float *logits, size_t ld, const float *u, size_t T, size_t vocab,
                      int32_t *tokens, float *logprob, void *stream) {
  DenseCtx c;
  RETURN_IF(dense_ctx(ctx, &c));
  if (!rule) return fail(MOE_ERR_INVALID, "null rule");
  RETURN_IF(check_tokens(T));
  if (!vocab || vocab > kMaxVocab) return fail(MOE_ERR_INVALID, "vocab %zu outside [1, %zu]", vocab, kMaxVocab);
  if (ld < vocab) return fail(MOE_ERR_INVALID, "ld %zu below vocab %zu", ld, vocab);
  if (!T) return MOE_OK;
  if (!logits || !u || !tokens) return fail(MOE_ERR_INVALID, "null logits, u or tokens");
  RETURN_IF(check_aligned({logits, u, tokens, logprob, rule->temperature, rule->top_k, rule->top_p, rule->min_p}, 4));
  RETURN_IF(check_distinct({tokens, logprob}, {logits, u, rule->temperature, rule->top_k, rule->top_p, rule->min_p}));
  const hipStream_t s = stream ? (hipStream_t)stream : c.stream;
  const size_t Tc = std::min(T, sample_rows(vocab));
  RETURN_IF(ensure(c, sample_workspace(Tc, vocab), s));
  for (size_t t0 = 0; t0 < T; t0 += Tc) {
    auto at = [&](auto *p) { return p ? p + t0 : nullptr; };
    const SampleArgs a{moe_sampling{at(rule->temperature), at(rule->top_k), at(rule->top_p), at(rule->min_p)}, logits + t0 * ld, ld, u + t0,
                       (uint32_t)std::min(Tc, T - t0), (uint32_t)vocab, tokens + t0, at(logprob), c.work->p};
    HIP_TRY(launch_sample(a, s));
  }
  return MOE_OK;
}

}  // extern "C"
