/*
 * moe_serve.h — C ABI of the operators that serve a model's other layers beside the MXFP4 mixture-of-experts
 * path: rows and weights quantised to MXFP4, products with a resident MXFP4 matrix for any number of rows, the
 * choice of experts by other rules than the path's own (with its gradient), and the choice of a token from
 * logits. Status codes, moe_last_error(), contexts, types of rows, workspace and graph capture are those of
 * mxfp4_moe.h and moe_dense.h. The reference has no counterpart: it decodes checkpoints that others
 * quantised (src/gpt_oss/weights.rs:350-371), takes matvecs of one row (src/gpt_oss/session.rs:16-85), knows
 * one routing rule (session.rs:818-841), and samples on the host.
 *
 * All calls take device pointers and are asynchronous on `stream` (a hipStream_t, NULL = the context's
 * stream). Matrices are contiguous, rows first, unless a stride is given. No output may overlap an input or
 * another output. Results depend on the arguments' values and shapes, and on nothing else. What lies behind the last row
 * of an output is left as it was. n_tokens is at most 2^20.
 */
#ifndef MOE_SERVE_H
#define MOE_SERVE_H

#include "moe_dense.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Beside enum moe_dtype, for rows that a product takes: MXFP4, moe_mxfp4_quantize_device's form. */
enum { MOE_MXFP4 = 3 };

/* ------------------------------------------------------------------ MXFP4 quantisation */

/* Rows x [n_rows, cols] (dtype MOE_F32 or MOE_BF16, 16-byte aligned) as MXFP4 in the checkpoint's layout:
 * blocks [n_rows, cols / 32, 16] (16-byte aligned) and scales [n_rows, cols / 32]. cols is a multiple of 32, at
 * most 2^20; n_rows at most 2^24. A block of 32 values has the OCP MX scale 2^(floor(log2 of its largest
 * magnitude) - 2), at least 2^-126 (byte 1: moe_mxfp4_dequant_device reads byte 0 as 0); codes are E2M1,
 * rounded to nearest even, at most 6. A block that holds a value that is not finite has scale byte 255 and
 * codes 0, which read back as NaN. moe_mxfp4_dequant_device reads rows back, moe_mxfp4_pack_device makes
 * weights resident, moe_preload_layer_device takes experts so quantised. */
int moe_mxfp4_quantize_device(moe_ctx *ctx, const void *x, int dtype, size_t n_rows, size_t cols, uint8_t *blocks,
                              uint8_t *scales, void *stream);

/* ------------------------------------------------------------------ MXFP4 product */

/* y [n_tokens, rows] = x W^T (+ bias [rows], f32, may be NULL) of a resident MXFP4 matrix W [rows, cols]
 * (moe_mxfp4_pack_device), y of type dtype (MOE_F32 or MOE_BF16). Rows x [n_tokens, cols] by x_type:
 *   MOE_F32: of a block of 32 values those down to 2^-5 of its largest magnitude enter exactly, none is off
 *     by more than 2^-29 of that;
 *   MOE_BF16: exactly (weights of 2^128 and above are infinite, as in f32);
 *   MOE_MXFP8: moe_act8_pack_device's codes, their scales at x_scales, or behind the codes if that is NULL;
 *   MOE_MXFP4: blocks as moe_mxfp4_quantize_device writes them, their scales at x_scales.
 * Products are exact, sums f32. Blocks of f32 rows whose largest magnitude is below 2^-99 keep 2^-129 absolute. A row that
 * holds a value that is not finite, or a scale byte of 255, gives NaN, as does a scale byte of 255 in W; a scale byte of 0
 * counts as 2^-127. packed, x, y and bias are 16-byte aligned; rows is a multiple of 16, at most 2^24, cols of 32, at most
 * 2^20. Workspace: the rows as the product takes them, 0.53 cols bytes a token for MOE_MXFP4, 2.03 for MOE_MXFP8, 2 for
 * MOE_BF16 and 4.53 for MOE_F32, of 65536 tokens at a time (fewer of above 65536 cols); none for one row of MOE_F32 of up to
 * 10624 cols, two of up to 5248, and up to 16 rows of MOE_BF16 of 48 KB in all (each 2 cols, rounded up to 256, and 16
 * bytes). (moe_mxfp4_matvec_device takes one f32 row as well, exact to 2^-16 of it: 4.8 us over 5760 x 2880, where this
 * takes 5.1.) */
int moe_mxfp4_matmul_device(moe_ctx *ctx, const uint8_t *packed, size_t rows, size_t cols, const float *bias,
                            const void *x, int x_type, const uint8_t *x_scales, size_t n_tokens, void *y, int dtype,
                            void *stream);

/* ------------------------------------------------------------------ routing */

enum moe_score { MOE_SCORE_SOFTMAX = 0, MOE_SCORE_SIGMOID = 1 };
enum moe_group_score { MOE_GROUP_MAX = 0, MOE_GROUP_TOP2 = 1 };

/* A routing rule. With normalize 1, scale 1 and zeros otherwise: the path's own. */
typedef struct moe_routing {
  int score;         /* of a token's logits: softmax over all experts, or the sigmoid of each */
  int normalize;     /* not 0: the weights are divided by their sum */
  size_t top_k;      /* 1 to 32 */
  size_t n_groups;   /* 0 or 1: none; else the experts form n_groups (at most 64) groups of as many, side by side */
  size_t top_groups; /* groups that experts are chosen from, with n_groups above 1 */
  int group_score;   /* a group's score: its largest, or the sum of its two largest */
  float scale;       /* of the weights; finite */
  const float *bias; /* [n_experts] on the device or NULL: added to the scores for the choice alone, not for the weights */
} moe_routing;

/* For each of n_tokens rows of logits [n_experts] (f32, n_experts at most 1024) the chosen experts idx
 * [n_tokens, top_k] in falling order of score (+ bias) and their weights [n_tokens, top_k]; counts [n_experts]
 * (may be NULL): how often each was chosen. Equal scores go to the lower index, for groups as well. Without a bias
 * the order of experts is that of their logits; otherwise scores are compared in 64 bits. An expert whose logit is
 * -inf or NaN is never chosen: slots without an expert hold idx -1, weight 0. (A group with one expert left has
 * that one's score, a group with none is taken last.) Infinite logits share a softmax among them; a score of a
 * softmax below 2^-1075 is 0. Weights whose sum is 0 are uniform if normalised (and have no gradient); those of a sigmoid's
 * finite logits, however far below 0, are what the formula says. All pointers 4-byte aligned. n_tokens 0 zeroes counts. */
int moe_route_device(moe_ctx *ctx, const moe_routing *rule, const float *logits, size_t n_tokens, size_t n_experts,
                     int32_t *idx, float *weights, int32_t *counts, void *stream);
/* Gradient of sum(dweights * weights) with respect to the logits, dlogits [n_tokens, n_experts], for the choice idx that
 * moe_route_device made (the choice itself has no gradient, nor has the bias). Slots of idx outside [0, n_experts)
 * are left out. */
int moe_route_backward_device(moe_ctx *ctx, const moe_routing *rule, const float *logits, const int32_t *idx,
                              const float *dweights, size_t n_tokens, size_t n_experts, float *dlogits, void *stream);

/* ------------------------------------------------------------------ sampling */

/* Settings of each row, device arrays [n_tokens] (4-byte aligned); NULL: 1, off, off, off. */
typedef struct moe_sampling {
  const float *temperature; /* not above 0 (or NaN): the largest logit */
  const int32_t *top_k;     /* the k largest logits; below 1: all */
  const float *top_p;       /* of these the fewest largest whose probabilities reach top_p of theirs; 1 and above: all */
  const float *min_p;       /* those with at least min_p times the largest probability; 0 and below: all */
} moe_sampling;

/* A token for each of n_tokens rows of logits [vocab] (f32, 4-byte aligned, row t at logits + t ld, vocab at most
 * 2^28): among the tokens that the settings leave (of equal logits the lower index first, and always a largest one), the
 * first in the vocabulary's order at which the sum of their probabilities passes u[t] (in [0, 1); below counts as 0,
 * 1 and above as the last). tokens [n_tokens]; logprob [n_tokens] (may be NULL): the logarithm of its
 * probability among those left, 0 where the temperature is not above 0. Probabilities are multiples of 2^-44 of the
 * largest (2^-(62 - log2 vocab), the logarithm rounded up, for a vocab above 2^18), their sums exact. A NaN logit counts as -inf, infinite ones
 * share the row; a row without a logit above -inf gives token -1, logprob NaN. Workspace: 57 KB a row and 21 bytes for every
 * 1024 logits, of 4096 rows at a time (fewer of a vocab above 2^23). Where more than 4096 logits have to be looked at for a
 * row's border (those within 1/64 of a temperature of it; of a top-k up to 2048 all that are not surely below its border) the
 * row takes longer: of 201088 logits 1 to 2.6 ms. */
int moe_sample_device(moe_ctx *ctx, const moe_sampling *rule, const float *logits, size_t ld, const float *u, size_t n_tokens,
                      size_t vocab, int32_t *tokens, float *logprob, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* MOE_SERVE_H */
