/*
 * moe_dense.h — C ABI of the dense operators beside the MXFP4 mixture-of-experts path: the loss over
 * the LM head and its gradient, a gated feed-forward block with bf16 weights and its backward pass,
 * and activation checkpoints in 8 bits. Status codes, moe_last_error() and contexts are those of
 * mxfp4_moe.h. The reference has no counterpart: it answers with logits and does not train
 * (src/gpt_oss/session.rs:983-1030 is its LM head, :87-124 its feed-forward arithmetic).
 *
 * All calls take device pointers, 16-byte aligned unless said otherwise, and are asynchronous on
 * `stream` (a hipStream_t, NULL = the context's stream). Matrices are contiguous, rows first. No
 * output may overlap an input or another output.
 *
 * Types of activations and of their gradients (`dtype`): MOE_F32, the rows that the other calls of a
 * context take and return, or MOE_BF16. Weights are bf16, biases f32. Products accumulate in f32: bf16
 * values enter as they are, f32 values as three bf16 terms (their 24 bits, as far as those lie above
 * 2^-126; a finite value that rounds to bf16's infinity, above 3.39e38, as an infinity). An infinity or NaN
 * among the rows makes of the results what it does in f32; an infinite weight makes NaN of the results of
 * f32 rows that it enters. The logits' gradient, the activation h and the gradients of gate and up enter
 * the products after them in `dtype`'s precision: one bf16 rounding (2^-8 relative) for MOE_BF16, none that
 * f32 would not make for MOE_F32. Results depend on the arguments' values, the shapes and which gradients
 * are asked for, and on nothing else: no atomics.
 *
 * Workspace: the context's, which grows at need (the old one is kept if a captured graph may hold it). A
 * call that grows it allocates and waits for the device; lengths that rise little by little do so now and
 * then, as it grows with room. Bytes a token, about: the loss 6 H for MOE_F32 (of up to 16384 tokens at
 * once) and up to 512 MB; its gradient 2 H (MOE_BF16) or 12 H (MOE_F32), 4 H for dx of MOE_BF16, and up to
 * 2 GB; the block forward 2 I or 6 (H + I), backward 14 I or 24 H + 44 I, all tokens at once, and K parts
 * (65536 tokens of 2880 x 2880 backward: 2.7 or 14.2 GB). MOE_ERR_OOM where there is no memory for it.
 * During stream capture it cannot grow (MOE_ERR_STATE): run the same call once before. As for every call of
 * a context, calls that share one, replays of graphs that hold one included, must not overlap. A graph also
 * holds the LM head: capture it again after a moe_init_lm_head_bf16(_device) with more rows.
 */
#ifndef MOE_DENSE_H
#define MOE_DENSE_H

#include "mxfp4_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

enum moe_dtype {
  MOE_F32 = 0,
  MOE_BF16 = 1,
  MOE_MXFP8 = 2 /* moe_act8_pack_device's form, where a call says that it takes it */
};

/* ------------------------------------------------------------------ loss over the LM head */

/* Softmax cross entropy over the LM head's first `vocab` rows (moe_init_lm_head_bf16(_device), with the
 * hidden sizes that it takes; not the f32 head), at most 2^28, in pieces of the vocabulary: no logits are kept. For each of n_tokens rows x [H]:
 *   lse = log sum_v exp(x . W_v), loss = lse - x . W_target.
 * targets [n_tokens] (4-byte aligned, as are loss, lse and dloss): a negative target is ignored (loss 0, no
 * gradient); one of vocab or more gives NaN. n_tokens 0 does nothing; at most 2^20. */
int moe_lm_head_loss_device(moe_ctx *ctx, const void *x, int dtype, const int32_t *targets, size_t n_tokens,
                            size_t vocab, float *loss, float *lse, void *stream);
/* Its gradient: with p = exp(x . W - lse), d = dloss (p - [v = target]) (0 for ignored tokens):
 *   dx [n_tokens, H] = d W, dw [vocab, H] = d^T x, both of type `dtype`, either may be NULL. The rows of
 * ignored tokens may hold anything.
 * lse as moe_lm_head_loss_device returned it; dloss [n_tokens] f32, the gradient of each token's loss.
 * (dloss at tokens with a gradient has one scale: terms of d below 2^-126 of its largest magnitude may
 * count as 0; at the others it may hold anything.)
 * n_tokens 0 zeroes dw. The head's rows are read, not changed: after an update of the weights call
 * moe_init_lm_head_bf16_device again. */
int moe_lm_head_loss_backward_device(moe_ctx *ctx, const void *x, int dtype, const int32_t *targets,
                                     const float *lse, const float *dloss, size_t n_tokens, size_t vocab,
                                     void *dx, void *dw, void *stream);

/* ------------------------------------------------------------------ gated feed-forward block */

/* Weights of a block: hidden size H of the context, inner size `inter` (a multiple of 8). Layout of the
 * experts' (row 2i of gate_up is gate i, row 2i + 1 up i). Biases may be NULL. */
typedef struct moe_ffn {
  size_t inter;
  const uint16_t *gate_up;   /* [2 inter, H] bf16 bits */
  const float *gate_up_bias; /* [2 inter] */
  const uint16_t *down;      /* [H, inter] */
  const float *down_bias;    /* [H] */
} moe_ffn;

/* y [n_tokens, H] = down(h), h = (clamp(u, +-c) + 1) min(g, c) sigmoid(1.702 min(g, c)), the experts'
 * activation with the context's swiglu_clamp c; a NaN stays a NaN. x8 (may be NULL): also x as an 8-bit
 * checkpoint (moe_act8_bytes(n_tokens, H) bytes), for the backward pass to read in place of x. */
int moe_ffn_forward_device(moe_ctx *ctx, const moe_ffn *block, const void *x, int dtype, size_t n_tokens,
                           void *y, uint8_t *x8, void *stream);

/* Gradients to compute; each may be NULL. x [n_tokens, H], gate_up [2 inter, H] and down [H, inter] of
 * type `dtype`, the biases f32. They are written, not added to. */
typedef struct moe_ffn_grads {
  void *x;
  void *gate_up;
  float *gate_up_bias;
  void *down;
  float *down_bias;
} moe_ffn_grads;

/* The gradients from x and dy = d loss / d y. Nothing else is kept from the forward pass: gate and up are
 * computed again. x_type: `dtype`, or MOE_MXFP8 for the checkpoint that the forward pass wrote (its
 * values, exactly, take x's place). At and below a clamp's limit the gradient passes, above it is 0.
 * n_tokens 0 zeroes the gradients. */
int moe_ffn_backward_device(moe_ctx *ctx, const moe_ffn *block, const void *x, int x_type, const void *dy,
                            int dtype, size_t n_tokens, const moe_ffn_grads *grads, void *stream);

/* ------------------------------------------------------------------ 8-bit activation checkpoints */

/* MXFP8: e4m3 codes [n_tokens, cols], then one E8M0 scale per 32 values [n_tokens, cols / 32]. cols is a
 * multiple of 32. The scale is the smallest power of two (at least 2^-127) at which no value of the block
 * exceeds e4m3's 448; codes are rounded to nearest even. A block that holds a value that is not finite
 * has scale byte 255 and reads back as NaN. Every code times its scale is exact in bf16 and f32 (bf16:
 * down to 2^-133). moe_act8_bytes returns 0 for cols that are no multiple of 32. */
size_t moe_act8_bytes(size_t n_tokens, size_t cols);
int moe_act8_pack_device(moe_ctx *ctx, const void *x, int dtype, size_t n_tokens, size_t cols, uint8_t *packed,
                         void *stream);
int moe_act8_unpack_device(moe_ctx *ctx, const uint8_t *packed, size_t n_tokens, size_t cols, void *out,
                           int dtype, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* MOE_DENSE_H */
