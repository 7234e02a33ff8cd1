/*
 * mi_moe_layer.h -- what a decoder layer runs around the expert block of mi_moe.h: the norm with the residual's addition (and its backward pass), the choice
 * of experts for routers that mi_moe_route does not cover (and its backward pass), the block on a routing of the caller's, and linear layers on rows in
 * eight bits.  Same library, same conventions as mi_moe.h: int status and mi_moe_last_error, device pointers, work enqueued on `stream`, nothing
 * allocated and nothing kept by a call; arrays are row-major and contiguous, and need no more alignment than their elements' unless a comment says so.
 */
#ifndef MI_MOE_LAYER_H
#define MI_MOE_LAYER_H

#include "mi_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- norm ---- */
/* The residual's addition and the norm behind it in one pass: sum = round(x + residual), y = the norm of sum (what stands
 * between two sublayers, mlx-lm/src/models/qwen3.rs:310-325; in bfloat16 the bits of mi_moe_rms_norm on sum).
 * x, residual, weight, sum, y: element type dtype (mi_moe_dtype), [T, hidden] and [hidden]; hidden: any number up to 32768.  residual NULL: nothing is added, and sum may be NULL, too.  sum may be x or residual itself (an
 * update in place); y must overlap none of the others. */
int mi_moe_add_rms_norm(const void *x, const void *residual, const void *weight, float eps, int64_t T,
                        int32_t hidden, int32_t dtype, void *sum, void *y, void *stream);
/* The same with the normalised rows z in eight bits: row_scales[t] = max |z[t]| / 127 (f32 [T]) and rows8 (signed bytes [T, hidden]) the integers
 * nearest to z / row_scales, ties to even, decided on the exact products of weight and sum.  A row of zeros has a scale of zero;
 * one that holds an infinity or a NaN has zeros in rows8 and a NaN for its scale. */
int mi_moe_add_rms_norm_rows8(const void *x, const void *residual, const void *weight, float eps,
                              int64_t T, int32_t hidden, int32_t dtype, void *sum, void *rows8,
                              float *row_scales, void *stream);
/* Its backward pass.  sum: what the forward call returned (or its x); dy, dsum: the gradients that arrive at y and at sum (dsum NULL:
 * none).  dx [T, hidden]: the gradient of x and of residual alike; dweight [hidden]: summed over the rows in float32 in a fixed
 * order (T = 0: zeros).  dx may be dy, dsum or sum itself.  workspace >= mi_moe_add_rms_norm_grad_workspace_size, 16-byte aligned. */
int mi_moe_add_rms_norm_grad_workspace_size(int64_t T, int32_t hidden, size_t *bytes);
int mi_moe_add_rms_norm_grad(const void *dy, const void *sum, const void *dsum, const void *weight,
                             float eps, int64_t T, int32_t hidden, int32_t dtype, void *dx, void *dweight,
                             void *workspace, size_t workspace_bytes, void *stream);

/* ---- Experts from logits, for routers that mi_moe_route does not cover (the op sequence softmax or sigmoid / add / reshape / topk / where /
 * argpartition / take_along_axis / divide; mlx-rs/src/ops/sort.rs:211-260, ops/indexing/mod.rs:433-453).
 * Scores s of a token's logits [n_experts] (element type dtype): softmax over the experts, or sigmoid.  Experts are ordered by s + bias
 * (f32 [n_experts], takes part in the choice alone), without a bias by the logits themselves; ties go to the lower id.  n_groups
 * (a divisor of n_experts, up to 64) runs of consecutive experts: only the best top_groups of them are open, by their largest key or by the sum of their two
 * largest s + bias (group_score; the largest alone in groups of one; an expert whose logit is -inf or NaN has a part in such a sum with a score of zero, one
 * whose bias is -inf or NaN none).  A group without an expert whose logit and bias are above -inf comes after all others.  Weights: scale * s, divided by the sum of the chosen s with renormalize
 * (a sum of zero gives zeros).  Scores are computed and compared in float64.  topk_idx [T, top_k], best first; topk_w of element type
 * w_dtype.  An expert whose logit is -inf is chosen only where no other of the open groups is left, one whose logit is NaN after those; neither changes another's score.
 * n_experts 1..512, top_k 1..min(32, top_groups * n_experts / n_groups). ---- */
typedef enum { MI_MOE_SCORING_SOFTMAX = 0, MI_MOE_SCORING_SIGMOID = 1 } mi_moe_scoring;
typedef enum { MI_MOE_GROUP_SCORE_MAX = 0, MI_MOE_GROUP_SCORE_TOP2 = 1 } mi_moe_group_score;
int mi_moe_select_experts(const void *logits, int32_t dtype, const float *bias, int64_t T,
                          int32_t n_experts, int32_t top_k, int32_t scoring, int32_t n_groups,
                          int32_t top_groups, int32_t group_score, int32_t renormalize, float scale,
                          uint32_t *topk_idx, void *topk_w, int32_t w_dtype, void *stream);
/* The gradient of the weights with respect to the logits, the choice taken as given: dlogits [T, n_experts] of element type dtype from dw
 * [T, top_k] of element type w_dtype.  Ids outside the experts contribute nothing; an expert named twice gets both terms. */
int mi_moe_select_experts_grad(const void *dw, int32_t w_dtype, const void *logits, int32_t dtype,
                               const uint32_t *topk_idx, int64_t T, int32_t n_experts, int32_t top_k,
                               int32_t scoring, int32_t renormalize, float scale, void *dlogits,
                               void *stream);

/* The block with a routing of the caller's (mi_moe_select_experts, or any other): mi_moe_forward behind its router.
 * topk_idx [T, top_k], topk_w bf16 [T, top_k]; the handle's router is not used.  A token that names an expert twice gets it
 * once, with the sum of its weights (one rounding to bf16); an id outside the experts (a padded slot) contributes nothing.  dbg->topk_idx and topk_w
 * hold the routing as the kernels took it: another expert with a weight of -0 in such slots, whose result is computed and left out (also where it is not finite).  Same workspace as mi_moe_forward. */
int mi_moe_forward_routed(mi_moe_handle h, const uint16_t *x, const uint32_t *topk_idx,
                          const uint16_t *topk_w, int64_t T, uint16_t *out, void *workspace,
                          size_t workspace_bytes, const mi_moe_debug_out *dbg, void *stream);

/* ---- The linear layer on rows in eight bits (mi_moe_add_rms_norm_rows8 makes such rows): y = (row_scales x) . dequantize(w)^T + linear_bias, each result
 * rounded once.  x: signed bytes [M, K]; row_scales: f32 [M]; w [N, K*bits/32]; scales, biases [N, K/group_size], linear_bias [N]
 * (or NULL) and y [M, N] of element type dtype.  bits 4 or 8; group_size 32, 64 or 128; K a multiple of group_size; N up to 2^26 - 4.  Products of rows and codes are summed exactly, as integers,
 * over runs of a group; everything else in float32.
 * The fast kernels want K a multiple of 128 and x, w, scales and biases 16-byte aligned; those for many rows an even number of 16-bit scales a column and
 * workspace >= mi_moe_quantized_linear_rows8_workspace_size (16-byte aligned; 0 for up to 16 rows), too.  Without these, slower kernels give the same product. ---- */
int mi_moe_quantized_linear_rows8_workspace_size(int64_t M, int32_t K, size_t *bytes);
int mi_moe_quantized_linear_rows8(const void *x, const float *row_scales, const uint32_t *w,
                                  const void *scales, const void *biases, const void *linear_bias,
                                  int64_t M, int32_t N, int32_t K, int32_t group_size, int32_t bits,
                                  int32_t dtype, void *y, void *workspace, size_t workspace_bytes,
                                  void *stream);

#ifdef __cplusplus
}
#endif
#endif /* MI_MOE_LAYER_H */
