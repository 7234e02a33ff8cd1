/*
 * mi_moe_f8.h -- experts and linear layers whose weights are 8-bit floating point (e4m3: sign, four bits of exponent, three of mantissa, largest value 448, no
 * infinity), with a float32 scale for each block of 128 x 128, as checkpoints in that form hold them; tokens sorted by expert and back; and the gradients of all of
 * these for fine-tuning on frozen weights.  Same library, same conventions as mi_moe.h: int status and mi_moe_last_error, device pointers, work enqueued on `stream`,
 * nothing allocated and nothing kept by a call; arrays are row-major and contiguous, and need no more alignment than their elements' unless a comment says so.  What a call writes
 * overlaps none of its operands.
 */
#ifndef MI_MOE_F8_H
#define MI_MOE_F8_H

#include "mi_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Tokens sorted by expert (the op sequence argsort / floor_divide / take of a gather-sorted block; mlx-rs/src/ops/sort.rs:75-109, ops/indexing/mod.rs:386-401).
 * topk_idx [T, top_k].  The pairs t * top_k + s are sorted by expert, stably; slots whose id is outside the experts (padding) come last.
 *   rows [T * top_k, hidden]   row r is x[order[r] / top_k]; rows of slots that name no expert are zeros
 *   order u32 [T * top_k]      the sorted pairs
 *   inverse i32 [T, top_k]     a slot's row, -1 - row where it names no expert
 *   offsets u32 [n_experts+1]  expert e has the rows from offsets[e] to offsets[e + 1]
 * x and rows of element type dtype; hidden any number, top_k 1..32, n_experts 1..512, T * top_k up to 2^24 - 1; rows and x may be NULL (then only the places are found).
 * workspace >= mi_moe_sort_tokens_workspace_size, 16-byte aligned (0 bytes for up to 2048 pairs). ---- */
int mi_moe_sort_tokens_workspace_size(int64_t T, int32_t top_k, int32_t n_experts, size_t *bytes);
int mi_moe_sort_tokens(const void *x, const uint32_t *topk_idx, int64_t T, int32_t top_k, int32_t n_experts,
                       int32_t hidden, int32_t dtype, void *rows, uint32_t *order, int32_t *inverse,
                       uint32_t *offsets, void *workspace, size_t workspace_bytes, void *stream);
/* Its gradient: dx[t] = the sum of drows over the rows of token t's named slots, in float32 in the slots' order. */
int mi_moe_sort_tokens_grad(const void *drows, const int32_t *inverse, int64_t T, int32_t top_k,
                            int32_t hidden, int32_t dtype, void *dx, void *stream);
/* Back to tokens: out[t] = sum over the named slots of topk_w[t][s] * row, in float32 in the slots' order, rounded once.  topk_w [T, top_k] of element type
 * w_dtype.  What rows hold where no slot names them has no part in it, whatever it is.  A place in `inverse` outside the T * top_k rows counts as no expert. */
int mi_moe_unsort_tokens(const void *rows, const void *topk_w, int32_t w_dtype, const int32_t *inverse,
                         int64_t T, int32_t top_k, int32_t hidden, int32_t dtype, void *out, void *stream);
/* Its gradients: drows (zeros in the rows of slots that name no expert) and dweights [T, top_k] of element type w_dtype (zeros in such slots). */
int mi_moe_unsort_tokens_grad(const void *dout, const void *rows, const void *topk_w, int32_t w_dtype,
                              const int32_t *inverse, int64_t T, int32_t top_k, int32_t hidden, int32_t dtype,
                              void *drows, void *dweights, void *stream);

/* ---- e4m3 with scales.  x [rows, cols] of element type dtype.  block_rows 128: a scale for each block of 128 x 128 (weights); 1: for each run of 128 values of a row.
 * scales f32 [ceil(rows / block_rows), ceil(cols / 128)] = round(max |x| / 448), codes the e4m3 values nearest to round(x / scale), ties to even, both roundings to
 * float32.  A block of zeros has a scale of zero and codes of zero; one that holds an infinity or a NaN a scale that is NaN and codes of zero.  cols up to 2^22. ---- */
int mi_moe_quantize_f8(const void *x, int32_t dtype, int64_t rows, int64_t cols, int32_t block_rows,
                       void *codes, float *scales, void *stream);
int mi_moe_dequantize_f8(const void *codes, const float *scales, int64_t rows, int64_t cols,
                         int32_t block_rows, int32_t dtype, void *out, void *stream);

/* ---- The linear layer on such weights: y = q(x) . W^T + linear_bias (transpose), or y = q(x) . W, which is its gradient with respect to its input.
 * q: rows to e4m3 with a scale for each run of 128 values, as mi_moe_quantize_f8 makes them.  x [M, K], y [M, N] and linear_bias [N] (transpose only; or NULL) of element
 * type dtype, sums in float32, each result rounded once.  W [N, K] (transpose; K a multiple of 16) or [K, N] (N a multiple of 16), 16-byte aligned; scales of its blocks.
 * M N and M K up to 2^35, N and K up to 2^22.  float16 and float32 results, and those of a few rows, are float32 sums of exact products.  bfloat16 results of more rows are summed on the
 * f8 matrix instructions, which cut each eight products along the summed axis (from a multiple of eight on) towards zero at 2^-13 of the largest of them (codes below 2^-6 counted as 2^-6): a
 * sum of eight is off by up to 7 * 2^-13 of its largest product, which shows where large products cancel each other.  A row's scale times a block's is made in float32 and has to lie in its range.
 * workspace >= mi_moe_linear_f8_workspace_size, 16-byte aligned. ---- */
int mi_moe_linear_f8_workspace_size(int64_t M, int32_t N, int32_t K, size_t *bytes);
int mi_moe_linear_f8(const void *x, const void *w, const float *scales, const void *linear_bias, int64_t M,
                     int32_t N, int32_t K, int32_t transpose, int32_t dtype, void *y, void *workspace,
                     size_t workspace_bytes, void *stream);
/* The same for rows sorted by expert (mi_moe_sort_tokens): matrix e of w [n_experts, N, K] (or [n_experts, K, N]) for the rows from offsets[e] to offsets[e + 1]; rows of y
 * behind the last are zeros.  offsets ascend from 0 to at most `rows`: others reach no memory but the operands', and what rows of y hold that are in no expert's range is not
 * said.  n_experts 1..512. */
int mi_moe_grouped_linear_f8(const void *x, const void *w, const float *scales, const uint32_t *offsets,
                             int64_t rows, int32_t n_experts, int32_t N, int32_t K, int32_t transpose,
                             int32_t dtype, void *y, void *workspace, size_t workspace_bytes, void *stream);

/* ---- SwiGLU experts on such weights, from tokens to tokens on a routing of the caller's (mi_moe_select_experts, mi_moe_route, or any other):
 *   out[t] = sum over s of topk_w[t][s] * q(silu(q(x[t]) . gate_e^T) * (q(x[t]) . up_e^T)) . down_e^T,   e = topk_idx[t][s]
 * gate, up [n_experts, intermediate, hidden], down [n_experts, hidden, intermediate], scales of their blocks (f32 [n_experts, ceil(rows / 128), ceil(cols / 128)]); 16-byte
 * aligned; hidden and intermediate multiples of 16, up to 2^22; x and out [T, hidden] bfloat16 or float16; topk_w of element type w_dtype.  Products are summed as mi_moe_linear_f8's of
 * x's type (with bfloat16, a code of the rounded silu(gate) * up that lies at a border may so be its neighbour).  Experts' results are summed over the slots in float32, those of
 * bfloat16 tokens from 11 significant bits of each or more (of those below 2^-28 of the largest of 64 beside each other, fewer).  Slots that name no expert have no part in it.
 * T times hidden, this rounded up to whole runs of 128, below 2^32 - 256; T * top_k up to 2^24 - 1, and times hidden or intermediate up to 2^35.
 * workspace >= mi_moe_switch_glu_f8_workspace_size (grad: of the gradient), 16-byte aligned. ---- */
typedef struct {
  const void *gate;
  const void *up;
  const void *down;
  const float *gate_scales;
  const float *up_scales;
  const float *down_scales;
} mi_moe_f8_experts;
int mi_moe_switch_glu_f8_workspace_size(int64_t T, int32_t hidden, int32_t intermediate, int32_t n_experts,
                                        int32_t top_k, int32_t grad, size_t *bytes);
int mi_moe_switch_glu_f8(const void *x, const uint32_t *topk_idx, const void *topk_w, int32_t w_dtype,
                         const mi_moe_f8_experts *experts, int64_t T, int32_t hidden, int32_t intermediate,
                         int32_t n_experts, int32_t top_k, int32_t dtype, void *out, void *workspace,
                         size_t workspace_bytes, void *stream);
/* Its gradients with respect to x and topk_w, from dout, the gradient at out; nothing of the forward call is needed (gate and up are computed again).  Roundings to e4m3
 * pass a gradient on as it is: what is differentiated is the call above without the rounding of h = silu(gate) * up, on rounded x.  So dweights[t][s] is the product of h as float32
 * with the gradient at it, not of the codes that the forward call makes of h (a few percent of its length).  dout and the gradients at gate and up are themselves rounded to e4m3 by
 * runs of 128 ahead of their products with the weights.
 * dx [T, hidden] of element type dtype, dweights [T, top_k] of element type w_dtype (zeros in slots that name no expert). */
int mi_moe_switch_glu_f8_grad(const void *dout, const void *x, const uint32_t *topk_idx, const void *topk_w,
                              int32_t w_dtype, const mi_moe_f8_experts *experts, int64_t T, int32_t hidden,
                              int32_t intermediate, int32_t n_experts, int32_t top_k, int32_t dtype, void *dx,
                              void *dweights, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* MI_MOE_F8_H */
