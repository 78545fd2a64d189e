/*
 * prefree_moe.h — C ABI of the expert-layer operators (libprefree.so): the sparse product of language models.
 *
 * A layer of experts multiplies each token with the weights of a few experts.  Its sparse matrix is the routing:
 * tokens x experts, top_k entries a row.  Its transpose is a CSR whose row_ptr are the experts' `offsets` and whose
 * entries are named by `order`; the blocks it multiplies with are the experts' weights.  As in prefree_c.h the
 * pointers are device memory, `stream` is a hipStream_t as void*, every function returns a pf_status and
 * pf_last_error() says more.  All calls are asynchronous on `stream`: no allocation, no synchronisation, no host copy
 * of the offsets (each workgroup finds its expert and its rows by searching them), and they may be captured into a
 * graph.  Results do not depend on the order in which workgroups run: no atomics on floating-point numbers, same bits each time.
 *
 * Value types: PF_F16 and PF_BF16 (sums in fp32, each result rounded once, to nearest even), PF_F32 where noted.
 * Leading dimensions (ld*) count elements between rows; 0 stands for the row's length.  Any alignment that the
 * element type has is accepted, less is refused (PF_ERR_ALIGN); rows that all start at multiples of 16 bytes are read
 * faster.  Sizes: up to 1024 experts, 16 experts a token, 2^30 entries (tokens * top_k), 2^24 columns; offsets pass 32 bits.
 * Products have a second limit that only costs time: 4 GiB of x or dy, or of one expert's weights.  From there on they
 * are formed as unaligned ones are (2^20 slots of 16 experts, 2048 x 2048: 1.4 to 2.3 times as long), and 4-bit ones
 * as those with few rows an expert are (32768 slots of 16 experts, 4096 -> 2048: 9 times as long).
 * No output may overlap an input.  The reference has no counterpart of any of these.
 */
#ifndef PREFREE_MOE_H
#define PREFREE_MOE_H

#include "prefree_c.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Value type of these entry points only (the SpMV entry points refuse it with PF_ERR_INVALID). */
enum { PF_BF16 = 3 };

enum pf_act {
    PF_ACT_NONE = 0,
    PF_ACT_SWIGLU = 1 /* w holds 2n rows an expert, n of the gate, then n of the rest: silu(gate) * rest */
};

#define PF_MOE_MAX_EXPERTS 1024
#define PF_MOE_MAX_TOP_K 16

/* ---- routing ------------------------------------------------------------------
 * logits [tokens][experts] (f32, f16, bf16).  Each token takes the top_k experts of its largest logits (of equal ones
 * the lowest index; a NaN counts as larger than any number, and makes its row's weights NaN).  A logit of -infinity is
 * never chosen: a row may have fewer than top_k experts, or none.
 *   choice [tokens*top_k]  the experts, best first, -1 where there is none
 *   weight [tokens*top_k]  exp(logit) / sum of exp(logits), the sum over the chosen experts (normalise 1) or over all
 *                          experts (normalise 0); 0 where there is none
 *   offsets [experts+1]    slots of expert e: offsets[e] .. offsets[e+1]
 *   order [tokens*top_k]   slot s holds entry order[s] = token*top_k + j; by expert, then by entry; -1 from
 *                          offsets[experts] on
 *   slot [tokens*top_k]    the inverse: the slot of each entry, -1 where there is none
 * workspace: pf_moe_route_workspace() bytes, 4-byte aligned (none up to 64 tokens); what it holds before and after does not matter. */
size_t pf_moe_route_workspace(int tokens, int experts);
int pf_moe_route(const void *logits, long long ld_logits, int dtype, int tokens, int experts, int top_k, int normalise,
                 int *choice, float *weight, int *offsets, int *order, int *slot, void *workspace,
                 size_t workspace_bytes, void *stream);
/* dlogits [tokens][experts] (the type of logits) from dweight [tokens*top_k], with choice and weight as
 * pf_moe_route wrote them.  Every element is written: 0 for rows without an expert and logits of -infinity. */
int pf_moe_route_backward(const void *logits, long long ld_logits, int dtype, int tokens, int experts, int top_k,
                          int normalise, const int *choice, const float *weight, const float *dweight, void *dlogits,
                          long long ld_dlogits, void *stream);

/* ---- routing by scores ----------------------------------------------------------
 * As pf_moe_route, but the choice goes by scores plus a bias that balances the experts' load, inside the best groups of experts:
 *   s = sigmoid(logit), or exp(logit) / sum of exp(logits) over all experts;  r = s + bias (f32 [experts], NULL: 0)
 *   the experts form `groups` groups of equal size, side by side; a group counts the sum of its group_best (1 or 2) largest
 *   r, as far as it has as many, and the groups_kept groups that count most are kept (of equal ones the lowest index)
 *   choice: the top_k largest r of their experts (of equal ones the lowest index), best first, -1 where there is none
 *   weight: scale * s / sum of the chosen s (normalise 1), or scale * s (normalise 0); the bias is not part of it
 * A logit of -infinity and an r of -infinity are never chosen and count in no group.  A NaN counts as larger than any number.
 * r is compared as of 64 bits (and as its logit, where there is no bias and groups count one score: scores that 64 bits
 * do not tell apart are then in the order of their logits).  experts is a multiple of groups; groups: 1 to 16; scale: a positive number.
 * To leave an expert out use a logit or a bias of -infinity: finite ones far from the others (-1e9, the type's lowest) give the same
 * choice, but up to 3.5 times as late.
 * offsets, order, slot, workspace: as of pf_moe_route. */
enum pf_score { PF_SCORE_SOFTMAX = 0, PF_SCORE_SIGMOID = 1 };
#define PF_MOE_MAX_GROUPS 16
int pf_moe_route_scores(const void *logits, long long ld_logits, int dtype, int tokens, int experts, int top_k, int score,
                        const float *bias, int groups, int groups_kept, int group_best, int normalise, float scale,
                        int *choice, float *weight, int *offsets, int *order, int *slot, void *workspace,
                        size_t workspace_bytes, void *stream);
/* dlogits [tokens][experts] (the type of logits) from dweight [tokens*top_k], with choice and weight as
 * pf_moe_route_scores wrote them; the choice itself, and so bias and groups, has no gradient.  Every element is written. */
int pf_moe_route_scores_backward(const void *logits, long long ld_logits, int dtype, int tokens, int experts, int top_k,
                                 int score, int normalise, float scale, const int *choice, const float *weight,
                                 const float *dweight, void *dlogits, long long ld_dlogits, void *stream);
/* The next bias from the experts' load: next[e] = bias[e] + rate where expert e has fewer slots than the mean of all, - rate
 * where it has more.  offsets [experts+1] as the routing wrote them; next may be bias. */
int pf_moe_balance(const int *offsets, int experts, float rate, const float *bias, float *next, void *stream);

/* out[t] = sum over j of weight[t,j] * y[slot[t,j]]: y [slots][width], out [tokens][width] (f16, bf16).  Entries whose
 * slot is outside [0, slots) are left out, and their rows not read; a token without any gets zeros.  weight NULL:
 * all 1 (the gradient of the tokens from that of their slots). */
int pf_moe_combine(const void *y, long long ld_y, int dtype, int slots, const int *slot, const float *weight, int tokens,
                   int top_k, int width, void *out, long long ld_out, void *stream);
/* dy[slot[t,j]] = weight[t,j] * dout[t] and dweight[t,j] = sum of dout[t] * y[slot[t,j]] (0 without a slot).  Rows of
 * dy that no entry names are not written. */
int pf_moe_combine_backward(const void *dout, long long ld_dout, const void *y, long long ld_y, int dtype, int slots,
                            const int *slot, const float *weight, int tokens, int top_k, int width, void *dy,
                            long long ld_dy, float *dweight, void *stream);

/* ---- products grouped by expert -------------------------------------------------
 * Slot s of expert e (offsets[e] <= s < offsets[e+1]; offsets NULL: one expert has all slots):
 *   y[s] = act(x[rows ? rows[s] / row_div : s] w[e]^T)
 * x [x_rows][k], w [experts][n or 2n][k] without gaps, y [slots][n].  With rows = order and row_div = top_k of
 * pf_moe_route the tokens are gathered on the way in.  pre (PF_ACT_SWIGLU only, may be NULL): [slots][2n], what
 * the activation was applied to, for pf_swiglu_backward.  SwiGLU is formed in
 * fp32 from the sums and then rounded: silu(g) within (8 + |g|) 2^-23 of itself and within 2^-134 at the least, also where
 * sigmoid(g) is no normal number any more.  Slots from offsets[experts] on are not written.  A row index outside [0, x_rows) gives an unspecified row (nothing outside x is read); so do offsets that decrease. */
int pf_moe_mm(const void *x, long long ld_x, int x_rows, const int *rows, int row_div, const void *w,
              const int *offsets, int experts, int slots, int n, int k, int dtype, int act, void *y, long long ld_y,
              void *pre, long long ld_pre, void *stream);
/* dx[s] = dy[s] w[e]: dy [slots][n], w [experts][n][k], dx [slots][k]. */
int pf_moe_mm_dx(const void *dy, long long ld_dy, const void *w, const int *offsets, int experts, int slots, int n,
                 int k, int dtype, void *dx, long long ld_dx, void *stream);
/* dw[e] = sum over the slots of e of dy[s]^T x[row of s]: dw [experts][n][k] without gaps, of the type dw_dtype
 * (dtype or PF_F32); zeros for an expert without slots. */
int pf_moe_mm_dw(const void *dy, long long ld_dy, const void *x, long long ld_x, int x_rows, const int *rows,
                 int row_div, const int *offsets, int experts, int slots, int n, int k, int dtype, void *dw,
                 int dw_dtype, void *stream);
/* dpre [rows][2n] from dh [rows][n] and pre [rows][2n] (f16, bf16), the activation's gradient. */
int pf_swiglu_backward(const void *dh, long long ld_dh, const void *pre, long long ld_pre, int dtype, int rows, int n,
                       void *dpre, long long ld_dpre, void *stream);

/* ---- 4-bit blocks (microscaling format MX, elements e2m1, scales e8m0) -----------
 * Blocks of 32 along a row: scale 2^(floor(log2(largest magnitude)) - 2), at least 2^-127, held as the exponent plus
 * 127 in a byte; elements x / scale rounded to the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 (ties to even, above 6 to 6),
 * sign kept.  A block that holds an infinity or a NaN has scale 255, which stands for NaN; its elements are 0.
 *   x [rows][k] (f32, f16, bf16), k a multiple of 32;
 *   codes [rows][k/2]: element 2i in the low half of byte i;  scales [rows][k/32].  No gaps; codes 16-byte aligned. */
int pf_mx4_quantize(const void *x, long long ld_x, int dtype, int rows, int k, void *codes, void *scales, void *stream);
/* What the blocks stand for, in f32 (exact), or rounded to f16 or bf16. */
int pf_mx4_dequantize(const void *codes, const void *scales, int rows, int k, int dtype, void *y, long long ld_y,
                      void *stream);
/* pf_moe_mm of 4-bit operands: x (x_codes, x_scales) [x_rows][k], w (w_codes, w_scales) [experts][n or 2n][k]; y in
 * dtype (f16, bf16).  k is a multiple of 32; products and sums as of the values that the blocks stand for, in fp32. */
int pf_moe_mm_mx4(const void *x_codes, const void *x_scales, int x_rows, const int *rows, int row_div,
                  const void *w_codes, const void *w_scales, const int *offsets, int experts, int slots, int n, int k,
                  int dtype, int act, void *y, long long ld_y, void *stream);

/* ---- 8-bit integers with a scale a row --------------------------------------------
 * A row of x: scale = largest magnitude / 127 (the largest magnitude at least 2^-100); integers from -127 to 127, the nearest
 * to 127 x / largest magnitude, ties to even.  A row that holds an infinity or a NaN has the scale NaN and zeros.
 *   x [rows][k] (f32, f16, bf16), 1 <= k <= 2^24;
 *   codes [rows][PF_I8_ROW(k)]: k signed bytes, zeros behind them, 16-byte aligned;  scales [rows], f32. */
#define PF_I8_ROW(k) (((long long)(k) + 15) / 16 * 16)
int pf_i8_quantize(const void *x, long long ld_x, int dtype, int rows, int k, void *codes, float *scales, void *stream);
/* Integer times scale, formed in f32 and rounded to dtype. */
int pf_i8_dequantize(const void *codes, const float *scales, int rows, int k, int dtype, void *y, long long ld_y, void *stream);
/* pf_moe_mm of such rows: x (x_codes, x_scales) [x_rows][k], w (w_codes, w_scales) [experts][n or 2n][k], a scale for each
 * token and each row of w; y in dtype (f16, bf16).  Sums are exact (k at most 131056); they are scaled, by the token's scale and
 * then by the row's, and the activation formed, in f32.  Codes behind a row's k elements are zeros, as pf_i8_quantize writes them; -128 is allowed. */
int pf_moe_mm_i8(const void *x_codes, const float *x_scales, int x_rows, const int *rows, int row_div, const void *w_codes,
                 const float *w_scales, const int *offsets, int experts, int slots, int n, int k, int dtype, int act, void *y,
                 long long ld_y, void *stream);

/* ---- orthogonal updates --------------------------------------------------------------
 * out = the update of each of `batch` matrices g [rows][columns] (f32, f16, bf16) made nearly orthogonal by Newton-Schulz
 * products: X = g / |g| (the root of its sum of squares), then for each of n_steps triples (a, b, c) of `steps`, which is host memory
 * and read during the call, X <- a X + (b A + c A A) X with A = X X^T (of the transpose where rows > columns).  Every singular value x
 * becomes a x + b x^3 + c x^5 in each step: with (3.4445, -4.7750, 2.0315) five times those from 0.01 of |g| on come out
 * between 0.7 and 1.2.  out [rows][columns] (f16, bf16).  Matrices follow each other, rows * ld elements apart.
 * Up to 64 rows (or columns) the result is as exact as its type.  Larger matrices: products of f16 values with sums in f32,
 * X held in two f16 pieces, of which the products take the first: within 2^-8 of the formula, in the 2-norm over all elements,
 * besides the result's rounding, in f16 too; within 2^-6 where the elements of a matrix are all of one magnitude, and so
 * round alike.  That is after up to six such steps.  Each further one may multiply it by a: in all of them what rounding puts
 * where a matrix has nothing grows as its own smallest singular values do.  Steps have to keep singular values of 1 and less
 * under 4.  A matrix of zeros gives zeros, one that holds an infinity or a NaN gives NaN; others of the batch are not touched by it.
 * Of larger matrices f16 results are rounded more finely than bf16 ones, and are no closer to the formula otherwise.
 * rows, columns: 1 to 2^20, rows * columns at most 2^29; batch at most 1024; n_steps 1 to 64.
 * workspace: pf_orthogonalize_workspace() bytes, 16-byte aligned; what it holds before and after does not matter. */
size_t pf_orthogonalize_workspace(int batch, int rows, int columns);
int pf_orthogonalize(const void *g, long long ld_g, int dtype, int batch, int rows, int columns, const float *steps,
                     int n_steps, void *out, long long ld_out, int out_dtype, void *workspace, size_t workspace_bytes,
                     void *stream);

#ifdef __cplusplus
}
#endif
#endif
