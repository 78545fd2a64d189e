/*
 * prefree_moe_kernels.h — thin extern "C" HIP layer of the expert-layer operators (libprefree_kernels.so).
 *
 * Only libprefree.so calls these, with arguments it has checked; applications use prefree_moe.h, which says what each
 * computes.  Every function launches on `stream` and returns a pf_status.
 */
#ifndef PREFREE_MOE_KERNELS_H
#define PREFREE_MOE_KERNELS_H

#include <stddef.h>
#include <stdint.h>

#include "prefree_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Workspace of the routing kernels.  With one block of PFK_MOE_ROUTE_BLOCK tokens there is none.  Else it holds the counts,
 * a row of bytes a block, each row as many whole words as hold a byte an expert; and behind them, for more than
 * PFK_MOE_ROUTE_DIRECT blocks, the sums of each PFK_MOE_ROUTE_SUPER whole blocks, a word an expert.  The library that
 * says how large it is and the one that fills it both take it from here. */
#define PFK_MOE_ROUTE_BLOCK 64
#define PFK_MOE_ROUTE_DIRECT 1024
#define PFK_MOE_ROUTE_SUPER 64
#define PFK_MOE_ROUTE_BLOCKS(tokens) (((long long)(tokens) + PFK_MOE_ROUTE_BLOCK - 1) / PFK_MOE_ROUTE_BLOCK)
#define PFK_MOE_ROUTE_ROW_WORDS(experts) (((experts) + 3) / 4)
/* words of the counts, and of the sums behind them */
#define PFK_MOE_ROUTE_COUNT_WORDS(blocks, experts) ((long long)(blocks) * PFK_MOE_ROUTE_ROW_WORDS(experts))
#define PFK_MOE_ROUTE_SUPER_WORDS(blocks, experts) \
    ((blocks) > PFK_MOE_ROUTE_DIRECT ? (long long)(blocks) / PFK_MOE_ROUTE_SUPER * (experts) : 0LL)

int pfk_moe_route(const void *logits, long long ld, int dtype, int tokens, int experts, int top_k, int normalise,
                  int *choice, float *weight, int *offsets, int *order, int *slot, int *counts, void *stream);
int pfk_moe_route_backward(const void *logits, long long ld, int dtype, int tokens, int experts, int top_k,
                           int normalise, const int *choice, const float *weight, const float *dweight, void *dlogits,
                           long long ld_d, void *stream);
int pfk_moe_combine(const void *y, long long ld_y, int dtype, int slots, const int *slot, const float *weight,
                    int tokens, int top_k, int width, void *out, long long ld_out, void *stream);
int pfk_moe_combine_backward(const void *dout, long long ld_dout, const void *y, long long ld_y, int dtype, int slots,
                             const int *slot, const float *weight, int tokens, int top_k, int width, void *dy,
                             long long ld_dy, float *dweight, void *stream);
int pfk_swiglu_backward(const void *dh, long long ld_dh, const void *pre, long long ld_pre, int dtype, int rows, int n,
                        void *dpre, long long ld_dpre, void *stream);
int pfk_mx4_quantize(const void *x, long long ld_x, int dtype, int rows, int k, void *codes, void *scales,
                     void *stream);
int pfk_mx4_dequantize(const void *codes, const void *scales, int rows, int k, int dtype, void *y, long long ld_y,
                       void *stream);

/* One grouped product.  Sizes in elements, strides in bytes. */
typedef struct pfk_moe_mm_args {
    const void *p;          /* rows operand: x or dy */
    long long ld_p;
    const void *p_scales;   /* 4-bit operands: [p_rows][k / 32] */
    int p_rows;             /* rows behind p when it is gathered */
    const void *q;          /* the weights, or x for the weights' gradient (then gathered) */
    long long ld_q;
    const void *q_scales;
    const int *rows;        /* row of each slot times row_div, or NULL */
    int row_div;
    const int *offsets;
    int experts, slots, n, k;
    int dtype, act;
    void *out;
    long long ld_out;
    int out_f32;            /* weights' gradient: 1 = fp32 results */
    void *pre;              /* pre-activations, or NULL */
    long long ld_pre;
} pfk_moe_mm_args;

int pfk_moe_mm(const pfk_moe_mm_args *a, void *stream);
int pfk_moe_mm_dx(const pfk_moe_mm_args *a, void *stream);
int pfk_moe_mm_dw(const pfk_moe_mm_args *a, void *stream);
int pfk_moe_mm_mx4(const pfk_moe_mm_args *a, void *stream);

#ifdef __cplusplus
}
#endif
#endif
