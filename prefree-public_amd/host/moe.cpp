// moe.cpp — the C ABI of the expert-layer operators (include/prefree_moe.h): argument checks, then one call of the
// thin HIP layer.  No allocation and no synchronisation.
#include "prefree_moe.h"
#include "prefree_kernels.h"
#include "prefree_moe_kernels.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <string>

#include "error.h"

namespace {

int bad(const char *what, const char *why) { return pf_internal_fail(PF_ERR_INVALID, std::string(what) + ": " + why); }

int from_kernels(int status, const char *what)
{
    return status == PF_OK ? PF_OK : pf_internal_fail(status, std::string(what) + ": " + pfk_last_error());
}

int bytes_of(int dtype) { return dtype == PF_F32 ? 4 : dtype == PF_F16 || dtype == PF_BF16 ? 2 : 0; }
bool half_type(int dtype) { return dtype == PF_F16 || dtype == PF_BF16; }

bool aligned(const void *p, int bytes) { return (uintptr_t)p % bytes == 0; }

// A leading dimension of `width` elements (0: the width itself); -1 when it is too small.
long long lead(long long ld, long long width) { return ld == 0 ? width : ld < width ? -1 : ld; }

#define PF_CHECK(cond, why)              \
    do {                                 \
        if (!(cond)) return bad(what, why); \
    } while (0)

#define PF_CHECK_ALIGN(p, bytes, why)                                                             \
    do {                                                                                          \
        if (!aligned(p, bytes)) return pf_internal_fail(PF_ERR_ALIGN, std::string(what) + ": " why); \
    } while (0)

// whether arrays of 32-bit numbers lie on words (NULL does)
template <typename... P>
bool on_words(const P *...p) { return (aligned(p, 4) && ...); }

#define PF_CHECK_WORDS(...)                                                                                              \
    do {                                                                                                                 \
        if (!on_words(__VA_ARGS__)) return pf_internal_fail(PF_ERR_ALIGN, std::string(what) + ": " #__VA_ARGS__ ": not 4-byte aligned"); \
    } while (0)

const char *routing(int tokens, int experts, int top_k)
{
    if (tokens < 0) return "negative number of tokens";
    if (experts < 1 || experts > PF_MOE_MAX_EXPERTS) return "experts: 1 to 1024";
    if (top_k < 1 || top_k > PF_MOE_MAX_TOP_K || top_k > experts) return "top_k: 1 to 16, and no more than the experts";
    if ((long long)tokens * top_k > (1 << 30)) return "tokens * top_k: at most 2^30";
    return nullptr;
}

const char *grouped(const int *offsets, int experts, int slots, int n, int k)
{
    if (experts < 1 || experts > PF_MOE_MAX_EXPERTS) return "experts: 1 to 1024";
    if (!offsets && experts != 1) return "more than one expert without offsets";
    if (slots < 0 || n < 0 || k < 0) return "negative size";
    if (n > (1 << 24) || k > (1 << 24) || slots > INT_MAX - 4096) return "size too large";
    return nullptr;
}

}  // namespace

extern "C" {

size_t pf_moe_route_workspace(int tokens, int experts)
{
    if (tokens < 1 || experts < 1) return 0;
    const long long blocks = PFK_MOE_ROUTE_BLOCKS(tokens);
    const long long words = PFK_MOE_ROUTE_COUNT_WORDS(blocks, experts) + PFK_MOE_ROUTE_SUPER_WORDS(blocks, experts);
    // A word for each expert of a block holds both, but for one expert above 1024 blocks.  It stays the least that is
    // asked for, so that a caller's reservation does not depend on how counts are packed.
    return 4 * (size_t)std::max(words, blocks * experts);
}

int pf_moe_route(const void *logits, long long ld_logits, int dtype, int tokens, int experts, int top_k, int normalise,
                 int *choice, float *weight, int *offsets, int *order, int *slot, void *workspace, size_t workspace_bytes,
                 void *stream)
{
    const char *what = "pf_moe_route", *why = routing(tokens, experts, top_k);
    PF_CHECK(!why, why);
    PF_CHECK(bytes_of(dtype), "logits are f32, f16 or bf16");
    PF_CHECK(offsets, "NULL pointer");
    PF_CHECK(tokens == 0 || (logits && choice && weight && order && slot), "NULL pointer");
    const long long ld = lead(ld_logits, experts);
    PF_CHECK(ld >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(logits, bytes_of(dtype), "logits not aligned to their elements");
    PF_CHECK_WORDS(choice, weight, offsets, order, slot);
    const size_t need = tokens > PFK_MOE_ROUTE_BLOCK ? pf_moe_route_workspace(tokens, experts) : 0;
    PF_CHECK(need == 0 || (workspace && workspace_bytes >= need), "workspace smaller than pf_moe_route_workspace()");
    PF_CHECK_ALIGN(workspace, 4, "workspace not 4-byte aligned");
    return from_kernels(pfk_moe_route(logits, ld, dtype, tokens, experts, top_k, normalise != 0, choice, weight, offsets, order,
                                      slot, (int *)workspace, stream), what);
}

int pf_moe_route_backward(const void *logits, long long ld_logits, int dtype, int tokens, int experts, int top_k,
                          int normalise, const int *choice, const float *weight, const float *dweight, void *dlogits,
                          long long ld_dlogits, void *stream)
{
    const char *what = "pf_moe_route_backward", *why = routing(tokens, experts, top_k);
    PF_CHECK(!why, why);
    PF_CHECK(bytes_of(dtype), "logits are f32, f16 or bf16");
    if (tokens == 0) return PF_OK;
    PF_CHECK(logits && choice && weight && dweight && dlogits, "NULL pointer");
    const long long ld = lead(ld_logits, experts), ld_d = lead(ld_dlogits, experts);
    PF_CHECK(ld >= 0 && ld_d >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(logits, bytes_of(dtype), "logits not aligned to their elements");
    PF_CHECK_ALIGN(dlogits, bytes_of(dtype), "dlogits not aligned to their elements");
    PF_CHECK_WORDS(choice, weight, dweight);
    return from_kernels(pfk_moe_route_backward(logits, ld, dtype, tokens, experts, top_k, normalise != 0, choice, weight,
                                               dweight, dlogits, ld_d, stream), what);
}

int pf_moe_route_scores(const void *logits, long long ld_logits, int dtype, int tokens, int experts, int top_k, int score,
                        const float *bias, int groups, int groups_kept, int group_best, int normalise, float scale, int *choice,
                        float *weight, int *offsets, int *order, int *slot, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *what = "pf_moe_route_scores", *why = routing(tokens, experts, top_k);
    PF_CHECK(!why, why);
    PF_CHECK(bytes_of(dtype), "logits are f32, f16 or bf16");
    PF_CHECK(score == PF_SCORE_SOFTMAX || score == PF_SCORE_SIGMOID, "unknown score");
    PF_CHECK(groups >= 1 && groups <= PF_MOE_MAX_GROUPS && experts % groups == 0, "groups: 1 to 16, of equal size");
    PF_CHECK(groups_kept >= 1 && groups_kept <= groups, "groups_kept: 1 to groups");
    PF_CHECK(group_best == 1 || group_best == 2, "group_best: 1 or 2");
    PF_CHECK(scale > 0 && std::isfinite(scale), "scale: a positive number");
    PF_CHECK(offsets, "NULL pointer");
    PF_CHECK(tokens == 0 || (logits && choice && weight && order && slot), "NULL pointer");
    const long long ld = lead(ld_logits, experts);
    PF_CHECK(ld >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(logits, bytes_of(dtype), "logits not aligned to their elements");
    PF_CHECK_WORDS(choice, weight, offsets, order, slot, bias);
    const size_t need = tokens > PFK_MOE_ROUTE_BLOCK ? pf_moe_route_workspace(tokens, experts) : 0;
    PF_CHECK(need == 0 || (workspace && workspace_bytes >= need), "workspace smaller than pf_moe_route_workspace()");
    PF_CHECK_ALIGN(workspace, 4, "workspace not 4-byte aligned");
    return from_kernels(pfk_moe_route_scores(logits, ld, dtype, tokens, experts, top_k, score, bias, groups, groups_kept, group_best,
                                             normalise != 0, scale, choice, weight, offsets, order, slot, (int *)workspace, stream), what);
}

int pf_moe_route_scores_backward(const void *logits, long long ld_logits, int dtype, int tokens, int experts, int top_k, int score,
                                 int normalise, float scale, const int *choice, const float *weight, const float *dweight,
                                 void *dlogits, long long ld_dlogits, void *stream)
{
    const char *what = "pf_moe_route_scores_backward", *why = routing(tokens, experts, top_k);
    PF_CHECK(!why, why);
    PF_CHECK(bytes_of(dtype), "logits are f32, f16 or bf16");
    PF_CHECK(score == PF_SCORE_SOFTMAX || score == PF_SCORE_SIGMOID, "unknown score");
    PF_CHECK(scale > 0 && std::isfinite(scale), "scale: a positive number");
    if (tokens == 0) return PF_OK;
    PF_CHECK(logits && choice && weight && dweight && dlogits, "NULL pointer");
    const long long ld = lead(ld_logits, experts), ld_d = lead(ld_dlogits, experts);
    PF_CHECK(ld >= 0 && ld_d >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(logits, bytes_of(dtype), "logits not aligned to their elements");
    PF_CHECK_ALIGN(dlogits, bytes_of(dtype), "dlogits not aligned to their elements");
    PF_CHECK_WORDS(choice, weight, dweight);
    return from_kernels(pfk_moe_route_scores_backward(logits, ld, dtype, tokens, experts, top_k, score, normalise != 0, scale, choice,
                                                      weight, dweight, dlogits, ld_d, stream), what);
}

int pf_moe_balance(const int *offsets, int experts, float rate, const float *bias, float *next, void *stream)
{
    const char *what = "pf_moe_balance";
    PF_CHECK(experts >= 1 && experts <= PF_MOE_MAX_EXPERTS, "experts: 1 to 1024");
    PF_CHECK(offsets && bias && next, "NULL pointer");
    PF_CHECK_WORDS(offsets, bias, next);
    return from_kernels(pfk_moe_balance(offsets, experts, rate, bias, next, stream), what);
}

int pf_moe_combine(const void *y, long long ld_y, int dtype, int slots, const int *slot, const float *weight, int tokens,
                   int top_k, int width, void *out, long long ld_out, void *stream)
{
    const char *what = "pf_moe_combine", *why = routing(tokens, PF_MOE_MAX_EXPERTS, top_k);
    PF_CHECK(!why, why);
    PF_CHECK(half_type(dtype), "values are f16 or bf16");
    PF_CHECK(slots >= 0 && width >= 0 && width <= (1 << 24), "negative or too large size");
    if (tokens == 0 || width == 0) return PF_OK;
    PF_CHECK((y || slots == 0) && slot && out, "NULL pointer");
    const long long ly = lead(ld_y, width), lo = lead(ld_out, width);
    PF_CHECK(ly >= 0 && lo >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(y, 2, "y not aligned to its elements");
    PF_CHECK_ALIGN(out, 2, "out not aligned to its elements");
    PF_CHECK_WORDS(slot, weight);
    return from_kernels(pfk_moe_combine(y, ly, dtype, slots, slot, weight, tokens, top_k, width, out, lo, stream), what);
}

int pf_moe_combine_backward(const void *dout, long long ld_dout, const void *y, long long ld_y, int dtype, int slots,
                            const int *slot, const float *weight, int tokens, int top_k, int width, void *dy,
                            long long ld_dy, float *dweight, void *stream)
{
    const char *what = "pf_moe_combine_backward", *why = routing(tokens, PF_MOE_MAX_EXPERTS, top_k);
    PF_CHECK(!why, why);
    PF_CHECK(half_type(dtype), "values are f16 or bf16");
    PF_CHECK(slots >= 0 && width >= 0 && width <= (1 << 24), "negative or too large size");
    if (tokens == 0) return PF_OK;
    PF_CHECK((dout || width == 0) && slot && dweight && ((y && dy) || slots == 0 || width == 0), "NULL pointer");
    const long long lo = lead(ld_dout, width), ly = lead(ld_y, width), ld = lead(ld_dy, width);
    PF_CHECK(lo >= 0 && ly >= 0 && ld >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(dout, 2, "dout not aligned to its elements");
    PF_CHECK_ALIGN(y, 2, "y not aligned to its elements");
    PF_CHECK_ALIGN(dy, 2, "dy not aligned to its elements");
    PF_CHECK_WORDS(slot, weight, dweight);
    return from_kernels(pfk_moe_combine_backward(dout, lo, y, ly, dtype, slots, slot, weight, tokens, top_k, width, dy, ld,
                                                 dweight, stream), what);
}

int pf_moe_mm(const void *x, long long ld_x, int x_rows, const int *rows, int row_div, const void *w, const int *offsets,
              int experts, int slots, int n, int k, int dtype, int act, void *y, long long ld_y, void *pre, long long ld_pre,
              void *stream)
{
    const char *what = "pf_moe_mm", *why = grouped(offsets, experts, slots, n, k);
    PF_CHECK(!why, why);
    PF_CHECK(half_type(dtype), "values are f16 or bf16");
    PF_CHECK(act == PF_ACT_NONE || act == PF_ACT_SWIGLU, "unknown activation");
    PF_CHECK(!pre || act == PF_ACT_SWIGLU, "pre-activations are those of PF_ACT_SWIGLU");
    PF_CHECK(!rows || row_div >= 1, "row_div: at least 1");
    PF_CHECK(x_rows >= 0 && (slots == 0 || x_rows >= (rows ? 1 : slots)), "x has too few rows");
    if (slots == 0 || n == 0) return PF_OK;
    PF_CHECK(y && (k == 0 || (x && w)), "NULL pointer");
    const long long lx = lead(ld_x, k), ly = lead(ld_y, n), lp = lead(ld_pre, 2LL * n);
    PF_CHECK(lx >= 0 && ly >= 0 && lp >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(x, 2, "x not aligned to its elements");
    PF_CHECK_ALIGN(w, 2, "w not aligned to its elements");
    PF_CHECK_ALIGN(y, 2, "y not aligned to its elements");
    PF_CHECK_ALIGN(pre, 2, "pre not aligned to its elements");
    PF_CHECK_WORDS(rows, offsets);
    pfk_moe_mm_args a = {};
    a.p = x; a.ld_p = 2 * lx; a.p_rows = x_rows; a.rows = rows; a.row_div = row_div;
    a.q = w; a.ld_q = 2LL * k; a.offsets = offsets; a.experts = experts; a.slots = slots; a.n = n; a.k = k;
    a.dtype = dtype; a.act = act; a.out = y; a.ld_out = 2 * ly; a.pre = pre; a.ld_pre = 2 * lp;
    return from_kernels(pfk_moe_mm(&a, stream), what);
}

int pf_moe_mm_dx(const void *dy, long long ld_dy, const void *w, const int *offsets, int experts, int slots, int n, int k,
                 int dtype, void *dx, long long ld_dx, void *stream)
{
    const char *what = "pf_moe_mm_dx", *why = grouped(offsets, experts, slots, n, k);
    PF_CHECK(!why, why);
    PF_CHECK(half_type(dtype), "values are f16 or bf16");
    if (slots == 0 || k == 0) return PF_OK;
    PF_CHECK(dx && (n == 0 || (dy && w)), "NULL pointer");
    const long long ly = lead(ld_dy, n), lx = lead(ld_dx, k);
    PF_CHECK(lx >= 0 && ly >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(dy, 2, "dy not aligned to its elements");
    PF_CHECK_ALIGN(w, 2, "w not aligned to its elements");
    PF_CHECK_ALIGN(dx, 2, "dx not aligned to its elements");
    PF_CHECK_WORDS(offsets);
    pfk_moe_mm_args a = {};
    a.p = dy; a.ld_p = 2 * ly; a.p_rows = slots; a.q = w; a.ld_q = 2LL * k;
    a.offsets = offsets; a.experts = experts; a.slots = slots; a.n = n; a.k = k;
    a.dtype = dtype; a.out = dx; a.ld_out = 2 * lx;
    return from_kernels(pfk_moe_mm_dx(&a, stream), what);
}

int pf_moe_mm_dw(const void *dy, long long ld_dy, const void *x, long long ld_x, int x_rows, const int *rows, int row_div,
                 const int *offsets, int experts, int slots, int n, int k, int dtype, void *dw, int dw_dtype, void *stream)
{
    const char *what = "pf_moe_mm_dw", *why = grouped(offsets, experts, slots, n, k);
    PF_CHECK(!why, why);
    PF_CHECK(half_type(dtype), "values are f16 or bf16");
    PF_CHECK(dw_dtype == dtype || dw_dtype == PF_F32, "dw is of the values' type or f32");
    PF_CHECK(!rows || row_div >= 1, "row_div: at least 1");
    PF_CHECK(x_rows >= 0 && (slots == 0 || x_rows >= (rows ? 1 : slots)), "x has too few rows");
    if (n == 0 || k == 0) return PF_OK;
    PF_CHECK(dw && (slots == 0 || (dy && x)), "NULL pointer");
    const long long ly = lead(ld_dy, n), lx = lead(ld_x, k);
    PF_CHECK(lx >= 0 && ly >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(dy, 2, "dy not aligned to its elements");
    PF_CHECK_ALIGN(x, 2, "x not aligned to its elements");
    PF_CHECK_ALIGN(dw, bytes_of(dw_dtype), "dw not aligned to its elements");
    PF_CHECK_WORDS(rows, offsets);
    pfk_moe_mm_args a = {};
    a.p = dy; a.ld_p = 2 * ly; a.p_rows = x_rows; a.q = x; a.ld_q = 2 * lx; a.rows = rows; a.row_div = row_div;
    a.offsets = offsets; a.experts = experts; a.slots = slots; a.n = n; a.k = k;
    a.dtype = dtype; a.out = dw; a.ld_out = (long long)bytes_of(dw_dtype) * k; a.out_f32 = dw_dtype == PF_F32;
    return from_kernels(pfk_moe_mm_dw(&a, stream), what);
}

int pf_swiglu_backward(const void *dh, long long ld_dh, const void *pre, long long ld_pre, int dtype, int rows, int n,
                       void *dpre, long long ld_dpre, void *stream)
{
    const char *what = "pf_swiglu_backward";
    PF_CHECK(half_type(dtype), "values are f16 or bf16");
    PF_CHECK(rows >= 0 && n >= 0 && n <= (1 << 24), "negative or too large size");
    if (rows == 0 || n == 0) return PF_OK;
    PF_CHECK(dh && pre && dpre, "NULL pointer");
    const long long lh = lead(ld_dh, n), lp = lead(ld_pre, 2LL * n), ld = lead(ld_dpre, 2LL * n);
    PF_CHECK(lh >= 0 && lp >= 0 && ld >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(dh, 2, "dh not aligned to its elements");
    PF_CHECK_ALIGN(pre, 2, "pre not aligned to its elements");
    PF_CHECK_ALIGN(dpre, 2, "dpre not aligned to its elements");
    return from_kernels(pfk_swiglu_backward(dh, lh, pre, lp, dtype, rows, n, dpre, ld, stream), what);
}

int pf_mx4_quantize(const void *x, long long ld_x, int dtype, int rows, int k, void *codes, void *scales, void *stream)
{
    const char *what = "pf_mx4_quantize";
    PF_CHECK(bytes_of(dtype), "values are f32, f16 or bf16");
    PF_CHECK(rows >= 0 && k >= 0 && k <= (1 << 24), "negative or too large size");
    PF_CHECK(k % 32 == 0, "k is a multiple of 32");
    if (rows == 0 || k == 0) return PF_OK;
    PF_CHECK(x && codes && scales, "NULL pointer");
    const long long lx = lead(ld_x, k);
    PF_CHECK(lx >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(x, bytes_of(dtype), "x not aligned to its elements");
    PF_CHECK_ALIGN(codes, 16, "codes not 16-byte aligned");
    return from_kernels(pfk_mx4_quantize(x, lx, dtype, rows, k, codes, scales, stream), what);
}

int pf_mx4_dequantize(const void *codes, const void *scales, int rows, int k, int dtype, void *y, long long ld_y, void *stream)
{
    const char *what = "pf_mx4_dequantize";
    PF_CHECK(bytes_of(dtype), "values are f32, f16 or bf16");
    PF_CHECK(rows >= 0 && k >= 0 && k <= (1 << 24), "negative or too large size");
    PF_CHECK(k % 32 == 0, "k is a multiple of 32");
    if (rows == 0 || k == 0) return PF_OK;
    PF_CHECK(codes && scales && y, "NULL pointer");
    const long long ly = lead(ld_y, k);
    PF_CHECK(ly >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(y, bytes_of(dtype), "y not aligned to its elements");
    PF_CHECK_ALIGN(codes, 16, "codes not 16-byte aligned");
    return from_kernels(pfk_mx4_dequantize(codes, scales, rows, k, dtype, y, ly, stream), what);
}

int pf_moe_mm_mx4(const void *x_codes, const void *x_scales, int x_rows, const int *rows, int row_div, const void *w_codes,
                  const void *w_scales, const int *offsets, int experts, int slots, int n, int k, int dtype, int act, void *y,
                  long long ld_y, void *stream)
{
    const char *what = "pf_moe_mm_mx4", *why = grouped(offsets, experts, slots, n, k);
    PF_CHECK(!why, why);
    PF_CHECK(half_type(dtype), "results are f16 or bf16");
    PF_CHECK(act == PF_ACT_NONE || act == PF_ACT_SWIGLU, "unknown activation");
    PF_CHECK(k % 32 == 0, "k is a multiple of 32");
    PF_CHECK(!rows || row_div >= 1, "row_div: at least 1");
    PF_CHECK(x_rows >= 0 && (slots == 0 || x_rows >= (rows ? 1 : slots)), "x has too few rows");
    if (slots == 0 || n == 0) return PF_OK;
    PF_CHECK(y && (k == 0 || (x_codes && x_scales && w_codes && w_scales)), "NULL pointer");
    const long long ly = lead(ld_y, n);
    PF_CHECK(ly >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(x_codes, 16, "codes not 16-byte aligned");
    PF_CHECK_ALIGN(w_codes, 16, "codes not 16-byte aligned");
    PF_CHECK_ALIGN(y, 2, "y not aligned to its elements");
    PF_CHECK_WORDS(rows, offsets);
    pfk_moe_mm_args a = {};
    a.p = x_codes; a.ld_p = k / 2; a.p_scales = x_scales; a.p_rows = x_rows; a.rows = rows; a.row_div = row_div;
    a.q = w_codes; a.ld_q = k / 2; a.q_scales = w_scales; a.offsets = offsets; a.experts = experts; a.slots = slots;
    a.n = n; a.k = k; a.dtype = dtype; a.act = act; a.out = y; a.ld_out = 2 * ly;
    return from_kernels(pfk_moe_mm_mx4(&a, stream), what);
}

int pf_i8_quantize(const void *x, long long ld_x, int dtype, int rows, int k, void *codes, float *scales, void *stream)
{
    const char *what = "pf_i8_quantize";
    PF_CHECK(bytes_of(dtype), "values are f32, f16 or bf16");
    PF_CHECK(rows >= 0 && k >= 1 && k <= (1 << 24), "negative, zero or too large size");
    if (rows == 0) return PF_OK;
    PF_CHECK(x && codes && scales, "NULL pointer");
    const long long lx = lead(ld_x, k);
    PF_CHECK(lx >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(x, bytes_of(dtype), "x not aligned to its elements");
    PF_CHECK_ALIGN(codes, 16, "codes not 16-byte aligned");
    PF_CHECK_WORDS(scales);
    return from_kernels(pfk_i8_quantize(x, lx, dtype, rows, k, codes, scales, stream), what);
}

int pf_i8_dequantize(const void *codes, const float *scales, int rows, int k, int dtype, void *y, long long ld_y, void *stream)
{
    const char *what = "pf_i8_dequantize";
    PF_CHECK(bytes_of(dtype), "values are f32, f16 or bf16");
    PF_CHECK(rows >= 0 && k >= 1 && k <= (1 << 24), "negative, zero or too large size");
    if (rows == 0) return PF_OK;
    PF_CHECK(codes && scales && y, "NULL pointer");
    const long long ly = lead(ld_y, k);
    PF_CHECK(ly >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(y, bytes_of(dtype), "y not aligned to its elements");
    PF_CHECK_ALIGN(codes, 16, "codes not 16-byte aligned");
    PF_CHECK_WORDS(scales);
    return from_kernels(pfk_i8_dequantize(codes, scales, rows, k, dtype, y, ly, stream), what);
}

int pf_moe_mm_i8(const void *x_codes, const float *x_scales, int x_rows, const int *rows, int row_div, const void *w_codes,
                 const float *w_scales, const int *offsets, int experts, int slots, int n, int k, int dtype, int act, void *y,
                 long long ld_y, void *stream)
{
    const char *what = "pf_moe_mm_i8", *why = grouped(offsets, experts, slots, n, k);
    PF_CHECK(!why, why);
    PF_CHECK(half_type(dtype), "results are f16 or bf16");
    PF_CHECK(act == PF_ACT_NONE || act == PF_ACT_SWIGLU, "unknown activation");
    PF_CHECK(k <= 131056, "k: at most 131056, so that sums of products hold in 32 bits");
    PF_CHECK(!rows || row_div >= 1, "row_div: at least 1");
    PF_CHECK(x_rows >= 0 && (slots == 0 || x_rows >= (rows ? 1 : slots)), "x has too few rows");
    if (slots == 0 || n == 0) return PF_OK;
    PF_CHECK(y && x_scales && w_scales && (k == 0 || (x_codes && w_codes)), "NULL pointer");
    const long long ly = lead(ld_y, n);
    PF_CHECK(ly >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(x_codes, 16, "codes not 16-byte aligned");
    PF_CHECK_ALIGN(w_codes, 16, "codes not 16-byte aligned");
    PF_CHECK_ALIGN(y, 2, "y not aligned to its elements");
    PF_CHECK_WORDS(rows, offsets, x_scales, w_scales);
    pfk_moe_mm_args a = {};
    a.p = x_codes; a.ld_p = PF_I8_ROW(k); a.p_scales = x_scales; a.p_rows = x_rows; a.rows = rows; a.row_div = row_div;
    a.q = w_codes; a.ld_q = PF_I8_ROW(k); a.q_scales = w_scales; a.offsets = offsets; a.experts = experts; a.slots = slots;
    a.n = n; a.k = k; a.dtype = dtype; a.act = act; a.out = y; a.ld_out = 2 * ly;
    return from_kernels(pfk_moe_mm_i8(&a, stream), what);
}

size_t pf_orthogonalize_workspace(int batch, int rows, int columns)
{
    if (batch < 1 || rows < 1 || columns < 1) return 0;
    const size_t m = PFK_ORTH_SIDE((size_t)std::min(rows, columns)), n = PFK_ORTH_SIDE((size_t)std::max(rows, columns));
    if (m <= PFK_ORTH_NARROW) {
        const long long longer = std::max(rows, columns);
        const size_t shares = PFK_ORTH_SHARES(batch, longer), side = PFK_ORTH_NARROW;
        return batch * (shares * (4 * side * 32 * PFK_ORTH_BLOCKS(batch, longer) + 8 * side * side) + 8 * PFK_ORTH_PARTS);
    }
    return batch * (m * (8 * n + 4 * m) + 8 * PFK_ORTH_PARTS);
}

int pf_orthogonalize(const void *g, long long ld_g, int dtype, int batch, int rows, int columns, const float *steps, int n_steps, void *out,
                     long long ld_out, int out_dtype, void *workspace, size_t workspace_bytes, void *stream)
{
    const char *what = "pf_orthogonalize";
    PF_CHECK(bytes_of(dtype), "matrices are f32, f16 or bf16");
    PF_CHECK(half_type(out_dtype), "results are f16 or bf16");
    PF_CHECK(batch >= 0 && batch <= PF_MOE_MAX_EXPERTS, "batch: at most 1024");
    PF_CHECK(rows >= 0 && columns >= 0 && rows <= (1 << 20) && columns <= (1 << 20) && (long long)rows * columns <= (1 << 29),
             "negative or too large size");
    PF_CHECK(n_steps >= 1 && n_steps <= 64 && steps, "steps: 1 to 64 triples");
    if (batch == 0 || rows == 0 || columns == 0) return PF_OK;
    PF_CHECK(g && out, "NULL pointer");
    const long long lg = lead(ld_g, columns), lo = lead(ld_out, columns);
    PF_CHECK(lg >= 0 && lo >= 0, "leading dimension under the row's length");
    PF_CHECK_ALIGN(g, bytes_of(dtype), "g not aligned to its elements");
    PF_CHECK_ALIGN(out, 2, "out not aligned to its elements");
    PF_CHECK(workspace && workspace_bytes >= pf_orthogonalize_workspace(batch, rows, columns), "workspace smaller than pf_orthogonalize_workspace()");
    PF_CHECK_ALIGN(workspace, 16, "workspace not 16-byte aligned");
    return from_kernels(pfk_orthogonalize(g, lg, dtype, batch, rows, columns, steps, n_steps, out, lo, out_dtype, workspace, stream), what);
}

}  // extern "C"
