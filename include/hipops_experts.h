/*
 * hipops_experts - an MLP of experts: the router's choice, the products of each expert's rows in 8-bit floating point, and the sum
 * over a token's experts.  Beside hipops.h, whose conventions and error string these entry points share; exported by libhipops.so.
 * experts.py of the Python package puts them together.
 *
 * A token's place in the lists: the pair (token t, choice j) has number t * top_k + j; `order` holds the pairs' numbers sorted by expert
 * (in rising order within one), `begins[e]` where expert e's begin, and `slots` for each pair its place in `order`.
 *
 * No counterpart in the reference: a model of this kind reaches it as TopK, ScatterElementsUpdate, NonZero and a MatMul an expert
 * (src/ops/topk.cpp, src/ops/scatter_nd_update.cpp, src/ops/matmul.cpp:185-227 of modules/nvidia_plugin).
 */
#ifndef HIPOPS_EXPERTS_H_
#define HIPOPS_EXPERTS_H_

#include "hipops_fp8.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- routing ------------------------------------------------------------------------------------
 * logits [tokens, experts] (rows logits_row_stride elements apart, 0: packed).
 *   score(t, e)  = softmax over e, or sigmoid, of logits[t, e]
 *   choice(t, e) = score(t, e) + bias[e]         (bias [experts] fp32, or NULL)
 * groups > 1: the experts form that many groups of neighbours; the kept_groups with the largest sum of their group_top (1 or 2) best
 * choices stay.  The top_k experts with the largest choice among those are taken, largest first; ties, also between groups, go to the
 * lowest index.  Scores, choices and their sums are computed and compared in 64 bits, so that the order does not hang on roundings of
 * 32-bit exponentials; for a softmax without a bias, and with the best choice alone for a group, logits are compared, whose order the scores
 * have (those whose exponential is 0 in 64 bits are alike).
 *   indices[t, j] = the expert, weights[t, j] = its score (without the bias), divided by the sum of the token's top_k scores where
 *   `renormalise` is set, times `scale`; 0 where that sum is 0.
 * A NaN logit counts as minus infinity, an infinite one as the largest finite; a row of logits that are all minus infinity has scores 0.
 * A NaN choice counts as minus infinity; choices of minus infinity are taken, in the order of their index, where nothing else is left, but never
 * from a group that was not kept.
 * begins [experts + 1], order [tokens * top_k], slots [tokens, top_k]: the lists above, or NULL all three.
 * experts <= 1024, top_k <= 64, groups <= 64 and a divisor of experts; lists of 2^26 tokens at most (their cost grows with the square of the
 * tokens: of 2^20 they are a third of the call's 2.5 ms, of 2^24 most of 246).  The workspace holds what hipops_route_experts_workspace_size asks
 * for; without lists it is not looked at. */
#define HIPOPS_ROUTE_SOFTMAX 0
#define HIPOPS_ROUTE_SIGMOID 1
typedef struct hipops_route_desc {
    int logits_dtype; /* HIPATTN_F32 / F16 / BF16 */
    int score;        /* HIPOPS_ROUTE_* */
    int renormalise;
    int experts, top_k;
    int groups, kept_groups, group_top; /* groups 0 or 1: none, and the other two are not looked at */
    float scale;
    int64_t tokens;
    int64_t logits_row_stride;
} hipops_route_desc;
hipattn_status hipops_route_experts_workspace_size(const hipops_route_desc* desc, size_t* bytes);
hipattn_status hipops_route_experts(const hipops_route_desc* desc, const void* logits, const float* bias, int32_t* indices, float* weights,
                                    int32_t* begins, int32_t* order, int32_t* slots, void* workspace, size_t workspace_bytes,
                                    hipattn_stream stream);

/* ---- the experts' products ---------------------------------------------------------------------------
 * For each expert e and each place p in begins[e] .. begins[e + 1] - 1:
 *   c[p, j] = the product of hipops_matmul_fp8 (without bias and residual) of row r of a with row j of b[e],
 *   r = order[p] / order_divisor, or p where order is NULL (a_rows is at least rows then).
 * a [a_rows, k], rows lda bytes apart, with scales as there (strides both 0: 1 and a_rows); b [experts, n, k] and b_scales
 * [experts, ceil(n / 128), ceil(k / 128)] packed.  begins lies on the device; the call looks at `rows` places at most, and rows of c
 * ahead of begins[0] and behind begins[experts] stay as they are, their scales too.  An entry of begins outside [0, rows] or smaller than
 * the one before it, or one of order that names no row of a, gives undefined results in the places concerned; nothing outside the arrays is
 * read or written.
 * c: [rows, n] of F32 / F16 / BF16, packed; where `gated` is set, [rows, n / 2]: the GLU of the halves of that row (glu_activation,
 * glu_gate_first as hipops_glu), in fp32 and rounded once.  c_dtype HIPOPS_F8_E4M3 (gated alone): that GLU as codes [rows, n / 2] with
 * c_scales [ceil(n / 2 / 128), rows], as hipops_quantize_fp8 leaves them: the rows of the next product.  c_scales is not looked at otherwise.
 * F32 results are sums of exact products; those of 16 bits, and the fp32 values that become codes, come from the 8-bit matrix instruction and
 * are about 1.4e-5 off in the 2-norm on normal operands (hipops_fp8.h), ahead of a code's rounding of 2^-4 of the value at most.
 * The workspace holds what hipops_matmul_fp8_experts_workspace_size asks for.  The same call gives the same bits every time. */
typedef struct hipops_matmul_fp8_experts_desc {
    int c_dtype;
    int gated, glu_activation, glu_gate_first;
    int order_divisor; /* >= 1; top_k where order is the router's and a holds tokens */
    int experts;
    int64_t rows, n, k;
    int64_t a_rows;
    int64_t lda;
    int64_t a_scale_row_stride, a_scale_block_stride;
} hipops_matmul_fp8_experts_desc;
hipattn_status hipops_matmul_fp8_experts_workspace_size(const hipops_matmul_fp8_experts_desc* desc, size_t* bytes);
hipattn_status hipops_matmul_fp8_experts(const hipops_matmul_fp8_experts_desc* desc, const uint8_t* a, const float* a_scales, const uint8_t* b,
                                         const float* b_scales, const int32_t* begins, const int32_t* order, void* c, float* c_scales,
                                         void* workspace, size_t workspace_bytes, hipattn_stream stream);

/* ---- the sum over a token's experts ----------------------------------------------------------------------
 * out[t, i] = residual[t, i] + sum over j of weights[t, j] * y[slots[t, j], i], fp32, rounded once to out_dtype.
 * y [rows, n] of y_dtype, weights [tokens, top_k] fp32, slots [tokens, top_k]; residual [tokens, n] of out_dtype, or NULL; out may be
 * the residual.  All packed.  A slot outside [0, rows) adds nothing (an expert that another device holds).  Terms are added in the order of j. */
typedef struct hipops_combine_desc {
    int y_dtype, out_dtype; /* HIPATTN_F32 / F16 / BF16 */
    int top_k;
    int64_t tokens, rows, n;
} hipops_combine_desc;
hipattn_status hipops_combine_experts(const hipops_combine_desc* desc, const void* y, const float* weights, const int32_t* slots,
                                      const void* residual, void* out, hipattn_stream stream);

#ifdef __cplusplus
}
#endif
#endif /* HIPOPS_EXPERTS_H_ */
