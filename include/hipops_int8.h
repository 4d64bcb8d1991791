/*
 * hipops_int8 - the projections of a decoder layer in 8-bit integers, beside hipops.h, whose conventions and error string these
 * entry points share (plain C, device pointers, asynchronous on the given stream, scratch through the workspace argument,
 * nothing thrown).  Exported by libhipops.so.
 *
 * No counterpart in the reference: a quantised model reaches it as FakeQuantize nodes around floating-point MatMuls
 * (src/ops/fake_quantize.cpp, src/ops/matmul.cpp:185-227 of modules/nvidia_plugin).
 */
#ifndef HIPOPS_INT8_H_
#define HIPOPS_INT8_H_

#include "hipops.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- rows as 8-bit codes with a scale each ----------------------------------------------------
 * codes[r, i] = clamp(rint(y[r, i] * (1 / scales[r])), -127, 127), scales[r] = max_i |y[r, i]| * (1 / 127), all in fp32; a scale
 * below 1e-30 is 0, and so are its codes.  y is one of
 *   HIPOPS_QUANTIZE_PLAIN      x[r, i]
 *   HIPOPS_QUANTIZE_RMS_NORM   x[r, i] * 1/sqrt(mean_i(x[r, i]^2) + eps) * gamma[i]   (gamma [width], or NULL: ones; zeros where the root is of 0)
 *   HIPOPS_QUANTIZE_GLU        act(x[r, g + i]) * x[r, u + i], rows of x 2 * width long, as hipops_glu
 * in fp32, not rounded in between.  x_row_stride: elements between rows of x (0: packed); codes [rows, width] and scales [rows]
 * are packed.  A row that holds infinities or NaN has undefined codes and scale; other rows are not touched by it. */
#define HIPOPS_QUANTIZE_PLAIN 0
#define HIPOPS_QUANTIZE_RMS_NORM 1
#define HIPOPS_QUANTIZE_GLU 2
typedef struct hipops_quantize_desc {
    int source;      /* HIPOPS_QUANTIZE_* */
    int x_dtype;     /* HIPATTN_F32 / F16 / BF16 */
    int gamma_dtype; /* likewise */
    int glu_activation, glu_gate_first;
    float eps;
    int64_t rows, width;
    int64_t x_row_stride;
} hipops_quantize_desc;
hipattn_status hipops_quantize_rows(const hipops_quantize_desc* desc, const void* x, const void* gamma, int8_t* codes,
                                    float* scales, hipattn_stream stream);

/* ---- product of codes -------------------------------------------------------------------------
 * c[i, j] = a_scales[i] * b_scales[j] * sum_l a[i, l] * b[j, l] + bias[j] + residual[i, j]
 * a [m, k] and b [n, k] (a projection's weights as stored) are signed bytes, their rows lda and ldb bytes apart (0: packed);
 * a_scales [m] and b_scales [n] floats, NULL standing for ones; bias [n] and residual [m, n] (rows ldc elements apart) of c's type,
 * or NULL.  c is c_dtype (F32 / F16 / BF16), rows ldc elements apart (0: packed), and may be the residual.  The sum is
 * exact, in 32-bit integers, which is why k is at most 131,071 (codes of -128 included); the rest is fp32, rounded once.
 * Rows at multiples of 16 bytes (a, b, lda, ldb) take the kernels that load 16 bytes a lane; other strides and odd k a plainer one.
 * The workspace may be NULL / 0, or hold what hipops_matmul_i8_workspace_size asks for, with which k is split over workgroups
 * where m and n alone do not fill the device; the result is the same to the bit. */
typedef struct hipops_matmul_i8_desc {
    int c_dtype;
    int64_t m, n, k;
    int64_t lda, ldb, ldc;
} hipops_matmul_i8_desc;
hipattn_status hipops_matmul_i8_workspace_size(const hipops_matmul_i8_desc* desc, size_t* bytes);
hipattn_status hipops_matmul_i8(const hipops_matmul_i8_desc* desc, const int8_t* a, const float* a_scales, const int8_t* b,
                                const float* b_scales, const void* bias, const void* residual, void* c, void* workspace,
                                size_t workspace_bytes, hipattn_stream stream);

#ifdef __cplusplus
}
#endif
#endif /* HIPOPS_INT8_H_ */
