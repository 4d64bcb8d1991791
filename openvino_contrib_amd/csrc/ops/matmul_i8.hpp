// What the kernels of hipops_matmul_i8 share: operands, the matrix instruction and the end of a result.
#pragma once

#include "hipops_int8.h"
#include "ops/ops_common.hpp"
#include "ops/vec8.hpp"

namespace hipops {

typedef int int4_t __attribute__((ext_vector_type(4)));
typedef int int16v_t __attribute__((ext_vector_type(16)));

struct MatmulI8Params {
    const int8_t* a;  // [m, k]
    const int8_t* b;  // [n, k]
    const float* a_scales;
    const float* b_scales;
    const void* bias;
    const void* residual;
    void* c;
    int64_t m, n, k;
    int64_t lda, ldb, ldc;
    int c_dtype;
};

// 32 rows of each operand, 32 bytes of k: lane l holds the 16 bytes from 16 (l / 32) on of row l % 32; register r of the result is row
// 8 (r / 4) + 4 (l / 32) + r % 4 of a and row l % 32 of b
__device__ __forceinline__ int16v_t mma_i8(uint4_t a, uint4_t b, int16v_t c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(int4_t, a), __builtin_bit_cast(int4_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ float finished(const MatmulI8Params& p, int sum, int64_t i, int64_t j, float b_scale) {
    float x = (float)sum * ((p.a_scales ? p.a_scales[i] : 1.0f) * b_scale);
    if (p.bias) x += load_scalar(p.bias, j, p.c_dtype);
    if (p.residual) x += load_scalar(p.residual, i * p.ldc + j, p.c_dtype);
    return x;
}

}  // namespace hipops
