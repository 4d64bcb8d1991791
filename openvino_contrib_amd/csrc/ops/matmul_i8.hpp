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

// 16 rows of each operand, 64 bytes of k: lane l holds the 16 bytes from 16 (l / 16) on of row l % 16; register r of the result is row
// 4 (l / 16) + r of a and row l % 16 of b
__device__ __forceinline__ int4_t mma_i8_16(uint4_t a, uint4_t b, int4_t c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(int4_t, a), __builtin_bit_cast(int4_t, b), c, 0, 0, 0);
}

// 16 bytes of a row from `at` on, zeros where it has ended; at any address.
__device__ __forceinline__ uint4_t load_codes16(const int8_t* row, int64_t at, int64_t k) {
    uint4_t w = {0u, 0u, 0u, 0u};
    if (at + 16 <= k) {
        __builtin_memcpy(&w, row + at, 16);
    } else if (at < k) {  // (the row's last piece)
        const int rest = (int)(k - at);
        unsigned __int128 v = 0;
        if (k >= 16) {
            __builtin_memcpy(&v, row + k - 16, 16);
            v >>= 8 * (16 - rest);
        } else {
            for (int e = 0; e < rest; e++) v |= (unsigned __int128)(uint8_t)row[at + e] << (8 * e);
        }
        __builtin_memcpy(&w, &v, 16);
    }
    return w;
}

__device__ __forceinline__ float finished(const MatmulI8Params& p, int sum, int64_t i, int64_t j, float b_scale) {
    float x = fmaf((float)sum, (p.a_scales ? p.a_scales[i] : 1.0f) * b_scale, p.bias ? load_scalar(p.bias, j, p.c_dtype) : 0.0f);
    if (p.residual) x += load_scalar(p.residual, i * p.ldc + j, p.c_dtype);
    return x;
}

// `columns` (1 to 8) results of a row from element `to` on, with the residual if there is one.  (Rows may begin anywhere: copies of
// eight elements are whatever loads and stores the hardware has for that.)
__device__ __forceinline__ void store_columns(const MatmulI8Params& p, int64_t to, int columns, float (&y)[8]) {
    if (columns < 8) {
        for (int e = 0; e < columns; e++) {
            const float r = p.residual != nullptr ? load_scalar(p.residual, to + e, p.c_dtype) : 0.0f;
            float v = 0.0f;
#pragma unroll
            for (int u = 0; u < 8; u++) v = u == e ? y[u] : v;
            store_scalar(p.c, to + e, p.c_dtype, v + r);
        }
        return;
    }
    if (p.c_dtype == HIPATTN_F32) {
        if (p.residual != nullptr) {
            float r[8];
            __builtin_memcpy(r, (const float*)p.residual + to, 32);
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] += r[e];
        }
        __builtin_memcpy((float*)p.c + to, y, 32);
        return;
    }
    if (p.residual != nullptr) {
        uint16_t r[8];
        __builtin_memcpy(r, (const uint16_t*)p.residual + to, 16);
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] += p.c_dtype == HIPATTN_F16 ? f16_bits_to_float(r[e]) : bf16_bits_to_float(r[e]);
    }
    typedef float float2_t __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2_t pair = {y[2 * i], y[2 * i + 1]};
        w[i] = p.c_dtype == HIPATTN_F16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, half2_t))
                                        : __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, bf16x2_t));
    }
    __builtin_memcpy((uint16_t*)p.c + to, w, 16);
}

// ---- how a product is laid out over workgroups ----------------------------------------------------
enum I8Tile { kI8Any32, kI8Few, kI8Tile32, kI8Tile64, kI8Tile128, kI8Tile256, kI8Tile128Deep, kI8Any128, kI8FewWide };  // (the two without LDS: 16 or 32 weight rows to a workgroup)
struct I8Plan {
    I8Tile tile;
    int parts;  // of k, whose sums meet in the workspace
};
struct I8Grid {
    int tiles_m, tiles_n, tiles, parts;
    int group_rows;  // tiles of m that are gone through before the next tile of n
    int xcd_run;     // tiles that an XCD takes
    int rotate;      // tiles begin at different stages of k
    int* sums;       // null, or [parts][m][sums_stride]
    int64_t sums_stride;
};
hipError_t launch_matmul_i8_tiles(const MatmulI8Params& p, const I8Plan& plan, void* workspace, hipStream_t stream);  // matmul_i8_tiles.hip

}  // namespace hipops
