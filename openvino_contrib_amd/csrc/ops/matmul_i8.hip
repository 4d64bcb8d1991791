// Products of 8-bit codes (hipops_matmul_i8): c = a_scale b_scale (A B^T) + bias + residual on v_mfma_i32_32x32x32_i8, sums exact in
// 32-bit integers.
#include "ops/matmul_i8.hpp"

namespace hipops {

namespace {

// The plain kernel: any strides, alignment and k.  Four wavefronts, a tile of 64 x 64, 64 bytes of k at a time through LDS.
constexpr int kPlainTile = 64, kPlainK = 64;

__device__ __forceinline__ uint4_t load_codes16(const int8_t* row, int64_t at, int64_t k, bool there, bool aligned) {
    if (!there || at >= k) return (uint4_t){0u, 0u, 0u, 0u};
    if (aligned && at + 16 <= k) return *(const uint4_t*)(row + at);
    uint4_t w = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 16; e++)
        if (at + e < k) w[e >> 2] |= (uint32_t)(uint8_t)row[at + e] << (8 * (e & 3));
    return w;
}

__global__ __launch_bounds__(256) void matmul_i8_plain_kernel(MatmulI8Params p, int aligned) {
    __shared__ uint4_t tile[2][kPlainTile][kPlainK / 16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t m0 = (int64_t)blockIdx.y * kPlainTile, n0 = (int64_t)blockIdx.x * kPlainTile;
    const int row = threadIdx.x >> 2, piece = threadIdx.x & 3;
    const int8_t* const a = p.a + (m0 + row) * p.lda;
    const int8_t* const b = p.b + (n0 + row) * p.ldb;
    const bool a_there = m0 + row < p.m, b_there = n0 + row < p.n;
    int16v_t acc;
#pragma unroll
    for (int r = 0; r < 16; r++) acc[r] = 0;
    const int mi = 32 * (wave & 1), ni = 32 * (wave >> 1);
    for (int64_t k0 = 0; k0 < p.k; k0 += kPlainK) {
        const uint4_t x = load_codes16(a, k0 + 16 * piece, p.k, a_there, aligned), w = load_codes16(b, k0 + 16 * piece, p.k, b_there, aligned);
        __syncthreads();
        tile[0][row][piece ^ ((row >> 2) & 3)] = x;
        tile[1][row][piece ^ ((row >> 2) & 3)] = w;
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 2; s++) {
            const int c = 2 * s + (lane >> 5), r = lane & 31;
            acc = mma_i8(tile[0][mi + r][c ^ (((mi + r) >> 2) & 3)], tile[1][ni + r][c ^ (((ni + r) >> 2) & 3)], acc);
        }
    }
    const int64_t col = n0 + ni + (lane & 31);
    if (col >= p.n) return;
    const float scale = p.b_scales ? p.b_scales[col] : 1.0f;
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const int64_t i = m0 + mi + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
        if (i < p.m) store_scalar(p.c, i * p.ldc + col, p.c_dtype, finished(p, acc[r], i, col, scale));
    }
}

bool float_dtype(int d) { return d == HIPATTN_F32 || d == HIPATTN_F16 || d == HIPATTN_BF16; }

hipattn_status checked(const hipops_matmul_i8_desc* d) {
    if (!d) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_i8: null descriptor");
    if (!float_dtype(d->c_dtype)) return fail(HIPATTN_UNSUPPORTED, "matmul_i8: result type %d is not f32, f16 or bf16", d->c_dtype);
    if (d->m < 0 || d->n < 0 || d->k < 0)
        return fail(HIPATTN_INVALID_ARGUMENT, "matmul_i8: %lld x %lld x %lld", (long long)d->m, (long long)d->n, (long long)d->k);
    if (d->m > 0x7fffffff || d->n > 0x7fffffff) return fail(HIPATTN_UNSUPPORTED, "matmul_i8: more than 2^31 - 1 rows or columns");
    if (d->k > 131071) return fail(HIPATTN_UNSUPPORTED, "matmul_i8: k %lld: sums of more than 131,071 products may pass 32 bits", (long long)d->k);
    if ((d->lda && d->lda < d->k) || (d->ldb && d->ldb < d->k) || (d->ldc && d->ldc < d->n))
        return fail(HIPATTN_INVALID_ARGUMENT, "matmul_i8: rows %lld, %lld, %lld apart overlap", (long long)d->lda, (long long)d->ldb, (long long)d->ldc);
    return HIPATTN_OK;
}

}  // namespace

hipattn_status matmul_i8_workspace_size(const hipops_matmul_i8_desc* d, size_t* bytes) {
    if (!bytes) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_i8_workspace_size: null output");
    *bytes = 0;
    return checked(d);
}

hipattn_status matmul_i8(const hipops_matmul_i8_desc* d, const int8_t* a, const float* a_scales, const int8_t* b, const float* b_scales, const void* bias,
                         const void* residual, void* c, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (const hipattn_status st = checked(d)) return st;
    if (d->m == 0 || d->n == 0) return HIPATTN_OK;
    if (!c || (d->k > 0 && (!a || !b))) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_i8: null pointer");
    const MatmulI8Params p{a, b, a_scales, b_scales, bias, residual, c, d->m, d->n, d->k, d->lda ? d->lda : d->k, d->ldb ? d->ldb : d->k,
                           d->ldc ? d->ldc : d->n, d->c_dtype};
    (void)workspace;
    (void)workspace_bytes;
    const bool aligned = (((uintptr_t)a | (uintptr_t)b | (uintptr_t)p.lda | (uintptr_t)p.ldb) & 15) == 0;
    const dim3 grid((unsigned)((p.n + kPlainTile - 1) / kPlainTile), (unsigned)((p.m + kPlainTile - 1) / kPlainTile));
    if (grid.y > 65535) return fail(HIPATTN_UNSUPPORTED, "matmul_i8: %lld rows", (long long)p.m);
    hipLaunchKernelGGL(matmul_i8_plain_kernel, grid, dim3(256), 0, stream, p, aligned ? 1 : 0);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return fail(HIPATTN_HIP_ERROR, "matmul_i8: %s", hipGetErrorString(e));
    return HIPATTN_OK;
}

}  // namespace hipops
