// Products of 8-bit codes (hipops_matmul_i8): c = a_scale b_scale (A B^T) + bias + residual, sums exact in 32-bit integers on the
// matrix cores.  The entry, the choice among the kernels, and the one for up to 16 activation rows; the others: matmul_i8_tiles.hip.
#include <algorithm>
#include <cmath>

#include "ops/matmul_i8.hpp"

namespace hipops {

namespace {

// Up to 16 activation rows: the weights, read once, are all of the time.  A workgroup takes 16 weight rows and its eight wavefronts an
// eighth of k each; a lane's loads are the matrix operands as they stand (16 bytes of k of weight row lane % 16, activations
// alike), kFewGroup steps multiplied while the next ones are on their way.  Only the eight partial sums meet in LDS.  One row on
// 4,096 x 4,096 6.0 us (2.8 TB/s: launch and one round of loads; in tiles 10.9), on 4,096 x 14,336 14.3.
constexpr int kFewWaves = 8, kFewGroup = 4;

__global__ __launch_bounds__(64 * kFewWaves) void matmul_i8_few_kernel(MatmulI8Params p) {
    __shared__ int4_t sums[kFewWaves][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, row = lane & 15, quarter = lane >> 4;
    const int64_t n0 = 16 * (int64_t)blockIdx.x;
    const int steps = (int)((p.k + 63) / 64);
    const int first = steps * wave / kFewWaves, last = steps * (wave + 1) / kFewWaves;
    const int8_t* const w = p.b + min(n0 + row, p.n - 1) * p.ldb + 16 * quarter;
    const int8_t* const x = p.a + (int64_t)min((int64_t)row, p.m - 1) * p.lda + 16 * quarter;
    const bool real = row < p.m;
    const int whole = (int)((p.k - 16 * quarter + 48) / 64);  // steps in which this lane has a piece (k is a multiple of 16)
    int4_t acc = {0, 0, 0, 0};
    struct Group {
        uint4_t w[kFewGroup], x[kFewGroup];
    } now, next;
    const auto load = [&](Group& g, int s) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kFewGroup; u++) {
            const int at = min(s + u, last - 1);  // (past the end: unused)
            g.w[u] = (uint4_t){0u, 0u, 0u, 0u};
            if (at < whole) g.w[u] = *(const uint4_t*)(w + 64 * (int64_t)at);
        }
        if (real) {
#pragma unroll
            for (int u = 0; u < kFewGroup; u++) {
                const int at = min(s + u, last - 1);
                if (at < whole) g.x[u] = *(const uint4_t*)(x + 64 * (int64_t)at);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto multiply = [&](const Group& g, int s) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kFewGroup; u++)
            if (s + u < last) acc = mma_i8_16(g.w[u], g.x[u], acc);
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int u = 0; u < kFewGroup; u++) now.x[u] = next.x[u] = (uint4_t){0u, 0u, 0u, 0u};  // (lanes without a row keep these)
    if (first < last) {
        load(now, first);
        for (int s = first; s < last; s += 2 * kFewGroup) {
            if (s + kFewGroup < last) load(next, s + kFewGroup);
            multiply(now, s);
            if (s + 2 * kFewGroup < last) load(now, s + 2 * kFewGroup);
            multiply(next, s + kFewGroup);
        }
    }
    // register r: weight row 4 quarter + r, activation row lane % 16
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave != 0 || !real) return;
    int4_t sum = sums[0][lane];
#pragma unroll
    for (int i = 1; i < kFewWaves; i++) sum += sums[i][lane];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int64_t column = n0 + 4 * quarter + r;
        if (column < p.n) store_scalar(p.c, row * p.ldc + column, p.c_dtype, finished(p, sum[r], row, column, p.b_scales ? p.b_scales[column] : 1.0f));
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

int64_t bytes_of_parts(int64_t m, int64_t n, int parts) { return parts > 1 ? parts * m * ((n + 3) / 4 * 4) * 4 : 0; }

// Which kernel, and how many parts of k: the least time by a model of what was measured (us; bf16 results, the weights of each call
// others than those of the calls before, 768 MB of them in turn, the activations the same), over 291 sizes: m of 1 to 8,192 on weights of 4,096 x
// 4,096, 28,672 x 4,096, 11,008 x 4,096, 4,096 x 14,336, 5,120 x 13,824, 2,560 x 10,240, 1,024 x 4,096, 6,144 x 4,096 and 2,048, 512 x 2,048, 320
// and 2,048 x 1,024, 128 x 8,192.  Its choice is 0.5 % from the best of all choices on average, 15 % at worst (256 x 4,096 x 4,096: 20.3 for 17.7).
// (Fitted to calls whose weights had stayed in the last cache, it was 2.3 % off on average and 64 % at worst.)
// A tile costs its start and end, and for each stage of 128 bytes of k the largest of: what a compute unit takes that has one tile
// (`alone`: the loads it waits for); with more tiles than compute units, what the fullest takes (`together`) and the whole device
// (`through`: power and the caches).  The operands' bytes bound it from below.  Parts of k cost the second launch and their sums' way
// through memory.  Where the sides cross (us, m x n x k): 64 x 4,096 x 4,096 tiles of 32 rows in four parts 13.5, of 64 in six 13.8; 512 x 4,096
// x 4,096 of 64 20.6, of 128 with a deep ring 22.8, of 128 in four parts 28.6, of 256 in six 34.4; 600 x 5,120 x 13,824 of 128 with a deep ring
// 61.3, of 256 in four parts 69.1, of 128 in two 70.8, of 64 84.9; 1,024 x 6,144 x 4,096 of 128 42.3, deep 45.4, of 256 in two parts 54.6; 1,111 x
// 4,096 x 14,336 of 256 in three parts 93.9, of 128 109; 1,500 x 4,096 x 14,336 of 128 112, of 256 in two parts 117; 3,000 x 4,096 x 14,336 of 256
// 174, of 128 201; 8,192 x 6,144 x 4,096 of 256 198, of 128 243; 16 x 4,096 x 4,096 without LDS 8.0, with 10.9; 16 x 28,672 x 4,096 38.3 and 24.9.
struct TileCost {
    I8Tile tile;
    int rows, columns, most_rows;  // tiles of more rows than this are never the faster ones
    float start, alone, together, through;
};
constexpr TileCost kTileCosts[] = {
    {kI8Tile32, 32, 128, 128, 3.94f, 0.434f, 0.534f, 0.517f},           {kI8Tile64, 64, 128, 1600, 4.48f, 0.449f, 0.388f, 0.483f},
    {kI8Tile128Deep, 128, 128, 1 << 30, 5.15f, 0.527f, 0.648f, 0.560f}, {kI8Tile128, 128, 128, 1 << 30, 6.42f, 0.775f, 0.505f, 0.534f},
    {kI8Tile256, 256, 256, 1 << 30, 12.5f, 1.14f, 1.66f, 1.37f},
};
// Rows at any address, through registers (us, tiles of 32 rows / 128 rows at their best parts: 64 x 4,095 x 4,095 16.8 / -; 512 x 4,095 x 4,095
// 39.6 / 37.1; 128 x 4,095 x 14,333 38.9 / 34.9; 100 x 2,001 x 1,001 10.4 / 17.8; 8,191 x 6,143 x 4,097 - / 391).
constexpr TileCost kAnyCosts[] = {{kI8Any32, 32, 128, 512, 3.8f, 0.90f, 0.55f, 0.55f}, {kI8Any128, 128, 128, 1 << 30, 6.5f, 1.65f, 0.94f, 0.94f}};
constexpr int kParts[] = {1, 2, 3, 4, 6, 8, 12, 16};
constexpr float kUnits = 256.0f, kBytesPerUs = 8.0e6f, kSumBytesPerUs = 3.88e6f, kSecondLaunch = 2.88f;

I8Plan plan_of(int64_t m, int64_t n, int64_t k, size_t workspace_bytes, bool aligned) {
    I8Plan best{aligned ? kI8Tile32 : kI8Any32, 1};
    float least = INFINITY;
    const int64_t stages = (k + 127) / 128;
    const auto consider = [&](const TileCost& t) {
        if (m > t.most_rows) return;
        const float tiles = (float)((m + t.rows - 1) / t.rows) * (float)((n + t.columns - 1) / t.columns);
        for (int parts : kParts) {
            if (parts > 1 && (stages < 2 * parts || m > 65535 || (size_t)bytes_of_parts(m, n, parts) > workspace_bytes)) break;
            const float steps = (float)((stages + parts - 1) / parts), each = tiles * parts / kUnits;
            const float stage = std::max({t.alone, each > 1.0f ? ceilf(each) * t.together : 0.0f, each * t.through});
            float us = t.start + std::max(steps * stage, ((float)m + (float)n) * (float)k / kBytesPerUs);
            if (parts > 1) us += kSecondLaunch + 8.0f * parts * (float)m * (float)n / kSumBytesPerUs;
            if (us < least) least = us, best = {t.tile, parts};
        }
    };
    if (!aligned) {
        for (const TileCost& t : kAnyCosts) consider(t);
        return best;
    }
    if (m <= 16) {
        const float steps = (float)k / 2048.0f, rounds = ceilf((float)n / 16.0f / kUnits);
        least = 3.98f + std::max({0.275f * steps, 0.565f * rounds * steps * (1.0f + 0.134f * (float)m), (float)n * (float)k / 5.76e6f});
        best = {kI8Few, 1};
    }
    for (const TileCost& t : kTileCosts) consider(t);
    return best;
}

}  // namespace

hipattn_status matmul_i8_workspace_size(const hipops_matmul_i8_desc* d, size_t* bytes) {
    if (!bytes) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_i8_workspace_size: null output");
    *bytes = 0;
    if (const hipattn_status st = checked(d)) return st;
    if (d->m == 0 || d->n == 0 || d->k == 0) return HIPATTN_OK;
    *bytes = (size_t)bytes_of_parts(d->m, d->n, std::max(plan_of(d->m, d->n, d->k, SIZE_MAX, true).parts, plan_of(d->m, d->n, d->k, SIZE_MAX, false).parts));
    return HIPATTN_OK;
}

hipattn_status matmul_i8(const hipops_matmul_i8_desc* d, const int8_t* a, const float* a_scales, const int8_t* b, const float* b_scales, const void* bias,
                         const void* residual, void* c, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (const hipattn_status st = checked(d)) return st;
    if (d->m == 0 || d->n == 0) return HIPATTN_OK;
    if (!c || (d->k > 0 && (!a || !b))) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_i8: null pointer");
    const MatmulI8Params p{a, b, a_scales, b_scales, bias, residual, c, d->m, d->n, d->k, d->lda ? d->lda : d->k, d->ldb ? d->ldb : d->k,
                           d->ldc ? d->ldc : d->n, d->c_dtype};
    if ((uintptr_t)workspace % 16) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_i8: workspace must be 16-byte aligned");
    // (tiles that load straight to LDS address a row from the tile's first in 32 bits)
    const bool aligned = (((uintptr_t)a | (uintptr_t)b | (uintptr_t)p.lda | (uintptr_t)p.ldb | (uintptr_t)p.k) & 15) == 0 && p.lda <= (1 << 23) && p.ldb <= (1 << 23);
    const I8Plan plan = plan_of(p.m, p.n, p.k, workspace ? workspace_bytes : 0, aligned);
    hipError_t e = hipSuccess;
    if (plan.tile == kI8Few) {
        hipLaunchKernelGGL(matmul_i8_few_kernel, dim3((unsigned)((p.n + 15) / 16)), dim3(64 * kFewWaves), 0, stream, p);
        e = hipGetLastError();
    } else {
        e = launch_matmul_i8_tiles(p, plan, workspace, stream);
    }
    if (e != hipSuccess) return fail(HIPATTN_HIP_ERROR, "matmul_i8: %s", hipGetErrorString(e));
    return HIPATTN_OK;
}

}  // namespace hipops
