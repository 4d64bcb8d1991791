// Products of 8-bit codes (hipops_matmul_i8): c = a_scale b_scale (A B^T) + bias + residual, sums exact in 32-bit integers on the
// matrix cores.  The entry, the choice among the kernels, and the one for up to 32 activation rows; the others: matmul_i8_tiles.hip.
#include <algorithm>
#include <cmath>

#include "ops/matmul_i8.hpp"

namespace hipops {

namespace {

// Up to 32 activation rows: the weights, read once, are most of the time.  A workgroup takes 16 kN weight rows and its eight wavefronts an
// eighth of k each; a lane's loads are the matrix operands as they stand (16 bytes of k of weight row lane % 16, of kM tiles of 16 activation
// rows alike), kGroup steps multiplied while the next ones are on their way.  Only the eight partial sums meet in LDS.  One row on
// 4,096 x 4,096 6.0 us alone (2.8 TB/s: launch and one round of loads; in tiles with LDS 10.1), 32 rows 10.1 (11.5): every workgroup reads
// all activations, 16 bytes of 16 rows at a time.  Twice the weight rows halve that, where n still fills the device: 32 x 6,144 x 2,048
// 10.1 -> 8.6 us (in tiles 10.7), 16 x 28,672 x 4,096 38.4 -> 33.0 (25.0).
constexpr int kFewWaves = 8;

template <bool kAligned>
__device__ __forceinline__ uint4_t piece_at(const int8_t* p) {
    if constexpr (kAligned) return *(const uint4_t*)p;
    uint4_t w;
    __builtin_memcpy(&w, p, 16);
    return w;
}

template <int kM, int kN, bool kAligned>
__global__ __launch_bounds__(64 * kFewWaves) void matmul_i8_few_kernel(MatmulI8Params p) {
    constexpr int kGroup = 4;
    static_assert(kM * kN <= kFewWaves, "a wavefront for each tile of the result");
    __shared__ int4_t sums[kFewWaves][kM * kN][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, row = lane & 15, quarter = lane >> 4;
    const int64_t n0 = 16 * kN * (int64_t)blockIdx.x;
    const int pieces = (int)(p.k / 16), steps = (pieces + 3) / 4;
    const int first = steps * wave / kFewWaves, last = steps * (wave + 1) / kFewWaves;
    const int8_t *w[kN], *x[kM];
#pragma unroll
    for (int j = 0; j < kN; j++) w[j] = p.b + min(n0 + 16 * j + row, p.n - 1) * p.ldb + 16 * quarter;
#pragma unroll
    for (int i = 0; i < kM; i++) x[i] = p.a + min((int64_t)(16 * i + row), p.m - 1) * p.lda + 16 * quarter;
    const bool real = kM > 1 || row < p.m;  // (a single tile: lanes without a row load nothing)
    const int whole = (pieces - quarter + 3) / 4;  // steps in which this lane has a piece
    int4_t acc[kN][kM];
#pragma unroll
    for (int j = 0; j < kN; j++)
#pragma unroll
        for (int i = 0; i < kM; i++) acc[j][i] = (int4_t){0, 0, 0, 0};
    struct Group {
        uint4_t w[kGroup][kN], x[kGroup][kM];
    } now, next;
    const auto load = [&](Group& g, int s) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kGroup; u++) {
            const int at = min(s + u, last - 1);  // (past the end: unused)
#pragma unroll
            for (int j = 0; j < kN; j++) {
                g.w[u][j] = (uint4_t){0u, 0u, 0u, 0u};
                if (at < whole) g.w[u][j] = piece_at<kAligned>(w[j] + 64 * (int64_t)at);
            }
        }
        if (real) {
#pragma unroll
            for (int u = 0; u < kGroup; u++) {
                const int at = min(s + u, last - 1);
#pragma unroll
                for (int i = 0; i < kM; i++)
                    if (at < whole) g.x[u][i] = piece_at<kAligned>(x[i] + 64 * (int64_t)at);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    const auto multiply = [&](const Group& g, int s) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < kGroup; u++)
            if (s + u < last) {
#pragma unroll
                for (int j = 0; j < kN; j++)
#pragma unroll
                    for (int i = 0; i < kM; i++) acc[j][i] = mma_i8_16(g.w[u][j], g.x[u][i], acc[j][i]);
            }
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int u = 0; u < kGroup; u++)
#pragma unroll
        for (int i = 0; i < kM; i++) now.x[u][i] = next.x[u][i] = (uint4_t){0u, 0u, 0u, 0u};  // (lanes without a row or a piece keep these)
    if (first < last) {
        load(now, first);
        for (int s = first; s < last; s += 2 * kGroup) {
            if (s + kGroup < last) load(next, s + kGroup);
            multiply(now, s);
            if (s + 2 * kGroup < last) load(now, s + 2 * kGroup);
            multiply(next, s + kGroup);
        }
    }
    if constexpr (!kAligned) {  // what is left of the rows behind their last whole piece
        if (wave == kFewWaves - 1 && p.k % 16 != 0) {
            uint4_t xs[kM];
#pragma unroll
            for (int i = 0; i < kM; i++) xs[i] = quarter == 0 ? load_codes16(x[i], 16 * (int64_t)pieces, p.k) : (uint4_t){0u, 0u, 0u, 0u};
#pragma unroll
            for (int j = 0; j < kN; j++) {
                const uint4_t ws = quarter == 0 ? load_codes16(w[j], 16 * (int64_t)pieces, p.k) : (uint4_t){0u, 0u, 0u, 0u};
#pragma unroll
                for (int i = 0; i < kM; i++) acc[j][i] = mma_i8_16(ws, xs[i], acc[j][i]);
            }
        }
    }
    // register r: weight row 4 quarter + r, activation row lane % 16 of a tile
#pragma unroll
    for (int j = 0; j < kN; j++)
#pragma unroll
        for (int i = 0; i < kM; i++) sums[wave][j * kM + i][lane] = acc[j][i];
    __syncthreads();
    if (wave >= kM * kN) return;
    const int64_t to_row = 16 * (wave % kM) + row, to_column = n0 + 16 * (wave / kM) + 4 * quarter;
    if (to_row >= p.m) return;
    int4_t sum = sums[0][wave][lane];
#pragma unroll
    for (int i = 1; i < kFewWaves; i++) sum += sums[i][wave][lane];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int64_t column = to_column + r;
        if (column < p.n)
            store_scalar(p.c, to_row * p.ldc + column, p.c_dtype, finished(p, sum[r], to_row, column, p.b_scales ? p.b_scales[column] : 1.0f));
    }
}

template <int kM, int kN, bool kAligned>
void launch_few(const MatmulI8Params& p, hipStream_t stream) {
    hipLaunchKernelGGL((matmul_i8_few_kernel<kM, kN, kAligned>), dim3((unsigned)((p.n + 16 * kN - 1) / (16 * kN))), dim3(64 * kFewWaves), 0, stream, p);
}
void launch_few(const MatmulI8Params& p, bool wide, bool aligned, hipStream_t stream) {
    if (!aligned)
        p.m <= 16 ? launch_few<1, 1, false>(p, stream) : launch_few<2, 1, false>(p, stream);
    else if (wide)
        p.m <= 16 ? launch_few<1, 2, true>(p, stream) : launch_few<2, 2, true>(p, stream);
    else
        p.m <= 16 ? launch_few<1, 1, true>(p, stream) : launch_few<2, 1, true>(p, stream);
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
// others than those of the calls before, 768 MB of them in turn, the activations the same), over 330 sizes: m of 1 to 8,192 on weights of 4,096 x
// 4,096, 28,672 x 4,096, 11,008 x 4,096, 4,096 x 14,336, 5,120 x 13,824, 2,560 x 10,240, 1,024 x 4,096, 6,144 x 4,096 and 2,048, 512 x 2,048, 320
// and 2,048 x 1,024, 128 x 8,192.  Its choice is 0.7 % from the best of all choices on average, 15 % at worst (256 x 4,096 x 4,096: 20.3 for 17.7).
// (Fitted to calls whose weights had stayed in the last cache, it was 2.3 % off on average and 64 % at worst.)
// A tile costs its start and end, and for each stage of 128 bytes of k the largest of: what a compute unit takes that has one tile
// (`alone`: the loads it waits for); with more tiles than compute units, what the fullest takes (`together`) and the whole device
// (`through`: power and the caches).  The operands' bytes bound it from below.  Parts of k cost the second launch and their sums' way
// through memory.  Where the sides cross (us, m x n x k): 64 x 4,096 x 4,096 tiles of 32 rows in four parts 13.5, of 64 in six 13.8; 512 x 4,096
// x 4,096 of 64 20.6, of 128 with a deep ring 22.8, of 128 in four parts 28.6, of 256 in six 34.4; 600 x 5,120 x 13,824 of 128 with a deep ring
// 61.3, of 256 in four parts 69.1, of 128 in two 70.8, of 64 84.9; 1,024 x 6,144 x 4,096 of 128 42.3, deep 45.4, of 256 in two parts 54.6; 1,111 x
// 4,096 x 14,336 of 256 in three parts 93.9, of 128 109; 1,500 x 4,096 x 14,336 of 128 112, of 256 in two parts 117; 3,000 x 4,096 x 14,336 of 256
// 174, of 128 201; 8,192 x 6,144 x 4,096 of 256 198, of 128 243; 24 x 4,096 x 4,096 without LDS 9.2, with 11.0; 24 x 6,144 x 4,096 12.5
// (wide) and 13.0; 16 x 28,672 x 4,096 33.0 (wide) and 25.0.
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
// Rows at any address: up to 32 without LDS (us: 1 x 512 x 2,047 7.1, in tiles 10.5; 1 x 4,096 x 4,095 11.6 and 14.1; 16 x 320 x 1,001 6.5 and 9.9; 16
// x 4,096 x 4,095 18.2 and 15.5: loads that cross lines), tiles through registers (us, tiles of 32 rows / 128 rows at their best parts: 64 x 4,095 x 4,095 16.8 / -; 512 x 4,095 x 4,095
// 39.6 / 37.1; 128 x 4,095 x 14,333 38.9 / 34.9; 100 x 2,001 x 1,001 10.4 / 17.8; 8,191 x 6,143 x 4,097 - / 391).
constexpr TileCost kAnyCosts[] = {{kI8Any32, 32, 128, 512, 5.63f, 1.12f, 0.746f, 0.763f}, {kI8Any128, 128, 128, 1 << 30, 6.8f, 1.84f, 1.21f, 0.556f}};
constexpr int kParts[] = {1, 2, 3, 4, 6, 8, 12, 16};
// (the device's 256 compute units: the other constants were fitted on them and hold for no other number)
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
    const float steps = (float)k / 2048.0f, rows = (float)m, bytes = (float)n * (float)k;
    if (!aligned) {
        if (m <= 32) {
            least = 2.86f + std::max(3.76f * steps * (1.0f + 0.0537f * rows), 3.47f * ceilf((float)n / (16.0f * kUnits)) * steps * (1.0f + 0.0755f * rows));
            best = {kI8Few, 1};
        }
        for (const TileCost& t : kAnyCosts) consider(t);
        return best;
    }
    if (m <= 32) {
        const float narrow = 3.88f + std::max({0.808f * steps * (1.0f + 0.0772f * rows), 0.962f * ceilf((float)n / (16.0f * kUnits)) * steps * (1.0f + 0.0527f * rows), bytes / 5.68e6f});
        const float wide = 3.69f + std::max({2.24f * steps * (1.0f + 0.0311f * rows), 1.29f * ceilf((float)n / (32.0f * kUnits)) * steps * (1.0f + 0.0786f * rows), bytes / 5.37e6f});
        least = std::min(narrow, wide);
        best = {wide < narrow ? kI8FewWide : kI8Few, 1};
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
    // A launch of 2^32 threads or more would run modulo 2^32 of them, without an error: calls that could come to that go in pieces.  (Without
    // LDS a column of results takes 32 lanes; in tiles 128 x 128 of them take 512 at most, the smaller tiles those of few rows.)
    const int64_t most_n = (int64_t)1 << 26, most_m = (((int64_t)1 << 30) - 1) / ((std::min(d->n, most_n) + 127) / 128);
    if (d->n > most_n || d->m > most_m) {
        const int64_t size = d->c_dtype == HIPATTN_F32 ? 4 : 2;
        const auto from = [](auto* base, int64_t bytes) { return base ? (decltype(base))((const uint8_t*)base + bytes) : nullptr; };
        for (int64_t i = 0; i < d->m; i += most_m)
            for (int64_t j = 0; j < d->n; j += most_n) {
                const hipops_matmul_i8_desc piece{d->c_dtype, std::min(d->m - i, most_m), std::min(d->n - j, most_n), d->k, p.lda, p.ldb, p.ldc};
                const int64_t at = size * (i * p.ldc + j);
                if (const hipattn_status st = matmul_i8(&piece, from(a, i * p.lda), from(a_scales, 4 * i), from(b, j * p.ldb), from(b_scales, 4 * j), from(bias, size * j),
                                                        from(residual, at), from(c, at), workspace, workspace_bytes, stream))
                    return st;
            }
        return HIPATTN_OK;
    }
    // (tiles that load straight to LDS address a row from the tile's first in 32 bits)
    const bool aligned = (((uintptr_t)a | (uintptr_t)b | (uintptr_t)p.lda | (uintptr_t)p.ldb | (uintptr_t)p.k) & 15) == 0 && p.lda <= (1 << 23) && p.ldb <= (1 << 23);
    const I8Plan plan = plan_of(p.m, p.n, p.k, workspace ? workspace_bytes : 0, aligned);
    hipError_t e = hipSuccess;
    if (plan.tile == kI8Few || plan.tile == kI8FewWide) {
        launch_few(p, plan.tile == kI8FewWide, aligned, stream);
        e = hipGetLastError();
    } else {
        e = launch_matmul_i8_tiles(p, plan, workspace, stream);
    }
    if (e != hipSuccess) return fail(HIPATTN_HIP_ERROR, "matmul_i8: %s", hipGetErrorString(e));
    return HIPATTN_OK;
}

}  // namespace hipops
