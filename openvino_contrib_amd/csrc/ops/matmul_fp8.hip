// Products of e4m3 codes with a scale for each 128 columns of a row of activations and each 128 x 128 block of weights (hipops_matmul_fp8,
// hipops_matmul_fp8_experts): the entries and the choice among the kernels.
//
//   c[i, j] = sum_b a_scale[i, b] b_scale[j / 128, b] (sum_{l in b} a[i, l] b[j, l]) + bias[j] + residual[i, j]
// A block's 128 products are summed by the matrix instruction from zero, then joined to the result by an fma with the product of its scales:
// the scales are fp32 numbers, which the instruction's own (powers of two) cannot stand for.
#include <algorithm>
#include <cmath>

#include "ops/fp8.hpp"

namespace hipops {

namespace {

bool float_dtype(int d) { return d == HIPATTN_F32 || d == HIPATTN_F16 || d == HIPATTN_BF16; }
int64_t blocks_of(int64_t k) { return (k + kFp8Block - 1) / kFp8Block; }

// the scales' strides as a descriptor has them
hipattn_status checked_strides(const char* what, int64_t row, int64_t block) {
    if (row < 0 || block < 0 || (row == 0) != (block == 0))
        return fail(HIPATTN_INVALID_ARGUMENT, "%s: scale strides %lld and %lld", what, (long long)row, (long long)block);
    return HIPATTN_OK;
}

hipattn_status checked(const hipops_matmul_fp8_desc* d) {
    if (!d) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8: null descriptor");
    if (!float_dtype(d->c_dtype)) return fail(HIPATTN_UNSUPPORTED, "matmul_fp8: result type %d is not f32, f16 or bf16", d->c_dtype);
    if (d->m < 0 || d->n < 0 || d->k < 0)
        return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8: %lld x %lld x %lld", (long long)d->m, (long long)d->n, (long long)d->k);
    if (d->m > 0x7fffffff || d->n > 0x7fffffff || d->k > 0x7fffffff) return fail(HIPATTN_UNSUPPORTED, "matmul_fp8: more than 2^31 - 1 rows or columns");
    if ((d->lda && d->lda < d->k) || (d->ldb && d->ldb < d->k) || (d->ldc && d->ldc < d->n))
        return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8: rows %lld, %lld, %lld apart overlap", (long long)d->lda, (long long)d->ldb, (long long)d->ldc);
    return checked_strides("matmul_fp8", d->a_scale_row_stride, d->a_scale_block_stride);
}

hipattn_status checked(const hipops_matmul_fp8_experts_desc* d) {
    if (!d) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8_experts: null descriptor");
    const bool codes = d->c_dtype == HIPOPS_F8_E4M3;
    if (!codes && !float_dtype(d->c_dtype)) return fail(HIPATTN_UNSUPPORTED, "matmul_fp8_experts: result type %d is not f32, f16, bf16 or e4m3", d->c_dtype);
    if (codes && !d->gated) return fail(HIPATTN_UNSUPPORTED, "matmul_fp8_experts: codes of results that are no gated units");
    if (d->gated && (d->glu_activation < HIPOPS_GLU_SWISH || d->glu_activation > HIPOPS_GLU_GELU_TANH))
        return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8_experts: activation %d", d->glu_activation);
    if (d->gated && d->n % 2) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8_experts: a gated unit of %lld columns has no halves", (long long)d->n);
    if (d->rows < 0 || d->n < 0 || d->k < 0 || d->a_rows < 0 || d->experts < 1)
        return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8_experts: %d experts, %lld rows of %lld, %lld x %lld", d->experts, (long long)d->rows, (long long)d->a_rows,
                    (long long)d->n, (long long)d->k);
    if (d->experts > 1024) return fail(HIPATTN_UNSUPPORTED, "matmul_fp8_experts: %d experts are more than 1024", d->experts);
    if (d->rows > 0x7fffffff || d->a_rows > 0x7fffffff || d->n > 0x7fffffff || d->k > 0x7fffffff)
        return fail(HIPATTN_UNSUPPORTED, "matmul_fp8_experts: more than 2^31 - 1 rows or columns");
    if (d->n > (int64_t)1 << 26) return fail(HIPATTN_UNSUPPORTED, "matmul_fp8_experts: %lld columns are more than 2^26", (long long)d->n);
    if (d->order_divisor < 1) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8_experts: order_divisor %d", d->order_divisor);
    if (d->lda && d->lda < d->k) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8_experts: rows %lld apart overlap", (long long)d->lda);
    return checked_strides("matmul_fp8_experts", d->a_scale_row_stride, d->a_scale_block_stride);
}

int64_t bytes_of_parts(int64_t m, int64_t n, int parts) { return parts > 1 ? parts * m * ((n + 3) / 4 * 4) * 4 : 0; }

// Tiles of 256 rows want whole stages, four of them, columns in whole runs of a wavefront's (gated: of a tile's), weight rows at multiples of 64 bytes from the
// first (a lane's two places in the swizzle differ in one bit of its offset), and scales that 32 bits reach from the first.
bool deep_takes(int64_t n, int64_t k, int64_t columns, int64_t ldb, int64_t rows, int64_t scale_row, int64_t scale_block) {
    const int64_t limit = (int64_t)1 << 30;
    return n % columns == 0 && ldb % 64 == 0 && k % kFp8Block == 0 && k / kFp8Block >= kFp8DeepStages && scale_row < limit && scale_block < limit && rows * scale_row < limit;
}

// Which tile, and how many parts of k: the least time by a model: a stage of 128 bytes of k of a workgroup that is alone, of those that share a compute unit
// in whole rounds, of many; what the weights take to come; the parts' sums and the second launch.  Fitted to the measured times of all tiles at 120 sizes
// (1 to 8,192 rows on weights of 2 to 117 MB): 0.2 % from the best choice on average, 9 % at worst; rows at any address 0.4 % and 6 %.
struct TileCost {
    Fp8Tile tile;
    int rows, columns, most_rows;  // tiles of more rows than this are never the faster ones
    float start, alone, together, through;
};
constexpr TileCost kTileCosts[] = {
    {kFp8Few, 16, 16, 64, 3.08f, 0.11f, 0.112f, 0.0133f},
    {kFp8Tile32, 32, 128, 1024, 5.04f, 0.416f, 0.696f, 0.513f},
    {kFp8Tile64, 64, 128, 2048, 5.88f, 0.462f, 0.594f, 0.543f},
    {kFp8Tile128, 128, 128, 1 << 30, 6.03f, 1.08f, 0.655f, 0.396f},
    {kFp8Tile256, 256, 256, 1 << 30, 8.91f, 1.58f, 1.77f, 1.94f},
};
constexpr TileCost kAnyCosts[] = {{kFp8Any32, 32, 128, 1024, 4.74f, 1.02f, 0.57f, 0.367f}, {kFp8Any128, 128, 128, 1 << 30, 6.33f, 1.29f, 1.41f, 0.257f}};
constexpr int kParts[] = {1, 2, 3, 4, 6, 8, 12, 16};
// (the device's 256 compute units: the other constants were fitted on them and hold for no other number)
constexpr float kUnits = 256.0f;
struct MemoryCost {
    float bytes_per_us, sum_bytes_per_us, second_launch;
};
constexpr MemoryCost kTileMemory = {7.9e6f, 5.14e6f, 2.11f}, kAnyMemory = {4.09e6f, 5.48e6f, 2.22f};

struct Planned {
    Fp8Plan plan;
    float us;
};
Planned plan_of(int64_t m, int64_t n, int64_t k, size_t workspace_bytes, bool aligned, bool exact, bool deep) {
    Planned best{{aligned ? kFp8Tile32 : kFp8Any32, 1}, INFINITY};
    const int64_t stages = blocks_of(k);
    const MemoryCost& memory = aligned ? kTileMemory : kAnyMemory;
    const auto consider = [&](const TileCost& t) {
        if (m > t.most_rows || (exact && t.rows != 16 && t.rows != 32 && t.rows != 128)) return;
        if (t.tile == kFp8Few && (k == 0 || k % kFp8Block != 0)) return;
        const float tiles = (float)((m + t.rows - 1) / t.rows) * (float)((n + t.columns - 1) / t.columns);
        if (t.tile == kFp8Tile256 && !deep) return;
        for (int parts : kParts) {
            if (parts > 1 && (t.tile == kFp8Few || t.tile == kFp8Tile256 || stages < 2 * parts || m > 65535 || (size_t)bytes_of_parts(m, n, parts) > workspace_bytes)) break;
            const float steps = (float)((stages + parts - 1) / parts), each = tiles * parts / kUnits;
            const float stage = std::max({t.alone, each > 1.0f ? ceilf(each) * t.together : 0.0f, each * t.through});
            float us = t.start + std::max(steps * stage, ((float)m + (float)n) * (float)k / memory.bytes_per_us);
            if (parts > 1) us += memory.second_launch + 8.0f * parts * (float)m * (float)n / memory.sum_bytes_per_us;
            if (us < best.us) best = {{t.tile, parts}, us};
        }
    };
    if (aligned)
        for (const TileCost& t : kTileCosts) consider(t);
    else
        for (const TileCost& t : kAnyCosts) consider(t);
    return best;
}

// The columns of a product's first launch: all, or whole runs of 64 for tiles of 256 rows where those and a second launch for the rest are the faster (8,192 x
// 6,150 x 4,096 291 -> 215 us, 512 x 50,257 x 4,096 167 -> 141).
int64_t first_columns(const MatmulFp8Params& p, size_t workspace_bytes, bool aligned, bool exact) {
    const int64_t runs = p.n / 64 * 64;
    if (!aligned || exact || runs == 0 || runs == p.n || !deep_takes(runs, p.k, 64, p.ldb, p.m, p.a_scale_row, p.a_scale_block)) return p.n;
    const float whole = plan_of(p.m, p.n, p.k, workspace_bytes, aligned, exact, false).us;
    const float first = plan_of(p.m, runs, p.k, workspace_bytes, aligned, exact, true).us, rest = plan_of(p.m, p.n - runs, p.k, workspace_bytes, aligned, exact, false).us;
    return first + rest < whole ? runs : p.n;
}

// The tile of an experts' product: by the rows that an expert has on average (how many it has in the end only the device knows).  Measured on 8 experts of
// 28,672 x 4,096 (gated), 128 of 2,816 x 2,048 (gated), 64 of 2,048 x 4,096 and 256 of 1,024 x 2,048, rows spread at random, us of the tiles of 32, 64,
// 128 and 256 rows: 16 rows an expert 180, 185, 222, 235 on the first and 118, 121, 136, 133 on the third; 32 rows 218, 194, 225, 235 and 128, 122, 138, 136;
// 64 rows 297, 255, 233, 240 and 170, 151, 145, 138; 128 rows 457, 347, 321, 273 and 253, 207, 201, 151.  (Tiles of 256 rows load a stage and a half ahead
// and across tiles, so they are ahead long before an expert fills one.)
// Sixteen columns at a time are ahead while they do not fill the chip more than twice over: 8 rows on the 64 experts (1,024 workgroups) 16.8 against 19.7,
// 16 rows (2,048) 28 against 20.5, where a tile's 128 columns share what it takes to find the expert.
Fp8Tile expert_tile_of(const MatmulFp8Params& p, bool aligned, bool exact) {
    const int64_t rows = (p.last_place - p.first_place) / p.experts;
    if (!aligned) return rows <= 48 ? kFp8Any32 : kFp8Any128;  // (32 rows an expert 186 against 251 on 64 of 2,048 x 4,099, 64 rows 316 against 254)
    if (rows <= 16 && (!p.gated || p.n % 128 == 0) && p.k >= kFp8Block && p.k % kFp8Block == 0 && most_expert_tiles(p, 16) * ((p.n + 15) / 16) <= 1024) return kFp8Few;
    if (rows <= 24) return kFp8Tile32;
    if (exact) return kFp8Tile128;
    const bool deep = deep_takes(p.n, p.k, p.gated ? 256 : 64, p.ldb, p.a_rows, p.a_scale_row, p.a_scale_block);
    return rows <= (deep ? 44 : 64) ? kFp8Tile64 : deep ? kFp8Tile256 : kFp8Tile128;
}

hipError_t launch_experts(const MatmulFp8Params& p, bool exact, hipStream_t stream) {
    // (tiles that load straight to LDS address rows in 32 bits: those of a from its beginning or the tile's, weights from the tile's first row)
    const int64_t limit = (int64_t)1 << 32;
    const bool aligned = (((uintptr_t)p.a | (uintptr_t)p.b | (uintptr_t)p.lda | (uintptr_t)p.k) & 15) == 0 && p.lda < limit && (p.order ? p.a_rows : 256) * p.lda < limit &&
                         (p.gated ? p.n : 256) * p.ldb < limit;
    return launch_matmul_fp8_tiles<true>(p, {expert_tile_of(p, aligned, exact), 1}, exact, nullptr, stream);
}

}  // namespace

hipattn_status matmul_fp8_workspace_size(const hipops_matmul_fp8_desc* d, size_t* bytes) {
    if (!bytes) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8_workspace_size: null output");
    *bytes = 0;
    if (const hipattn_status st = checked(d)) return st;
    if (d->m == 0 || d->n == 0 || d->k == 0) return HIPATTN_OK;
    const bool exact = d->c_dtype == HIPATTN_F32;
    const bool strided = d->a_scale_row_stride != 0;
    MatmulFp8Params p{};
    p.m = d->m, p.n = d->n, p.k = d->k, p.ldb = d->ldb ? d->ldb : d->k, p.a_scale_row = strided ? d->a_scale_row_stride : 1, p.a_scale_block = strided ? d->a_scale_block_stride : d->m;
    for (bool aligned : {true, false}) {
        const int64_t first = first_columns(p, SIZE_MAX, aligned, exact);
        for (int64_t n : {first, d->n - first}) {
            const bool deep = deep_takes(n, p.k, 64, p.ldb, p.m, p.a_scale_row, p.a_scale_block);
            if (n > 0) *bytes = std::max(*bytes, (size_t)bytes_of_parts(p.m, n, plan_of(p.m, n, p.k, SIZE_MAX, aligned, exact, deep).plan.parts));
        }
    }
    return HIPATTN_OK;
}

hipattn_status matmul_fp8(const hipops_matmul_fp8_desc* d, const uint8_t* a, const float* a_scales, const uint8_t* b, const float* b_scales, const void* bias,
                          const void* residual, void* c, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (const hipattn_status st = checked(d)) return st;
    if (d->m == 0 || d->n == 0) return HIPATTN_OK;
    if (!c || (d->k > 0 && (!a || !b || !a_scales || !b_scales))) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8: null pointer");
    if ((uintptr_t)workspace % 16) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8: workspace must be 16-byte aligned");
    MatmulFp8Params p{};
    p.a = a, p.b = b, p.a_scales = a_scales, p.b_scales = b_scales, p.bias = bias, p.residual = residual, p.c = c;
    p.m = d->m, p.n = d->n, p.k = d->k, p.lda = d->lda ? d->lda : d->k, p.ldb = d->ldb ? d->ldb : d->k, p.ldc = d->ldc ? d->ldc : d->n, p.c_dtype = d->c_dtype;
    p.a_scale_row = d->a_scale_row_stride ? d->a_scale_row_stride : 1, p.a_scale_block = d->a_scale_row_stride ? d->a_scale_block_stride : d->m;
    // A launch of 2^32 threads or more would run modulo 2^32 of them, without an error: calls that could come to that go in pieces.  Tiles of any number of
    // rows have 128 columns, of which a single one may be there, and 512 threads for 128 rows at most: 2^28 rows of up to 128 columns are 2^30 threads.
    const int64_t most_n = (int64_t)1 << 22, most_m = (((int64_t)1 << 35) / std::max<int64_t>(std::min(d->n, most_n), 128) + 31) / 32 * 32;
    const int64_t size = d->c_dtype == HIPATTN_F32 ? 4 : 2;
    const bool exact = d->c_dtype == HIPATTN_F32;
    const auto from = [](const void* base, int64_t bytes) { return base ? (const uint8_t*)base + bytes : nullptr; };
    const size_t room = workspace ? workspace_bytes : 0;
    for (int64_t i = 0; i < d->m; i += most_m)
        for (int64_t j = 0; j < d->n;) {
            MatmulFp8Params q = p;
            q.m = std::min(d->m - i, most_m), q.n = std::min(d->n - j, most_n);
            q.a = from(a, i * p.lda), q.a_scales = (const float*)from(a_scales, 4 * i * p.a_scale_row);
            q.b = from(b, j * p.ldb), q.b_scales = (const float*)from(b_scales, 4 * (j / kFp8Block) * blocks_of(p.k));
            q.bias = from(bias, size * j), q.residual = from(residual, size * (i * p.ldc + j)), q.c = (uint8_t*)c + size * (i * p.ldc + j);
            // (tiles that load straight to LDS address a row from the tile's first in 32 bits)
            const bool aligned = (((uintptr_t)q.a | (uintptr_t)q.b | (uintptr_t)p.lda | (uintptr_t)p.ldb | (uintptr_t)p.k) & 15) == 0 && p.lda <= (1 << 23) && p.ldb <= (1 << 23);
            q.n = first_columns(q, room, aligned, exact);
            const bool deep = deep_takes(q.n, q.k, 64, q.ldb, q.m, q.a_scale_row, q.a_scale_block);
            const Fp8Plan plan = plan_of(q.m, q.n, q.k, room, aligned, exact, deep).plan;
            if (const hipError_t e = launch_matmul_fp8_tiles<false>(q, plan, exact, workspace, stream); e != hipSuccess)
                return fail(HIPATTN_HIP_ERROR, "matmul_fp8: %s", hipGetErrorString(e));
            j += q.n;  // (a rest of less than 64 columns lies in one block of scales)
        }
    return HIPATTN_OK;
}

// Results as codes go through fp32 results of some rows at a time: as many as the workspace holds, all of them where it has the size asked for.
constexpr int64_t kMostWorkspace = (int64_t)1 << 30;
static int64_t rows_at_once(const hipops_matmul_fp8_experts_desc* d, int64_t bytes) { return std::min(d->rows, bytes / (4 * (d->n / 2))); }

hipattn_status matmul_fp8_experts_workspace_size(const hipops_matmul_fp8_experts_desc* d, size_t* bytes) {
    if (!bytes) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8_experts_workspace_size: null output");
    *bytes = 0;
    if (const hipattn_status st = checked(d)) return st;
    if (d->c_dtype != HIPOPS_F8_E4M3 || d->rows == 0 || d->n == 0) return HIPATTN_OK;
    *bytes = (size_t)(std::max<int64_t>(rows_at_once(d, kMostWorkspace), 1) * 4 * (d->n / 2));
    return HIPATTN_OK;
}

hipattn_status matmul_fp8_experts(const hipops_matmul_fp8_experts_desc* d, const uint8_t* a, const float* a_scales, const uint8_t* b, const float* b_scales,
                                  const int32_t* begins, const int32_t* order, void* c, float* c_scales, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (const hipattn_status st = checked(d)) return st;
    if (d->rows == 0 || d->n == 0) return HIPATTN_OK;
    const bool codes = d->c_dtype == HIPOPS_F8_E4M3;
    if (!c || !begins || (codes && !c_scales) || (d->k > 0 && (!a || !b || !a_scales || !b_scales))) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8_experts: null pointer");
    if (d->a_rows == 0) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8_experts: places without rows of a");
    if (!order && d->a_rows < d->rows)
        return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8_experts: %lld rows of a for %lld places and no order", (long long)d->a_rows, (long long)d->rows);
    if ((uintptr_t)workspace % 16) return fail(HIPATTN_INVALID_ARGUMENT, "matmul_fp8_experts: workspace must be 16-byte aligned");
    MatmulFp8Params p{};
    p.a = a, p.b = b, p.a_scales = a_scales, p.b_scales = b_scales, p.c = codes ? workspace : c, p.m = d->rows, p.n = d->n, p.k = d->k;
    p.lda = d->lda ? d->lda : d->k, p.ldb = d->k, p.ldc = d->gated ? d->n / 2 : d->n, p.c_dtype = codes ? HIPATTN_F32 : d->c_dtype;
    p.a_scale_row = d->a_scale_row_stride ? d->a_scale_row_stride : 1, p.a_scale_block = d->a_scale_row_stride ? d->a_scale_block_stride : d->a_rows;
    p.begins = begins, p.order = order, p.experts = d->experts, p.divisor = d->order_divisor, p.a_rows = d->a_rows;
    p.gated = d->gated != 0, p.activation = d->glu_activation, p.gate_first = d->glu_gate_first;
    // (fewer than 2^32 threads and 2^16 rows of workgroups to a launch, whichever kernel: an expert's last tile may hold a single row)
    int64_t at_once = (int64_t)1 << 19;
    while ((std::min<int64_t>(at_once, d->experts) + at_once / 16) * (d->n / 64 + 1) * 512 >= (int64_t)1 << 32) at_once /= 2;
    at_once = std::min(at_once, d->rows);
    if (codes) {
        at_once = std::min(at_once, workspace ? rows_at_once(d, (int64_t)std::min<size_t>(workspace_bytes, (size_t)1 << 60)) : 0);
        if (at_once == 0) return fail(HIPATTN_WORKSPACE_TOO_SMALL, "matmul_fp8_experts: %zu bytes of workspace hold no row of results", workspace_bytes);
    }
    for (int64_t first = 0; first < d->rows; first += at_once) {
        p.first_place = first, p.last_place = std::min(first + at_once, d->rows);
        hipError_t e = launch_experts(p, d->c_dtype == HIPATTN_F32, stream);
        if (e == hipSuccess && codes) {
            const int64_t width = d->n / 2;
            const QuantizeFp8Params q{workspace, nullptr, (uint8_t*)c + first * width, c_scales + first, p.last_place - first, width, width, 1, d->rows,
                                      HIPATTN_F32, 0, 0, 0, 0.0f, begins, begins + d->experts, first};
            e = launch_quantize_fp8(HIPOPS_QUANTIZE_PLAIN, q, stream);
        } else if (!codes) {
            p.c = (uint8_t*)p.c + (d->c_dtype == HIPATTN_F32 ? 4 : 2) * at_once * p.ldc;
        }
        if (e != hipSuccess) return fail(HIPATTN_HIP_ERROR, "matmul_fp8_experts: %s", hipGetErrorString(e));
    }
    return HIPATTN_OK;
}

}  // namespace hipops
