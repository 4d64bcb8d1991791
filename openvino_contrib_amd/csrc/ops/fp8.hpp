// What the kernels of e4m3 codes share (hipops_quantize_fp8, hipops_matmul_fp8, hipops_matmul_fp8_experts): operands, the matrix
// instructions, the way from a workgroup to an expert's rows, and the end of a result.
#pragma once

#include "hipops_experts.h"
#include "ops/ops_common.hpp"
#include "ops/vec8.hpp"

namespace hipops {

typedef int int8v_t __attribute__((ext_vector_type(8)));

constexpr int kFp8Block = HIPOPS_FP8_BLOCK;
constexpr float kFp8Largest = 448.0f;

struct MatmulFp8Params {
    const uint8_t* a;  // [m or a_rows, k]
    const uint8_t* b;  // [n, k], or [experts, n, k]
    const float* a_scales;
    const float* b_scales;
    const void* bias;
    const void* residual;
    void* c;
    int64_t m, n, k;  // (experts: m places at most)
    int64_t lda, ldb, ldc;
    int64_t a_scale_row, a_scale_block;
    int c_dtype;
    // of experts alone
    const int32_t* begins;
    const int32_t* order;
    int experts, divisor;
    int64_t a_rows;
    int64_t first_place, last_place;  // the places that this launch looks at; place p's result is row p - first_place of c
    int gated, activation, gate_first;  // results are the GLU of the product's halves
};

// 16 rows of each operand, 128 bytes of k: lane l holds 32 bytes of row l % 16, the same ones for both operands whichever they are; register r of
// the result is row 4 (l / 16) + r of a and row l % 16 of b
__device__ __forceinline__ float4_t mma_fp8_16(int8v_t a, int8v_t b, float4_t c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
}
// the same of codes as fp16 numbers, whose products and sums keep 32 bits (mma_fp8_16 adds eight neighbouring products with 14 bits below the largest)
__device__ __forceinline__ float4_t mma_fp8_16_exact(int8v_t a, int8v_t b, float4_t c) {
#pragma unroll
    for (int s = 0; s < 4; s++) {
        const auto halves = [&](const int8v_t& v) __attribute__((always_inline)) {
            typedef _Float16 half8_v __attribute__((ext_vector_type(8)));
            half8_v h;
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[2 * s + w], 1.0f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[2 * s + w], 1.0f, true);
                h[4 * w] = lo[0], h[4 * w + 1] = lo[1], h[4 * w + 2] = hi[0], h[4 * w + 3] = hi[1];
            }
            return h;
        };
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(halves(a), halves(b), c, 0, 0, 0);
    }
    return c;
}
__device__ __forceinline__ int8v_t joined(uint4_t lo, uint4_t hi) {
    return (int8v_t){(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}

// 16 bytes of a row from `at` on, zeros where it has ended; at any address.
__device__ __forceinline__ uint4_t load_bytes16(const uint8_t* row, int64_t at, int64_t k) {
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
            for (int e = 0; e < rest; e++) v |= (unsigned __int128)row[at + e] << (8 * e);
        }
        __builtin_memcpy(&w, &v, 16);
    }
    return w;
}

typedef const __attribute__((address_space(1))) int32_t* GlobalIndex;
// The experts' tiles of `rows` rows each, in the order of the experts: how many there are, and for one of them its expert, its first place and the
// places from there to the expert's end.  A wavefront adds them up, up to sixteen experts a lane; every wavefront for itself.
template <bool kExperts>
struct ExpertTiles {
    int each, first, until, tiles;  // this lane's experts, and tiles up to and with them
    int64_t first_from, first_to;   // the first one's places
    int total;
    __device__ __forceinline__ static int64_t place_at(const MatmulFp8Params& p, int e, int64_t least) { return min(max((int64_t)((GlobalIndex)p.begins)[e], least), p.last_place); }
    __device__ __forceinline__ ExpertTiles(const MatmulFp8Params& p, int rows, int lane) {
        if constexpr (!kExperts) return;
        each = (p.experts + 63) >> 6, first = lane * each, tiles = 0;
        for (int i = 0; i < each && first + i < p.experts; i++) {
            const int64_t b = place_at(p, first + i, p.first_place), e = place_at(p, first + i + 1, b);
            tiles += (int)((e - b + rows - 1) / rows);
            if (i == 0) first_from = b, first_to = e;
        }
        until = tiles;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int other = __shfl_up(until, off, 64);
            if (lane >= off) until += other;
        }
        total = __builtin_amdgcn_readlane(until, 63);
    }
    // tile < total
    __device__ __forceinline__ void find(const MatmulFp8Params& p, int tile, int rows, int lane, int& expert, int64_t& place, int64_t& count) const {
        const int owner = __builtin_ctzll(__ballot(until > tile));
        int left = tile - (until - tiles), found = 0;
        int64_t from = 0, to = 0;
        if (lane == owner) {
            for (int i = 0; i < each && first + i < p.experts; i++) {
                const int64_t b = i == 0 ? first_from : place_at(p, first + i, p.first_place), e = i == 0 ? first_to : place_at(p, first + i + 1, b);
                const int here = (int)((e - b + rows - 1) / rows);
                if (left < here) {
                    found = first + i, from = b + (int64_t)left * rows, to = e;
                    break;
                }
                left -= here;
            }
        }
        expert = __builtin_amdgcn_readlane(found, owner);
        place = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)from, owner);  // (places are below 2^31)
        count = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)to, owner) - place;
    }
};
// the row of a that place p reads
__device__ __forceinline__ int64_t row_of_place(const MatmulFp8Params& p, int64_t place) {
    if (p.order == nullptr) return min(place, p.a_rows - 1);
    return min((int64_t)((uint32_t)max(((GlobalIndex)p.order)[place], 0) / (uint32_t)p.divisor), p.a_rows - 1);
}

// Eight elements as they lie in memory, at any address: loads that are all to be on their way before the first is looked at are of these, since a choice of the type at each
// load8 has it waited for there.
struct Raw8 {
    uint4_t lo, hi;  // (hi: of fp32 alone)
};
__device__ __forceinline__ Raw8 load_raw8(const void* base, int64_t idx, int dtype) {
    Raw8 r = {};
    if (dtype == HIPATTN_F32)
        __builtin_memcpy(&r, (const float*)base + idx, 32);
    else
        __builtin_memcpy(&r.lo, (const uint16_t*)base + idx, 16);
    return r;
}
__device__ __forceinline__ Float8 float8_of(const Raw8& r, int dtype) {
    Float8 y;
    if (dtype == HIPATTN_F32) {
#pragma unroll
        for (int e = 0; e < 8; e++) y.v[e] = __uint_as_float(e < 4 ? r.lo[e] : r.hi[e - 4]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint16_t v = (uint16_t)(r.lo[e >> 1] >> (16 * (e & 1)));
            y.v[e] = dtype == HIPATTN_F16 ? f16_bits_to_float(v) : bf16_bits_to_float(v);
        }
    }
    return y;
}

// swish with the exponential and the reciprocal instruction: a unit in the last place off each, and the exponent x log2 e is rounded to 24 bits: for negative x
// some (1.2 |x| + 8) 2^-24 of the value, which is |x| exp(-|x|) there
__device__ __forceinline__ float gated(float x, int activation) {
    if (activation == HIPOPS_GLU_SWISH) return x * __builtin_amdgcn_rcpf(1.0f + __expf(-x));
    return activate(x, activation, 1.0f);
}
__device__ __forceinline__ float finished_fp8(const MatmulFp8Params& p, float sum, int64_t to, int64_t column) {
    if (p.bias != nullptr) sum += load_scalar(p.bias, column, p.c_dtype);
    if (p.residual != nullptr) sum += load_scalar(p.residual, to, p.c_dtype);
    return sum;
}

// Eight elements to any address, rounded to nearest even.
__device__ __forceinline__ void store_loose8(void* base, int64_t to, int dtype, const float* y) {
    typedef float float2_t __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    if (dtype == HIPATTN_F32) {
        __builtin_memcpy((float*)base + to, y, 32);
        return;
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2_t pair = {y[2 * i], y[2 * i + 1]};
        w[i] = dtype == HIPATTN_F16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, half2_t)) : __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, bf16x2_t));
    }
    __builtin_memcpy((uint16_t*)base + to, w, 16);
}
// Eight neighbouring results from element `to` of c on, with the residual if there is one.  (Rows may begin anywhere: copies of eight elements
// are whatever loads and stores the hardware has for that.)
__device__ __forceinline__ void store8_fp8(const MatmulFp8Params& p, int64_t to, float (&y)[8]) {
    if (p.c_dtype == HIPATTN_F32) {
        if (p.residual != nullptr) {
            float r[8];
            __builtin_memcpy(r, (const float*)p.residual + to, 32);
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] += r[e];
        }
        store_loose8(p.c, to, HIPATTN_F32, y);
        return;
    }
    if (p.residual != nullptr) {
        uint16_t r[8];
        __builtin_memcpy(r, (const uint16_t*)p.residual + to, 16);
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] += p.c_dtype == HIPATTN_F16 ? f16_bits_to_float(r[e]) : bf16_bits_to_float(r[e]);
    }
    store_loose8(p.c, to, p.c_dtype, y);
}
// `columns` (1 to 8) of them
__device__ __forceinline__ void store_columns_fp8(const MatmulFp8Params& p, int64_t to, int columns, float (&y)[8]) {
    if (columns == 8) {
        store8_fp8(p, to, y);
        return;
    }
    for (int e = 0; e < columns; e++) {
        const float r = p.residual != nullptr ? load_scalar(p.residual, to + e, p.c_dtype) : 0.0f;
        float v = 0.0f;
#pragma unroll
        for (int u = 0; u < 8; u++) v = u == e ? y[u] : v;
        store_scalar(p.c, to + e, p.c_dtype, v + r);
    }
}

// ---- how a product is laid out over workgroups ----------------------------------------------------
enum Fp8Tile { kFp8Tile32, kFp8Tile64, kFp8Tile128, kFp8Tile256, kFp8Any32, kFp8Any128, kFp8Few };
constexpr int kFp8DeepStages = 4;  // of 128 bytes of k, that tiles of 256 rows take at least
struct Fp8Plan {
    Fp8Tile tile;
    int parts;  // of k, whose sums meet in the workspace
};
struct Fp8Grid {
    int tiles_m, tiles_n, parts;  // (experts: tiles_m counts what there may be)
    int group_rows;               // tiles of m that are gone through before the next tile of n
    int rotate;                   // tiles begin at different stages of k
    float* sums;                  // null, or [parts][m][sums_stride]
    int64_t sums_stride;
};
// The columns of a gated unit's tiles: 64, or less where the second half, which begins at row `width` of the weights, passes into its next block of scales: a
// tile's columns have one scale in each half.  Widths of whole 64 have two tiles for 128 columns, others three.
struct GatedTiles {
    int64_t width;
    int rest, next;  // columns beyond whole 128; where the second half's next block begins, of 128
    __host__ __device__ explicit GatedTiles(int64_t width) : width(width), rest((int)(width % kFp8Block)), next((kFp8Block - rest) % kFp8Block) {}
    __host__ __device__ bool whole() const { return rest % 64 == 0; }
    __host__ __device__ int begin(int part) const { return part == 0 ? 0 : part == 3 ? kFp8Block : (part == 1) == (next < 64) ? next : 64; }
    __host__ __device__ int64_t count() const {
        if (whole()) return width / 64;
        return 3 * (width / kFp8Block) + 1 + (begin(1) < rest) + (begin(2) < rest);
    }
    __device__ void find(int tile, int64_t& first, int64_t& end) const {
        if (whole()) {
            first = 64 * (int64_t)tile, end = first + 64;
        } else {
            const int64_t block = kFp8Block * (int64_t)(tile / 3);
            first = block + begin(tile % 3), end = min(block + begin(tile % 3 + 1), width);
        }
    }
};
// activation rows and columns of the product (gated: half of them results) that a tile takes
constexpr int fp8_tile_rows(Fp8Tile t) { return t == kFp8Tile32 || t == kFp8Any32 ? 32 : t == kFp8Tile64 ? 64 : t == kFp8Tile256 ? 256 : 128; }
constexpr int fp8_tile_columns(Fp8Tile t) { return t == kFp8Tile256 ? 256 : 128; }
template <bool kExperts>
hipError_t launch_matmul_fp8_few(const MatmulFp8Params& p, bool exact, hipStream_t stream);  // matmul_fp8_few.hip
template <bool kExperts>
hipError_t launch_matmul_fp8_deep(const MatmulFp8Params& p, hipStream_t stream);  // matmul_fp8_deep.hip
template <bool kExperts>
hipError_t launch_matmul_fp8_tiles(const MatmulFp8Params& p, const Fp8Plan& plan, bool exact, void* workspace, hipStream_t stream);  // matmul_fp8_tiles.hpp
// tiles of `rows` rows that the places of an experts' product can come to
inline int64_t most_expert_tiles(const MatmulFp8Params& p, int64_t rows) {
    const int64_t places = p.last_place - p.first_place;
    return (places < p.experts ? places : (int64_t)p.experts) + places / rows;
}

// codes of `rows` rows as quantize_fp8 makes them; of an experts' product, those of places between *row_begin and *row_limit alone (row r is place row_first + r)
struct QuantizeFp8Params {
    const void* x;
    const void* gamma;
    uint8_t* codes;
    float* scales;
    int64_t rows, width, x_row_stride, scale_row, scale_block;
    int x_dtype, gamma_dtype, activation, gate_first;
    float eps;
    const int32_t* row_begin;  // on the device, with row_limit; both null: all rows
    const int32_t* row_limit;
    int64_t row_first;
};
hipError_t launch_quantize_fp8(int source, const QuantizeFp8Params& p, hipStream_t stream);  // quantize_fp8.hip

}  // namespace hipops
