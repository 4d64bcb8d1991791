// Products of e4m3 codes with many rows (hipops_matmul_fp8, hipops_matmul_fp8_experts): tiles of 256 x 256 by workgroups that stay.
//
//   c[i, j] = sum_b a_scale[i, b] b_scale[j / 128, b] (sum_{l in b} a[i, l] b[j, l]) + bias[j] + residual[i, j]
// Bound by the matrix cores, and next to them by LDS: a stage of 128 bytes of k is 2,048 cycles of products on each SIMD, 1,536 of reads and 512
// of writes of the one LDS.  So both have to run all the time:
// * One workgroup a compute unit goes from tile to tile; what it loads runs a stage and a half ahead of what it multiplies, across tiles, so that
//   the first loads of a tile are not waited for.
// * Activations come in halves of a stage (four of them in LDS), weights in stages (two); a wavefront reads a stage's weight fragments, 32
//   registers, during the second half of the stage before.  That frees their room a stage early, and no stage begins with a burst of reads.
// * The two barriers of a stage stand ahead of the last products of a half, whose operands are in registers: the first fragment of the next half
//   is read behind the barrier while those run.
// * A block's sums are joined to the results by the fma of the group of products behind them, so that no product is waited for.
// A wavefront's columns are dealt out so that a lane ends with twice eight neighbouring ones of a row (gated: eight), stored from the registers.
// Where the experts' tiles lie is kept in LDS: until[], first and end of each expert.
//
// Measured: 8,001 x 6,144 x 4,096 in 193 - 207 us (2.0 PFLOP/s, matrix cores 45 % busy at the clock that the power limit leaves), 8,192 rows of 8 experts on
// 28,672 x 4,096 (gated) 1,100 (1.75).  A stage takes 1.53 - 1.66 us: the same products, reads and barriers without loads 1.43, the loads alone 1.0.  A tile
// has some 12 us besides, 6.5 of them its stores, which all compute units make at about the same time (half of the stores: half of that).  Not
// kept: stores during the last stage (a branch in every step of a stage costs more: 225 against 197 us; a form of the stage of its own
// spills), stores around the caches (270 against 261), workgroups that begin some us apart (the same), fewer loads waited for behind a tile's stores (the same).
#include "ops/fp8.hpp"
#include "ops/fp8_loads.hpp"

namespace hipops {

namespace {

constexpr int kTile = 256, kHalfBytes = 128 * kFp8Block, kStageOfB = 256 * kFp8Block;
constexpr int kBAt = 4 * kHalfBytes, kScalesAt = kBAt + 2 * kStageOfB, kScaleBytes = 1536;  // (activations' 256, weights' two, the idle wavefronts' room)
// where the rows of a tile's activations begin, their scales and the weights' two: of the tile that is loaded, and of the next
constexpr int kTableAt = kScalesAt + 4 * kScaleBytes, kTableBytes = 4 * (2 * kTile + 64), kExpertsAt = kTableAt + 2 * kTableBytes;
constexpr int kMostExperts = 1024;  // whose tiles up to and with it, first place and end are kept behind that
template <bool kExperts>
constexpr int kLdsBytes = kExpertsAt + (kExperts ? 3 * 4 * kMostExperts : 0);
constexpr int kHalfLoads = 2, kBLoads = 4, kInFlight = 2 * kHalfLoads + kBLoads + 1;  // of a wavefront behind the ones that a barrier waits for
constexpr int kTM = 8, kTN = 4;

__device__ __forceinline__ int swizzle_a(int row) { return (row >> 1) & 7; }
// (a weight fragment's rows are 16 (f / 4) + 4 j + f % 4)
__device__ __forceinline__ int swizzle_b(int row) { return ((row >> 3) & 6) | ((row >> 1) & 1); }

// the kernel's arguments, read again where they are used: what a tile's beginning and end need holds no registers over the products
struct Arguments {
    MatmulFp8Params p;
    Fp8Grid g;
};
__device__ __forceinline__ Arguments arguments() {
    struct Raw {
        uint32_t w[sizeof(Arguments) / 4];
    } raw;
    typedef const __attribute__((address_space(4))) uint32_t* Words;
    Words from = (Words)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(from));
#pragma unroll
    for (size_t i = 0; i < sizeof(Arguments) / 4; i++) raw.w[i] = from[i];
    return __builtin_bit_cast(Arguments, raw);
}

// the same for all lanes, and in scalar registers
__device__ __forceinline__ int scalar(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ const uint8_t* scalar(const uint8_t* v) {
    const uintptr_t u = (uintptr_t)v;
    return (const uint8_t*)((uintptr_t)(uint32_t)scalar((int)(uint32_t)u) | (uintptr_t)(uint32_t)scalar((int)(uint32_t)(u >> 32)) << 32);
}

// Addresses in LDS that are worked out at each use: the sums of what is the same for all lanes with what is not would each take a register over
// the whole loop, and there are none.
__device__ __forceinline__ int plus(int same, int lanes) {
    int r;
    asm volatile("v_add_u32 %0, %1, %2" : "=v"(r) : "s"(same), "v"(lanes));
    return r;
}
__device__ __forceinline__ int other_piece(int at) {
    int r;
    asm volatile("v_xor_b32 %0, 64, %1" : "=v"(r) : "v"(at));
    return r;
}

// Eight neighbouring numbers of a type, at any address of global memory (which the compiler cannot tell from an address that came as numbers).
typedef __attribute__((address_space(1))) uint8_t* Global;
typedef uint4_t __attribute__((aligned(2))) Loose;
typedef __attribute__((address_space(1))) Loose* GlobalLoose;
template <int kOut>
__device__ __forceinline__ void store8_as(Global to, const float* y) {
    typedef float float2_t __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    if constexpr (kOut == HIPATTN_F32) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            uint4_t w;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = __float_as_uint(y[4 * h + e]);
            *(GlobalLoose)(to + 16 * h) = w;
        }
    } else {
        uint4_t w;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2_t pair = {y[2 * i], y[2 * i + 1]};
            w[i] = kOut == HIPATTN_F16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, half2_t)) : __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, bf16x2_t));
        }
        *(GlobalLoose)to = w;
    }
}
template <int kOut>
__device__ __forceinline__ void load8_as(Global from, float* y) {
    static_assert(kOut != HIPATTN_F32, "bias and residual: of dense products alone, which have 16 bits here");
    const uint4_t w = *(GlobalLoose)from;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint16_t v = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
        y[e] = kOut == HIPATTN_F16 ? f16_bits_to_float(v) : bf16_bits_to_float(v);
    }
}

struct Place {  // of a tile: its first row (place), how many there are from it on, its first column
    int m0, count, n0;
};

template <bool kExperts, int kOut>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void matmul_fp8_deep_kernel(Arguments) {
    __shared__ __attribute__((aligned(128))) uint8_t lds[kLdsBytes<kExperts>];
    lds_byte* const base = (lds_byte*)lds;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = wave >> 2, wn = wave & 3, frow = lane & 15, quarter = lane >> 4;

    // Workgroups go to the eight XCDs in turn: each XCD takes a run of the tiles, which come in groups of rows so that those that run together
    // share rows of both operands in its L2.
    int tiles_m, tiles, first_tile, stages, is_gated, to_second, to_third;
    {
        const Arguments a = arguments();
        tiles_m = a.g.tiles_m;
        if constexpr (kExperts) {
            const ExpertTiles<true> all(a.p, kTile, lane);
            tiles_m = min(all.total, tiles_m);  // (more only where begins overlap)
            if (wave == 0) {
                int* const until = (int*)(lds + kExpertsAt);
                int tiles = all.until - all.tiles;
                for (int i = 0; i < all.each && all.first + i < a.p.experts; i++) {
                    const int e = all.first + i;
                    const int64_t b = all.place_at(a.p, e, a.p.first_place), end = all.place_at(a.p, e + 1, b);
                    tiles += (int)((end - b + kTile - 1) / kTile);
                    until[e] = tiles, until[kMostExperts + e] = (int)b, until[2 * kMostExperts + e] = (int)end;
                }
            }
            __syncthreads();
        }
        const int total = tiles_m * a.g.tiles_n, run = (total + 7) >> 3;
        first_tile = scalar(((int)blockIdx.x & 7) * run);
        tiles = scalar(min(run, total - first_tile));  // of this XCD
        stages = (int)(a.p.k / kFp8Block);
        is_gated = a.p.gated;
        // A wavefront's four loads of eight weight rows: a run of the first half of a wavefront's columns (the gate's) and one of the second (what they
        // meet), and the eight rows behind each.
        to_second = (int)(is_gated ? (a.p.n / 2) * a.p.ldb * (a.p.gate_first ? 1 : -1) : 32 * a.p.ldb);
        to_third = (int)(8 * a.p.ldb);
    }
    const int step = (int)gridDim.x >> 3;
    int mine = (int)blockIdx.x >> 3;  // the tile that is loaded, of the XCD's
    if (mine >= tiles) return;

    // ---- what is loaded ----
    // Lane l loads piece (l % 8) ^ swizzle(row) of row l / 8 of a load's eight.
    struct Source {
        const uint8_t *a, *b, *s;
    } from, then;  // of the stage that is loaded; of the next tile's first
    Place here, next;  // of the tile that is multiplied, and the one behind it
    int stage = 0, table = kTableAt;
    const int eighth = lane >> 3, eighth4 = 4 * eighth, lane4 = 4 * lane, frow4 = 4 * frow;
    const int a_piece = 16 * ((lane & 7) ^ swizzle_a(eighth));  // (the second load of eight rows: another by 64)
    uint32_t b_offset, scale_step;
    {
        const Arguments arg = arguments();
        b_offset = (uint32_t)(eighth * arg.p.ldb) + 16 * ((lane & 7) ^ swizzle_b(32 * wave + eighth));  // (the second sixteen rows: another by 32, for rows at multiples of 64)
        scale_step = wave < 4 ? (uint32_t)(4 * arg.p.a_scale_block) : 4u;
    }
    const auto open = [&](int index, int to) __attribute__((always_inline)) {
        const Arguments arg = arguments();
        const MatmulFp8Params& p = arg.p;
        int row = threadIdx.x;
        asm volatile("" : "+v"(row));  // (as the arguments)
        const int n = (int)p.n, width = p.gated ? n / 2 : n, gate = p.gate_first ? 0 : width, lane = row & 63;
        index += first_tile;
        const int in_group = arg.g.group_rows * arg.g.tiles_n, group = index / in_group;
        const int rows_here = min(arg.g.group_rows, tiles_m - group * arg.g.group_rows), in = index - group * in_group;
        const int m_tile = __builtin_amdgcn_readfirstlane(group * arg.g.group_rows + in % rows_here);
        next.n0 = __builtin_amdgcn_readfirstlane(in / rows_here) * (p.gated ? kTile / 2 : kTile);
        int expert = 0;
        if constexpr (kExperts) {
            const int* const until = (const int*)(lds + kExpertsAt);
            for (int e = lane; e < p.experts + lane; e += 64)  // (every lane as often) the experts whose tiles end before this one
                expert += __builtin_popcountll(__ballot(e < p.experts && until[min(e, kMostExperts - 1)] <= m_tile));
            const int before = expert > 0 ? until[expert - 1] : 0;
            next.m0 = scalar(until[kMostExperts + expert] + (m_tile - before) * kTile);
            next.count = scalar(until[2 * kMostExperts + expert]) - next.m0;
        } else {
            next.m0 = m_tile * kTile;
            next.count = (int)p.m - next.m0;
        }
        const int first_row = kExperts && p.order != nullptr ? 0 : next.m0;
        // Row 16 q + 4 j + r of a wavefront's 64 in LDS is column 8 q + 4 (j % 2) + r of its first 32 (gated: the gate's) for j below 2, of its other 32 (what
        // they meet) for the others: a lane ends with twice eight neighbouring columns, and the lanes of a row with twice 32.
        const int b_row = (p.gated ? gate + next.n0 + 32 * (wave >> 1) : min(next.n0 + 64 * (wave >> 1), n - 64)) + 16 * (wave & 1);
        then.a = scalar(p.a + first_row * p.lda);
        then.b = scalar(p.b + ((int64_t)expert * n + b_row) * p.ldb);
        uint32_t* const words = (uint32_t*)(lds + to);
        if (wave < 4) {
            const int at = next.m0 + min(row, next.count - 1);
            const int64_t source = kExperts ? row_of_place(p, at) : at;
            words[row] = (uint32_t)((source - first_row) * p.lda);
            words[kTile + row] = (uint32_t)(4 * source * p.a_scale_row);
            then.s = scalar((const uint8_t*)p.a_scales);
        } else {
            const int other = p.gated ? width - gate : kFp8Block;  // (the second half's columns, or the rows that the gate meets)
            const int second = row & 1;
            if (wave == 4) words[2 * kTile + lane] = (uint32_t)(4 * (min((p.gated ? (second ? other : gate) : second * other) + next.n0, n - 1) / kFp8Block) * stages);
            then.s = scalar((const uint8_t*)(p.b_scales + (int64_t)expert * ((n + kFp8Block - 1) / kFp8Block) * stages));
        }
    };
    // What the next loads begin at is read from the table some time ahead.
    uint32_t a_row[kHalfLoads], s_offset;
    const auto prepare = [&](int h) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kHalfLoads; i++) {
            const int row = 8 * (wave * kHalfLoads + i);  // in the half: 64 rows of each row of wavefronts
            a_row[i] = *(const uint32_t*)(lds + plus(table + 4 * ((row >> 6) * 128 + 64 * h + (row & 63)), eighth4));
        }
        if (h == 0) s_offset = *(const uint32_t*)(lds + plus(table + 4 * kTile + 256 * min(wave, 4), lane4));
    };
    const auto load_a = [&](int h, int u) __attribute__((always_inline)) {  // with the first half: the scales
#pragma unroll
        for (int i = 0; i < kHalfLoads; i++)
            load_to_lds_16(from.a, a_row[i] + (a_piece ^ (64 * i)), base + ((u & 1) * 2 + h) * kHalfBytes + 1024 * (wave * kHalfLoads + i));
        if (h == 0) load_to_lds_4(from.s, s_offset, base + kScalesAt + (u & 3) * kScaleBytes + 256 * min(wave, 5));
    };
    const auto load_b = [&](int u) __attribute__((always_inline)) {
        lds_byte* const to = base + kBAt + (u & 1) * kStageOfB + 1024 * wave * kBLoads;
        load_to_lds_16(from.b, b_offset, to);
        load_to_lds_16(from.b + to_second, b_offset, to + 1024);
        load_to_lds_16(from.b + to_third, b_offset ^ 32, to + 2048);
        load_to_lds_16(from.b + to_second + to_third, b_offset ^ 32, to + 3 * 1024);
    };
    // the next stage, of the next tile where this one has ended; behind the last tile its last stage again, which nobody reads
    const auto advance = [&]() __attribute__((always_inline)) {
        if (stage + 1 < stages) {
            stage++;
            from.a += kFp8Block, from.b += kFp8Block, from.s += scale_step;
        } else if (mine + step < tiles) {
            mine += step;
            stage = 0;
            from = then;
            table = 2 * kTableAt + kTableBytes - table;
        }
    };

    // ---- what is multiplied ----
    float4_t acc[kTN][kTM], sum[kTN];
    int8v_t w[2][kTN], x[2];  // w: of the stage that is multiplied, and of the next
    float a_scale[2];
    const auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kTN; j++)
#pragma unroll
            for (int i = 0; i < kTM; i++) acc[j][i] = (float4_t){0.0f, 0.0f, 0.0f, 0.0f};
    };
    const int x_at = (64 * wm + frow) * kFp8Block + 16 * (quarter ^ swizzle_a(frow));  // (its second piece: another by 64)
    const int b_row = 64 * wn + 16 * (frow >> 2) + (frow & 3), w_at = b_row * kFp8Block + 16 * (quarter ^ swizzle_b(b_row));
    const auto fragment = [&](int at, int where) __attribute__((always_inline)) {
        return joined(*(const uint4_t*)(lds + at + where), *(const uint4_t*)(lds + at + other_piece(where)));
    };
    const auto read_x = [&](int u, int i) __attribute__((always_inline)) {  // activation rows 16 i + ... of the wavefront's in stage u
        x[i & 1] = fragment(((u & 1) * 2 + i / 4) * kHalfBytes + 16 * (i & 3) * kFp8Block, x_at);
        a_scale[i & 1] = *(const float*)(lds + plus(kScalesAt + (u & 3) * kScaleBytes + 512 * wm, frow4) + 64 * i);
    };
    const auto read_w = [&](int8v_t (&to)[kTN], int u, int j) __attribute__((always_inline)) {
        to[j] = fragment(kBAt + (u & 1) * kStageOfB + 4 * j * kFp8Block, w_at);
    };
    const auto barrier = []() __attribute__((always_inline)) { barrier_keeping<kInFlight>(); };

    open(mine, table);
    from = then, here = next;
    __syncthreads();
    load_b(0);
    prepare(0);
    load_a(0, 0);
    prepare(1);
    load_a(1, 0);
    advance();
    load_b(1);
    prepare(0);
    load_a(0, 1);
    barrier();  // the first stage's weights and the first half of its activations
#pragma unroll
    for (int j = 0; j < kTN; j++) read_w(w[0], 0, j);
    prepare(1);
    barrier();  // (which are in registers now)
    load_a(1, 1);
    advance();
    load_b(2);
    read_x(0, 0);
    clear();
    int left = stages, tile = mine;  // of the tile that is multiplied
    const auto multiply = [&](int u, const int8v_t (&now)[kTN], int8v_t (&next_w)[kTN]) __attribute__((always_inline)) {
        const float* const scales = (const float*)(lds + kScalesAt + (u & 3) * kScaleBytes) + 256;
        // (columns of one wavefront share a block; of a gated unit, each half of them)
        const float scale_lo = scales[is_gated ? 0 : wn >> 1], scale_hi = scales[is_gated ? 1 : wn >> 1];
        float lo = 0.0f, hi = 0.0f;
        const bool busy = 128 * wm < here.count;  // (a wavefront without rows in the tile multiplies nothing)
#pragma unroll
        for (int i = 0; i < kTM; i++) {
            if (i == 2) prepare(0);
            if (i == 3) {
                barrier();  // the second half of the activations, and the next stage's weights
                load_a(0, u + 2);
                if (stage + 1 == stages && mine + step < tiles) open(mine + step, 2 * kTableAt + kTableBytes - table);
            }
            if (i == 6) prepare(1);
            if (i == 7) {
                barrier();  // the next stage's first half
                load_a(1, u + 2);
                advance();
                load_b(u + 3);
            }
            const float scale = a_scale[i & 1];
            if (i < 7)
                read_x(u, i + 1);
            else
                read_x(u + 1, 0);
            if (i == 4) read_w(next_w, u + 1, 0);
            if (i == 5) read_w(next_w, u + 1, 1);
            if (i == 6) {
                read_w(next_w, u + 1, 2);
                read_w(next_w, u + 1, 3);
            }
            if (busy) {
#pragma unroll
                for (int j = 0; j < kTN; j++) {
                    const float4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
                    if (i > 0) {
#pragma unroll
                        for (int r = 0; r < 4; r++) acc[j][i - 1][r] = fmaf(sum[j][r], j < kTN / 2 ? lo : hi, acc[j][i - 1][r]);
                        asm volatile("" : "+v"(acc[j][i - 1]));  // (here, and not behind the branches that follow)
                    }
                    sum[j] = mma_fp8_16(now[j], x[i & 1], zero);
                    __builtin_amdgcn_sched_barrier(0);  // (the compiler's own order has sums waited for)
                }
            }
            lo = scale * scale_lo, hi = scale * scale_hi;
            __builtin_amdgcn_sched_barrier(0);
        }
        if (!busy) return;
#pragma unroll
        for (int j = 0; j < kTN; j++) {
#pragma unroll
            for (int r = 0; r < 4; r++) acc[j][kTM - 1][r] = fmaf(sum[j][r], j < kTN / 2 ? lo : hi, acc[j][kTM - 1][r]);
            asm volatile("" : "+v"(acc[j][kTM - 1]));
        }
    };
    // the end of a tile; false where it was the last.  Register r of acc[j][i]: activation row 16 i + lane % 16 of the wavefront's, column
    // 8 (lane / 16) + 4 (j % 2) + r of half j / 2 of its columns
    const auto finish = [&]() __attribute__((always_inline)) -> bool {
        const Arguments arg = arguments();
        const MatmulFp8Params& p = arg.p;
        constexpr int kSize = kOut == HIPATTN_F32 ? 4 : 2;
        const int width = (int)(is_gated ? p.n / 2 : p.n), column = here.n0 + (is_gated ? 32 : 64) * wn + 8 * quarter;
        if (column < width) {  // (widths are whole runs of a wavefront's columns)
            const int64_t first = (here.m0 - p.first_place + 128 * wm + frow) * p.ldc + column;
            Global to = (Global)p.c + kSize * first;
            const int64_t step_of_i = 16 * kSize * p.ldc;
            const int rows = here.count - 128 * wm - frow;
            if (is_gated) {
#pragma unroll
                for (int i = 0; i < kTM; i++) {
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] = gated(acc[e >> 2][i][e & 3], p.activation) * acc[2 + (e >> 2)][i][e & 3];
                    if (16 * i < rows) store8_as<kOut>(to, y);
                    to += step_of_i;
                }
            } else {
                float bias[16];
#pragma unroll
                for (int e = 0; e < 16; e++) bias[e] = 0.0f;
                if constexpr (!kExperts) {
                    if (p.bias != nullptr) {
                        load8_as<kOut>((Global)p.bias + kSize * column, bias);
                        load8_as<kOut>((Global)p.bias + kSize * (column + 32), bias + 8);
                    }
                }
                Global other = kExperts || p.residual == nullptr ? nullptr : (Global)p.residual + kSize * first;
#pragma unroll
                for (int i = 0; i < kTM; i++) {
                    if (16 * i < rows) {
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            float y[8];
#pragma unroll
                            for (int e = 0; e < 8; e++) y[e] = acc[2 * h + (e >> 2)][i][e & 3] + bias[8 * h + e];
                            if constexpr (!kExperts) {
                                if (other != nullptr) {
                                    float r[8];
                                    load8_as<kOut>(other + 32 * kSize * h, r);
#pragma unroll
                                    for (int e = 0; e < 8; e++) y[e] += r[e];
                                }
                            }
                            store8_as<kOut>(to + 32 * kSize * h, y);
                        }
                    }
                    to += step_of_i;
                    if (other != nullptr) other += step_of_i;
                }
            }
        }
        tile += step;
        here = next;
        left = stages;
        clear();
        return tile < tiles;
    };
    for (int u = 0;; u += 2) {
        multiply(u, w[0], w[1]);
        if (--left == 0 && !finish()) break;
        multiply(u + 1, w[1], w[0]);
        if (--left == 0 && !finish()) break;
    }
    // (what was loaded behind the last stage may not land in the LDS of a workgroup that comes after this one)
    __builtin_amdgcn_s_waitcnt(0x0070);
}

}  // namespace

template <bool kExperts>
hipError_t launch_matmul_fp8_deep(const MatmulFp8Params& p, hipStream_t stream) {
    Fp8Grid g{};
    g.parts = 1;
    g.group_rows = 8;
    const int64_t columns = p.gated ? kTile / 2 : kTile;
    g.tiles_m = (int)(kExperts ? most_expert_tiles(p, kTile) : (p.m + kTile - 1) / kTile);
    g.tiles_n = (int)(((p.gated ? p.n / 2 : p.n) + columns - 1) / columns);
    const int64_t tiles = (int64_t)g.tiles_m * g.tiles_n, grid = 8 * ((tiles < 256 ? tiles + 7 : 256) / 8);
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(512), 0, stream, Arguments{p, g}); };
    if (p.c_dtype == HIPATTN_F16) {
        launch(matmul_fp8_deep_kernel<kExperts, HIPATTN_F16>);
    } else if (p.c_dtype == HIPATTN_BF16) {
        launch(matmul_fp8_deep_kernel<kExperts, HIPATTN_BF16>);
    } else {  // (of experts: what becomes codes.  Results in fp32 are exact products, which these tiles do not have)
        if constexpr (!kExperts) return hipErrorInvalidValue;
        if constexpr (kExperts) launch(matmul_fp8_deep_kernel<true, HIPATTN_F32>);
    }
    return hipGetLastError();
}
template hipError_t launch_matmul_fp8_deep<false>(const MatmulFp8Params&, hipStream_t);
template hipError_t launch_matmul_fp8_deep<true>(const MatmulFp8Params&, hipStream_t);

}  // namespace hipops
