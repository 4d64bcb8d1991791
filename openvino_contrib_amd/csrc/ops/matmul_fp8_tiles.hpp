// Products of e4m3 codes in tiles through LDS (hipops_matmul_fp8, hipops_matmul_fp8_experts).
//
//   c[i, j] = sum_b a_scale[i, b] b_scale[j / 128, b] (sum_{l in b} a[i, l] b[j, l]) + bias[j] + residual[i, j]
// v_mfma_f32_16x16x128_f8f6f4 sums a block of 128 from zero; an fma joins it to the result with the product of the block's scales.  Weights are the
// instruction's first operand, so a lane's four results are neighbouring columns of one activation row: one number scales all four.
//
// A gated unit's tile ends where either half's block of scales does (GatedTiles): 8,192 rows on 64 experts of 4,060 x 4,096 495 us, of 4,096 x 4,096 in tiles of 256
// rows 330.  Rows at any address: through registers, eight wavefronts for 128 rows (8,192 x 6,144 x 4,099 668 us, with four 717).
// Measured (us): 64 x 28,672 x 4,096 28.8 (weights at 4.1 TB/s: 224 tiles for 256 compute units, 0.75 us a stage), 32 rows 26.1; 64 tokens' 512 rows on 64
// experts 187 (the weights at 5.8 TB/s); rings of 4, 5 and 6 stages the same as 3; tiles of 128 rows with eight wavefronts 128 -> 137 (2,300 x 8,192 x 4,096).
// A stage is 128 bytes of k: the rows, and the block's scales, loaded straight to LDS while the one or two before it are multiplied (rows at any
// address: through registers).  Experts: the tiles of all experts' rows in one launch; which expert a workgroup's is it adds up itself.
#pragma once

#include "ops/fp8.hpp"
#include "ops/fp8_loads.hpp"

namespace hipops {

namespace {

constexpr int kStageBytes = 128;  // of a row in a stage
static_assert(kStageBytes == kFp8Block, "a stage is a block of scales");
// Rows lie side by side in a stage, their 16-byte pieces permuted so that the sixteen rows that a fragment's read touches at a time (one
// piece of each) lie on all 64 banks.
__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }

// kBM activation rows x kBN weight rows, kWM x kWN wavefronts, kRing stages.
// kDirect: rows at multiples of 16 bytes, k too, straight to LDS; otherwise any rows and k, through registers, one stage ahead.
// kExact: through fp16 copies of the codes.
template <int kBM, int kBN, int kWM, int kWN, int kRing, bool kDirect, bool kExperts, bool kExact>
__global__ __launch_bounds__(64 * kWM * kWN) __attribute__((amdgpu_waves_per_eu(kWM * kWN == 8 ? 2 : 1, 2))) void matmul_fp8_tiles_kernel(MatmulFp8Params p, Fp8Grid g) {
    constexpr int kWaves = kWM * kWN, kRows = kBM + kBN;
    constexpr int kTM = kBM / kWM / 16, kTN = kBN / kWN / 16;
    constexpr int kPieces = kStageBytes / 16, kRowsPerLoad = 64 / kPieces;
    constexpr int kLoads = kRows / kRowsPerLoad / kWaves;  // of a wavefront for a stage, and one more of scales
    // behind a stage's rows: the activations' scales (64 lanes at a time), the weights' two, and room for the wavefronts that have none to load
    constexpr int kScaleWaves = (kBM + 63) / 64, kScalesAt = kRows * kStageBytes, kSlot = kScalesAt + 256 * (kScaleWaves + 2);
    static_assert(kBN == kFp8Block, "a block of scales; of a gated unit: 64 columns of each half");
    static_assert(kRows % (kRowsPerLoad * kWaves) == 0 && kBM % kRowsPerLoad == 0 && kTM > 0 && kTN > 1 && kTN % 2 == 0, "whole loads and tiles");
    static_assert(kRing >= 2 && (kDirect || kRing == 2) && kWaves > kScaleWaves, "the stage that is read, and those on their way");
    constexpr int kOutColumns = 16 * kTN, kOutRow = 4 * kOutColumns + 16, kOutBytes = 16 * kOutRow;
    constexpr int kLds = kRing * kSlot > kWaves * kOutBytes ? kRing * kSlot : kWaves * kOutBytes;
    __shared__ __attribute__((aligned(128))) uint8_t lds[kLds];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t width = p.gated ? p.n / 2 : p.n;

    // Workgroups go to the eight XCDs in turn: each takes a run of the tiles, which come in groups of rows so that those that run together
    // share rows of both operands in the XCD's L2.
    int part = 0, tile, expert = 0;
    int64_t m0, count;  // the first row (place) and how many there are from it on
    int64_t n0, n_end;  // the first column of the result, and the one behind the last
    const auto spread = [&](int tiles_m) __attribute__((always_inline)) -> int {  // which tile of m, of a total that may be known here only
        const int tiles = tiles_m * g.tiles_n, total = tiles * g.parts, run = (total + 7) >> 3, at = (int)blockIdx.x >> 3;
        const int index = __builtin_amdgcn_readfirstlane(((int)blockIdx.x & 7) * run + at);
        if (at >= run || index >= total) return -1;
        part = index / tiles;
        tile = index - part * tiles;
        const int in_group = g.group_rows * g.tiles_n, group = tile / in_group;
        const int rows_here = min(g.group_rows, tiles_m - group * g.group_rows), in = tile - group * in_group;
        const int column_tile = __builtin_amdgcn_readfirstlane(in / rows_here);
        n0 = (int64_t)column_tile * kBN, n_end = p.n;
        if (p.gated) GatedTiles(width).find(column_tile, n0, n_end);
        return __builtin_amdgcn_readfirstlane(group * g.group_rows + in % rows_here);
    };
    if constexpr (kExperts) {
        const ExpertTiles<true> tiles(p, kBM, lane);
        const int mine = spread(min(tiles.total, g.tiles_m));  // (more only where begins overlap)
        if (mine < 0) return;
        tiles.find(p, mine, kBM, lane, expert, m0, count);
    } else {
        const int mine = spread(g.tiles_m);
        if (mine < 0) return;
        m0 = (int64_t)mine * kBM;
        count = p.m - m0;
    }
    const int stages = (int)((p.k + kStageBytes - 1) / kStageBytes);
    const int first = (int)((int64_t)stages * part / g.parts), last = (int)((int64_t)stages * (part + 1) / g.parts);

    // Weight rows of a wavefront's columns lie side by side; of a gated unit, half of them the gate's and half those that they meet.
    constexpr int kOfWave = kBN / kWN;
    const int64_t gate = p.gate_first ? 0 : width, up = p.gate_first ? width : 0;
    const auto weight_row = [&](int r) __attribute__((always_inline)) -> int64_t {
        if (!p.gated) return min(n0 + r, p.n - 1);
        const int of = r / kOfWave, in = r % kOfWave;
        return (in < kOfWave / 2 ? gate : up) + min(n0 + of * (kOfWave / 2) + in % (kOfWave / 2), n_end - 1);
    };
    const auto activation_row = [&](int r) __attribute__((always_inline)) -> int64_t {
        const int64_t at = m0 + min((int64_t)r, count - 1);
        return kExperts ? row_of_place(p, at) : at;
    };
    // lane l loads piece (l % 8) ^ swizzle(row) of row l / 8 of the load's rows
    lds_byte* const base = (lds_byte*)lds;
    const bool gathered = kExperts && p.order != nullptr;
    const uint8_t* const a0 = gathered ? p.a : p.a + m0 * p.lda;
    const int64_t b_first = p.gated ? min(gate, up) + n0 : n0;
    const uint8_t* const b0 = p.b + ((int64_t)expert * p.n + b_first) * p.ldb;
    uint32_t offset[kLoads], back[kLoads];  // back: of the piece in its row, taken off where the last stage has no such piece
    const uint8_t* source[kLoads];          // (kDirect: the former; otherwise this)
    uint4_t held[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
        const int row = kRowsPerLoad * (wave * kLoads + i) + lane / kPieces, piece = (lane % kPieces) ^ swizzle(row);
        const bool weights = kRowsPerLoad * (wave * kLoads + i) >= kBM;
        back[i] = 16 * piece;
        int64_t from;
        if (weights)
            from = (weight_row(row - kBM) - b_first) * p.ldb;
        else
            from = (activation_row(row) - (gathered ? 0 : m0)) * p.lda;
        if constexpr (kDirect)
            offset[i] = (uint32_t)from + back[i];
        else
            source[i] = (weights ? b0 : a0) + from;
    }
    // scales: wavefronts 0 .. kScaleWaves - 1 those of 64 activation rows each, the next the weights' (gated: of the two halves in turn), the others the same for nothing
    const int64_t blocks = stages, n_blocks = (p.n + kFp8Block - 1) / kFp8Block;
    const uint8_t* scale_at;
    int64_t scale_step;
    if (wave < kScaleWaves) {
        scale_at = (const uint8_t*)(p.a_scales + activation_row(min(64 * wave + lane, kBM - 1)) * p.a_scale_row);
        scale_step = 4 * p.a_scale_block;
    } else {
        const int64_t row = p.gated ? (lane & 1 ? up : gate) + n0 : n0;  // (a tile's columns share a block; of a gated unit, each half of them)
        scale_at = (const uint8_t*)(p.b_scales + ((int64_t)expert * n_blocks + row / kFp8Block) * blocks);
        scale_step = 4;
    }
    const auto load = [&](int stage, int slot) __attribute__((always_inline)) {
        const int64_t k0 = (int64_t)stage * kStageBytes;
        const uint32_t room = (uint32_t)min(p.k - k0, (int64_t)kStageBytes);
        lds_byte* const to = base + slot * kSlot;
        if constexpr (kDirect) {
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                const int row = kRowsPerLoad * (wave * kLoads + i);
                load_to_lds_16((row >= kBM ? b0 : a0) + k0, offset[i] - (back[i] < room ? 0u : back[i]), to + row * kStageBytes);
            }
        } else if (room == kStageBytes) {  // (all of them on their way at once; a choice at each piece has it waited for there)
#pragma unroll
            for (int i = 0; i < kLoads; i++) __builtin_memcpy(&held[i], source[i] + k0 + back[i], 16);
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; i++) held[i] = load_bytes16(source[i], k0 + back[i], p.k);
        }
        load_to_lds_4(scale_at + stage * scale_step, to + kScalesAt + 256 * min(wave, kScaleWaves + 1));
    };
    const auto deposit = [&](int slot) __attribute__((always_inline)) {  // (not kDirect)
#pragma unroll
        for (int i = 0; i < kLoads; i++) *(uint4_t*)(lds + slot * kSlot + kRowsPerLoad * (wave * kLoads + i) * kStageBytes + 16 * lane) = held[i];
    };
    float4_t acc[kTN][kTM];
#pragma unroll
    for (int j = 0; j < kTN; j++)
#pragma unroll
        for (int i = 0; i < kTM; i++) acc[j][i] = (float4_t){0.0f, 0.0f, 0.0f, 0.0f};
    const int wm = (wave / kWN) * (kBM / kWM), wn = kBM + (wave % kWN) * kOfWave;  // first rows in a slot
    const int frow = lane & 15, quarter = lane >> 4;
    const int steps = last - first;
    const int tail = (int)((p.k - (int64_t)(stages - 1) * kStageBytes) / 16);  // pieces of the last stage
    // stages without missing pieces (not kDirect: those are zeros already)
    const int whole = steps - (kDirect && last == stages && tail < kPieces ? 1 : 0);
    const auto multiply = [&](int slot, bool cut) __attribute__((always_inline)) {
        const uint8_t* const s = lds + slot * kSlot;
        const float* const scales = (const float*)(s + kScalesAt);
        const auto fragment = [&](int row) __attribute__((always_inline)) {
            const uint8_t* const r = s + (row + frow) * kStageBytes;
            return joined(*(const uint4_t*)(r + 16 * (quarter ^ swizzle(frow))), *(const uint4_t*)(r + 16 * ((quarter + 4) ^ swizzle(frow))));
        };
        int8v_t w[kTN];
#pragma unroll
        for (int j = 0; j < kTN; j++) {
            w[j] = fragment(wn + 16 * j);
            if (cut) {
#pragma unroll
                for (int e = 0; e < 8; e++) w[j][e] = (e < 4 ? quarter : quarter + 4) >= tail ? 0 : w[j][e];
            }
        }
        const float scale_lo = scales[64 * kScaleWaves], scale_hi = scales[64 * kScaleWaves + 1];
        float a_scale[kTM];
#pragma unroll
        for (int i = 0; i < kTM; i++) a_scale[i] = scales[wm + 16 * i + frow];
        // one activation fragment ahead of the products, and the products of one ahead of their fma
        int8v_t x[2];
        float4_t sum[2][kTN];
        x[0] = fragment(wm);
#pragma unroll
        for (int i = 0; i <= kTM; i++) {
            if (i + 1 < kTM) x[(i + 1) & 1] = fragment(wm + 16 * (i + 1));
#pragma unroll
            for (int j = 0; j < kTN; j++) {
                const float4_t zero = {0.0f, 0.0f, 0.0f, 0.0f};
                if (i < kTM) sum[i & 1][j] = kExact ? mma_fp8_16_exact(w[j], x[i & 1], zero) : mma_fp8_16(w[j], x[i & 1], zero);
                if (i > 0) {
                    const float scale = a_scale[i - 1] * (j < kTN / 2 ? scale_lo : scale_hi);
#pragma unroll
                    for (int r = 0; r < 4; r++) acc[j][i - 1][r] = fmaf(sum[(i - 1) & 1][j][r], scale, acc[j][i - 1][r]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // stage i has landed for every wavefront, and all have left the stages in front of it
    constexpr int kPerStage = kDirect ? kLoads + 1 : 1;
    const auto arrived = [&](int i) __attribute__((always_inline)) {
        if (i + kRing - 1 <= steps)
            barrier_keeping<kDirect ? (kRing - 2) * kPerStage : 0>();  // stages up to i + kRing - 2 are on their way
        else
            barrier_keeping<0>();
    };
    // (see matmul_i8_tiles.hip: with one row of tiles these begin at different stages, so that they do not all wait for the same memory channels)
    const int rotate = g.rotate && whole > 0 ? (int)((uint32_t)tile * 37u % (uint32_t)whole) : 0;
    const auto stage_at = [&](int i) __attribute__((always_inline)) { return first + (i >= whole ? i : i + rotate < whole ? i + rotate : i + rotate - whole); };
    if constexpr (kDirect) {
#pragma unroll
        for (int i = 0; i < kRing - 1; i++)
            if (i < steps) load(stage_at(i), i);
    } else if (steps > 0) {
        load(stage_at(0), 0);
        deposit(0);
    }
    const auto next_of = [](int s) __attribute__((always_inline)) { return s + 1 == kRing ? 0 : s + 1; };
    int slot = 0, fill = kRing - 1;
    for (int i = 0; i < whole; i++) {
        arrived(i);
        const bool more = i + kRing - 1 < steps;
        if (more) load(stage_at(i + kRing - 1), fill);  // (into the slot that every wavefront left before the barrier)
        multiply(slot, false);
        if constexpr (!kDirect) {
            if (more) deposit(fill);
        }
        slot = next_of(slot);
        fill = next_of(fill);
    }
    if (whole < steps) {
        arrived(whole);
        multiply(slot, true);
    }
    // register r of acc[j][i]: weight row 16 j + 4 (lane / 16) + r, activation row 16 i + lane % 16 of the wavefront's
    const int64_t n_first = n0 + (wave % kWN) * (p.gated ? kOfWave / 2 : kOfWave);
    if (g.sums != nullptr) {
#pragma unroll
        for (int i = 0; i < kTM; i++) {
            const int64_t row = m0 + wm + 16 * i + frow;
            if (row >= p.m) continue;
            float* const to = g.sums + ((int64_t)part * p.m + row) * g.sums_stride + n_first + 4 * quarter;
#pragma unroll
            for (int j = 0; j < kTN; j++)
                if (n_first + 16 * j + 4 * quarter < p.n) *(float4_t*)(to + 16 * j) = acc[j][i];  // (rows of sums are whole fours)
        }
        return;
    }
    // results through the wavefront's own LDS, to be stored as rows: eight columns a lane
    __syncthreads();
    uint8_t* const out = lds + wave * kOutBytes;
    const auto store_rows = [&](auto columns_of_wave, const auto& value) __attribute__((always_inline)) {
        constexpr int kColumns = decltype(columns_of_wave)::value, kPerRow = kColumns / 8, kRowsAtOnce = 64 / kPerRow < 16 ? 64 / kPerRow : 16;
        const int64_t column = n_first + 8 * (lane % kPerRow);
        const int columns = (int)max((int64_t)0, min(n_end - column, (int64_t)8));
        float bias[8];
#pragma unroll
        for (int e = 0; e < 8; e++) bias[e] = p.bias != nullptr && e < columns ? load_scalar(p.bias, column + e, p.c_dtype) : 0.0f;
#pragma unroll
        for (int i = 0; i < kTM; i++) {
#pragma unroll
            for (int j = 0; j < kColumns / 16; j++) *(float4_t*)(out + frow * kOutRow + 4 * (16 * j + 4 * quarter)) = value(j, i);
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int r0 = 0; r0 < 16; r0 += kRowsAtOnce) {
                const int r = r0 + lane / kPerRow;
                const int64_t at = wm + 16 * i + r;
                if (r < 16 && at < count && columns > 0) {
                    const float4_t lo = *(const float4_t*)(out + r * kOutRow + 32 * (lane % kPerRow)), hi = *(const float4_t*)(out + r * kOutRow + 32 * (lane % kPerRow) + 16);
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] = (e < 4 ? lo[e] : hi[e - 4]) + bias[e];
                    store_columns_fp8(p, (m0 - p.first_place + at) * p.ldc + column, columns, y);
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
    };
    if (p.gated) {
        store_rows(Constant<kOutColumns / 2>{}, [&](int j, int i) __attribute__((always_inline)) {
            float4_t y;
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = gated(acc[j][i][r], p.activation) * acc[j + kTN / 2][i][r];
            return y;
        });
    } else {
        store_rows(Constant<kOutColumns>{}, [&](int j, int i) __attribute__((always_inline)) { return acc[j][i]; });
    }
}

// The parts' sums and the end of the result, four columns a lane.
__global__ __launch_bounds__(256) void matmul_fp8_finish_kernel(MatmulFp8Params p, const float* sums, int64_t stride, int parts) {
    const int64_t column = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x), row = blockIdx.y;
    if (column >= p.n) return;
    const float* const s = sums + row * stride + column;
    float4_t sum = *(const float4_t*)s;
#pragma unroll 4
    for (int i = 1; i < parts; i++) sum += *(const float4_t*)(s + i * p.m * stride);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (column + e >= p.n) break;
        const int64_t to = row * p.ldc + column + e;
        store_scalar(p.c, to, p.c_dtype, finished_fp8(p, sum[e], to, column + e));
    }
}

template <int kBM, int kBN, int kWM, int kWN, int kRing, bool kDirect, bool kExperts>
hipError_t launch(const MatmulFp8Params& p, Fp8Grid g, bool exact, hipStream_t stream) {
    const int64_t tiles_m = kExperts ? most_expert_tiles(p, kBM) : (p.m + kBM - 1) / kBM;
    g.tiles_m = (int)tiles_m;
    g.tiles_n = (int)(p.gated ? GatedTiles(p.n / 2).count() : (p.n + kBN - 1) / kBN);
    g.rotate = !kExperts && tiles_m == 1 && g.parts == 1;
    const int64_t grid = 8 * ((tiles_m * g.tiles_n * g.parts + 7) / 8);
    const auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * kWM * kWN), 0, stream, p, g); };
    if (!exact) {
        run(matmul_fp8_tiles_kernel<kBM, kBN, kWM, kWN, kRing, kDirect, kExperts, false>);
    } else if constexpr (kBM == 32 || kBM == 128) {  // (results in fp32: tiles of these sizes alone)
        run(matmul_fp8_tiles_kernel<kBM, kBN, kWM, kWN, kRing, kDirect, kExperts, true>);
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace

template <bool kExperts>
hipError_t launch_matmul_fp8_tiles(const MatmulFp8Params& p, const Fp8Plan& plan, bool exact, void* workspace, hipStream_t stream) {
    Fp8Grid g{};
    g.parts = plan.parts;
    g.group_rows = 8;
    g.sums_stride = (p.n + 3) / 4 * 4;
    if (plan.parts > 1) g.sums = (float*)workspace;
    hipError_t e = hipSuccess;
    switch (plan.tile) {
        case kFp8Few: return launch_matmul_fp8_few<kExperts>(p, exact, stream);
        case kFp8Tile256: return launch_matmul_fp8_deep<kExperts>(p, stream);
        case kFp8Tile128: e = launch<128, 128, 2, 2, 2, true, kExperts>(p, g, exact, stream); break;
        // (eight wavefronts where a compute unit has one or two workgroups, as a rule of dense products: 256 x 8,192 x 4,096 25.0 -> 21.2 us, 64 x 28,672 x
        // 4,096 31.0 -> 28.8; experts' many small tiles want room for more workgroups: 8 experts of 28,672 x 4,096 with 32 rows each 194 us, with eight 235)
        case kFp8Tile64: e = launch<64, 128, kExperts ? 1 : 2, 4, 3, true, kExperts>(p, g, exact, stream); break;
        case kFp8Tile32: e = launch<32, 128, 1, 4, 3, true, kExperts>(p, g, exact, stream); break;
        case kFp8Any128: e = launch<128, 128, 2, 4, 2, false, kExperts>(p, g, exact, stream); break;
        default: e = launch<32, 128, 1, 4, 2, false, kExperts>(p, g, exact, stream); break;
    }
    if (e != hipSuccess || plan.parts == 1) return e;
    hipLaunchKernelGGL(matmul_fp8_finish_kernel, dim3((unsigned)((p.n + 1023) / 1024), (unsigned)p.m), dim3(256), 0, stream, p, g.sums, g.sums_stride, g.parts);
    return hipGetLastError();
}

}  // namespace hipops
