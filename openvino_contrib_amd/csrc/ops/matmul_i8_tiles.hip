// Products of 8-bit codes in tiles through LDS (hipops_matmul_i8).
//
//   c[i, j] = a_scale[i] b_scale[j] sum_l a[i, l] b[j, l] + bias[j] + residual[i, j]
// Sums on v_mfma_i32_32x32x32_i8, exact; the rest in fp32, rounded once, on the accumulators.
//
// With few activation rows the weights' bytes bound it, with many the matrix cores.  Tiles of 32, 64, 128 and 256 activation rows on 128 (256) weight
// rows: a large one reads less from L2 and LDS for a product, small ones fill the device; k in parts where even those do not, whose sums a second
// launch adds (matmul_i8.hip has the rule and where the sides cross).  A stage is 128 bytes of k, loaded straight to LDS while the one or two
// before it are multiplied (rows at any address: through registers).  8,192 x 8,192 x 8,192 502 us (2.19 POP/s; a library's product of the same 535),
// 8,192 x 6,144 x 4,096 205 (190), 64 x 28,672 x 4,096 27 (4.4 TB/s of weights), 1,111 x 4,096 x 14,336 94 in three parts.  At the large sizes the matrix
// cores are busy 48 % of the time at 1.95 GHz (2.4 without load): loads alone take 169 of the 205 us, products alone 175, 135 on operands of
// zeros.  Slower there: stages of 64 bytes, five on their way (220), four wavefronts of 128 x 128 (342), rows touched in the L2 a stage
// ahead (212 to 216).  Parts added by the workgroup that is last to be done with its own, without a second launch: 5.5 % slower over 291 sizes.
#include "ops/matmul_i8.hpp"

namespace hipops {

namespace {

typedef __attribute__((address_space(3))) uint8_t lds_byte;
// 16 bytes per lane from global memory to LDS: lane l's land at lds_base + 16 l.  Inline assembly, because the compiler waits
// for the intrinsic form at every access to LDS; waited for by hand.
__device__ __forceinline__ void load_to_lds_16(const int8_t* base, uint32_t lane_offset, lds_byte* lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(lane_offset), "s"(base), "s"((uint32_t)(uintptr_t)lds_base)
                 : "memory", "m0");
}
// everything but the kKeep most recent loads of this wavefront has landed, for every wavefront of the workgroup
template <int kKeep>
__device__ __forceinline__ void barrier_keeping() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | (kKeep & 15) | ((kKeep >> 4) << 14));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

constexpr int kStageBytes = 128;  // of a row in a stage
// Rows lie side by side in a stage, their 16-byte pieces permuted so that the sixteen rows that a fragment's read touches at a time (one
// piece of each) lie on all 64 banks.  (row % 8 instead: 25 times the bank conflicts, 8,192 x 6,144 x 4,096 207 -> 205 us all the same.)
__device__ __forceinline__ int swizzle(int row) { return (row >> 1) & 7; }

// kBM activation rows x kBN weight rows, kWM x kWN wavefronts, kRing stages of 128 bytes of k.
// kDirect: rows at multiples of 16 bytes, k too, straight to LDS; otherwise any rows and k, through registers, one stage ahead.
template <int kBM, int kBN, int kWM, int kWN, int kRing, bool kDirect>
__global__ __launch_bounds__(64 * kWM * kWN) __attribute__((amdgpu_waves_per_eu(kWM * kWN == 8 ? 2 : 1, 2))) void matmul_i8_tiles_kernel(MatmulI8Params p, I8Grid g) {
    constexpr int kWaves = kWM * kWN, kRows = kBM + kBN, kSlot = kRows * kStageBytes;
    constexpr int kTM = kBM / kWM / 32, kTN = kBN / kWN / 32;
    constexpr int kPieces = kStageBytes / 16, kRowsPerLoad = 64 / kPieces, kSteps = kStageBytes / 32;
    constexpr int kLoads = kRows / kRowsPerLoad / kWaves;  // of a wavefront for a stage
    static_assert(kRows % (kRowsPerLoad * kWaves) == 0 && kBM % kRowsPerLoad == 0 && kTM > 0 && kTN > 0, "whole loads and tiles");
    static_assert(kRing >= 2 && (kDirect || kRing == 2), "the stage that is read, and those on their way");
    constexpr int kOutColumns = 32 * kTN, kOutRow = 4 * kOutColumns + 16, kOutBytes = 32 * kOutRow;
    constexpr int kLds = kRing * kSlot > kWaves * kOutBytes ? kRing * kSlot : kWaves * kOutBytes;
    __shared__ __attribute__((aligned(128))) uint8_t lds[kLds];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    // workgroups go to the eight XCDs in turn: each takes a run of the tiles, which come in groups of rows so that those that run together
    // share rows of both operands in the XCD's L2
    int index = (int)blockIdx.x;
    if (g.xcd_run > 0) index = (index & 7) * g.xcd_run + (index >> 3);
    const int part = __builtin_amdgcn_readfirstlane(index / g.tiles);
    if (part >= g.parts) return;
    const int tile = index - part * g.tiles;
    const int in_group = g.group_rows * g.tiles_n, group = tile / in_group;
    const int rows_here = min(g.group_rows, g.tiles_m - group * g.group_rows), at = tile - group * in_group;
    const int64_t m0 = (int64_t)__builtin_amdgcn_readfirstlane(group * g.group_rows + at % rows_here) * kBM;
    const int64_t n0 = (int64_t)__builtin_amdgcn_readfirstlane(at / rows_here) * kBN;
    const int stages = (int)((p.k + kStageBytes - 1) / kStageBytes);
    const int first = (int)((int64_t)stages * part / g.parts), last = (int)((int64_t)stages * (part + 1) / g.parts);

    // lane l loads piece (l % 8) ^ swizzle(row) of row l / 8 of the load's rows
    lds_byte* const base = (lds_byte*)lds;
    const int8_t* const a0 = p.a + m0 * p.lda;
    const int8_t* const b0 = p.b + n0 * p.ldb;
    uint32_t offset[kLoads], back[kLoads];  // back: of the piece in its row, taken off where the last stage has no such piece
    const int8_t* source[kLoads];           // (kDirect: the former; otherwise this)
    uint4_t held[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; i++) {
        const int row = kRowsPerLoad * (wave * kLoads + i) + lane / kPieces, piece = (lane % kPieces) ^ swizzle(row);
        const bool weights = kRowsPerLoad * (wave * kLoads + i) >= kBM;
        const int64_t in_tile = weights ? min((int64_t)(row - kBM), p.n - 1 - n0) : min((int64_t)row, p.m - 1 - m0);
        back[i] = 16 * piece;
        if constexpr (kDirect)
            offset[i] = (uint32_t)(in_tile * (weights ? p.ldb : p.lda)) + back[i];
        else
            source[i] = (weights ? b0 : a0) + in_tile * (weights ? p.ldb : p.lda);
    }
    const auto load = [&](int stage, int slot) __attribute__((always_inline)) {
        const int64_t k0 = (int64_t)stage * kStageBytes;
        const uint32_t room = (uint32_t)min(p.k - k0, (int64_t)kStageBytes);
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const int row = kRowsPerLoad * (wave * kLoads + i);
            if constexpr (kDirect)
                load_to_lds_16((row >= kBM ? b0 : a0) + k0, offset[i] - (back[i] < room ? 0u : back[i]), base + slot * kSlot + row * kStageBytes);
            else
                held[i] = load_codes16(source[i], k0 + back[i], p.k);
        }
    };
    const auto deposit = [&](int slot) __attribute__((always_inline)) {  // (not kDirect)
#pragma unroll
        for (int i = 0; i < kLoads; i++) *(uint4_t*)(lds + slot * kSlot + kRowsPerLoad * (wave * kLoads + i) * kStageBytes + 16 * lane) = held[i];
    };
    int16v_t acc[kTN][kTM];
#pragma unroll
    for (int j = 0; j < kTN; j++)
#pragma unroll
        for (int i = 0; i < kTM; i++)
#pragma unroll
            for (int r = 0; r < 16; r++) acc[j][i][r] = 0;
    const int wm = (wave / kWN) * (kBM / kWM), wn = kBM + (wave % kWN) * (kBN / kWN);  // first rows in a slot
    const int frow = lane & 31, fhalf = lane >> 5;
    struct Fragments {
        uint4_t w[kTN], x[kTM];
    };
    const int count = last - first;
    const int tail = (int)((p.k - (int64_t)(stages - 1) * kStageBytes) / 16);  // pieces of the last stage
    // stages without missing pieces (not kDirect: those are zeros already)
    const int whole = count - (kDirect && last == stages && tail < kPieces ? 1 : 0);
    const auto multiply = [&](int slot, bool cut) __attribute__((always_inline)) {
        const auto read = [&](Fragments& f, int step) __attribute__((always_inline)) {
            const uint8_t* const s = lds + slot * kSlot + frow * kStageBytes;
            const int piece = 2 * step + fhalf, where = 16 * (piece ^ swizzle(frow));
#pragma unroll
            for (int j = 0; j < kTN; j++) {
                f.w[j] = *(const uint4_t*)(s + (wn + 32 * j) * kStageBytes + where);
                if (cut && piece >= tail) f.w[j] = (uint4_t){0u, 0u, 0u, 0u};
            }
#pragma unroll
            for (int i = 0; i < kTM; i++) f.x[i] = *(const uint4_t*)(s + (wm + 32 * i) * kStageBytes + where);
        };
        // (one step's fragments ahead of the products, and no further: the accumulators leave no registers for more)
        Fragments f[2];
        read(f[0], 0);
#pragma unroll
        for (int step = 0; step < kSteps; step++) {
            if (step + 1 < kSteps) read(f[(step + 1) & 1], step + 1);
#pragma unroll
            for (int i = 0; i < kTM; i++)
#pragma unroll
                for (int j = 0; j < kTN; j++) acc[j][i] = mma_i8(f[step & 1].w[j], f[step & 1].x[i], acc[j][i]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // stage i has landed for every wavefront, and all have left the stages in front of it
    const auto arrived = [&](int i) __attribute__((always_inline)) {
        if (i + kRing - 1 <= count)
            barrier_keeping<kDirect ? (kRing - 2) * kLoads : 0>();  // stages up to i + kRing - 2 are on their way
        else
            barrier_keeping<0>();
    };
    // With one row of tiles these begin at different stages (the sums do not mind): rows whose distance is a power of two would have all
    // of them wait for the same memory channels (64 x 28,672 x 4,096 29.4 -> 27.4 us, 16 x 28,672 x 4,096 27.1 -> 24.2).  Tiles that share
    // weights in the L2 go through k together (8,192 x 6,144 x 4,096 206 us, 232 apart), and so do parts, which begin apart.
    const int rotate = g.rotate && whole > 0 ? (int)((uint32_t)tile * 37u % (uint32_t)whole) : 0;
    const auto stage_at = [&](int i) __attribute__((always_inline)) { return first + (i >= whole ? i : i + rotate < whole ? i + rotate : i + rotate - whole); };
    if constexpr (kDirect) {
#pragma unroll
        for (int i = 0; i < kRing - 1; i++)
            if (i < count) load(stage_at(i), i);
    } else if (count > 0) {
        load(stage_at(0), 0);
        deposit(0);
    }
    const auto next_of = [](int s) __attribute__((always_inline)) { return s + 1 == kRing ? 0 : s + 1; };
    int slot = 0, fill = kRing - 1;
    for (int i = 0; i < whole; i++) {
        arrived(i);
        const bool more = i + kRing - 1 < count;
        if (more) load(stage_at(i + kRing - 1), fill);  // (into the slot that every wavefront left before the barrier)
        multiply(slot, false);
        if constexpr (!kDirect) {
            if (more) deposit(fill);
        }
        slot = next_of(slot);
        fill = next_of(fill);
    }
    if (whole < count) {
        arrived(whole);
        multiply(slot, true);
    }
    // register r of acc[j][i]: weight row 32 j + 8 (r / 4) + 4 (lane / 32) + r % 4, activation row 32 i + lane % 32 of the wavefront's
    const int64_t m_first = m0 + wm, n_first = n0 + wn - kBM;
    if (g.sums != nullptr) {
#pragma unroll
        for (int i = 0; i < kTM; i++) {
            const int64_t row = m_first + 32 * i + frow;
            if (row >= p.m) break;
            int* const to = g.sums + ((int64_t)part * p.m + row) * g.sums_stride + n_first + 4 * fhalf;
#pragma unroll
            for (int j = 0; j < kTN; j++)
#pragma unroll
                for (int q = 0; q < 4; q++)
                    if (n_first + 32 * j + 8 * q + 4 * fhalf < p.n)  // (rows of sums are whole fours)
                        *(int4_t*)(to + 32 * j + 8 * q) = (int4_t){acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
        }
        return;
    }
    // results through the wavefront's own LDS, to be stored as rows: eight columns a lane
    __syncthreads();
    uint8_t* const out = lds + wave * kOutBytes;
    constexpr int kPerRow = kOutColumns / 8, kRowsAtOnce = 64 / kPerRow;
    const int64_t column = n_first + 8 * (lane % kPerRow);
    const int columns = (int)max((int64_t)0, min(p.n - column, (int64_t)8));
    float scale[8], bias[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
        scale[e] = p.b_scales != nullptr && e < columns ? p.b_scales[column + e] : 1.0f;
        bias[e] = p.bias != nullptr && e < columns ? load_scalar(p.bias, column + e, p.c_dtype) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kTM; i++) {
#pragma unroll
        for (int j = 0; j < kTN; j++)
#pragma unroll
            for (int q = 0; q < 4; q++)
                *(int4_t*)(out + frow * kOutRow + 4 * (32 * j + 8 * q + 4 * fhalf)) =
                    (int4_t){acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r0 = 0; r0 < 32; r0 += kRowsAtOnce) {
            const int r = r0 + lane / kPerRow;
            const int4_t lo = *(const int4_t*)(out + r * kOutRow + 32 * (lane % kPerRow)), hi = *(const int4_t*)(out + r * kOutRow + 32 * (lane % kPerRow) + 16);
            const int64_t row = m_first + 32 * i + r;
            if (row >= p.m || columns == 0) continue;
            const float row_scale = p.a_scales != nullptr ? p.a_scales[row] : 1.0f;
            const int64_t to = row * p.ldc + column;
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = fmaf((float)(e < 4 ? lo[e] : hi[e - 4]), row_scale * scale[e], bias[e]);
            store_columns(p, to, columns, y);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// The parts' sums and the end of the result, four columns a lane.
__global__ __launch_bounds__(256) void matmul_i8_finish_kernel(MatmulI8Params p, const int* sums, int64_t stride, int parts) {
    const int64_t column = 4 * ((int64_t)blockIdx.x * 256 + threadIdx.x), row = blockIdx.y;
    if (column >= p.n) return;
    const int* const s = sums + row * stride + column;
    int4_t sum = *(const int4_t*)s;
#pragma unroll 4
    for (int i = 1; i < parts; i++) sum += *(const int4_t*)(s + i * p.m * stride);
    const float row_scale = p.a_scales != nullptr ? p.a_scales[row] : 1.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (column + e >= p.n) break;
        float y = fmaf((float)sum[e], row_scale * (p.b_scales != nullptr ? p.b_scales[column + e] : 1.0f),
                       p.bias != nullptr ? load_scalar(p.bias, column + e, p.c_dtype) : 0.0f);
        const int64_t to = row * p.ldc + column + e;
        if (p.residual != nullptr) y += load_scalar(p.residual, to, p.c_dtype);
        store_scalar(p.c, to, p.c_dtype, y);
    }
}

template <int kBM, int kBN, int kWM, int kWN, int kRing, bool kDirect>
void launch(const MatmulI8Params& p, I8Grid g, hipStream_t stream) {
    g.tiles_m = (int)((p.m + kBM - 1) / kBM);
    g.tiles_n = (int)((p.n + kBN - 1) / kBN);
    g.tiles = g.tiles_m * g.tiles_n;
    g.rotate = g.tiles_m == 1 && g.parts == 1;
    const int64_t total = (int64_t)g.tiles * g.parts;
    g.xcd_run = (int)((total + 7) / 8);
    const int64_t grid = 8 * (int64_t)g.xcd_run;
    hipLaunchKernelGGL((matmul_i8_tiles_kernel<kBM, kBN, kWM, kWN, kRing, kDirect>), dim3((unsigned)grid), dim3(64 * kWM * kWN), 0, stream, p, g);
}

}  // namespace

hipError_t launch_matmul_i8_tiles(const MatmulI8Params& p, const I8Plan& plan, void* workspace, hipStream_t stream) {
    I8Grid g{};
    g.parts = plan.parts;
    g.group_rows = 8;
    g.sums_stride = (p.n + 3) / 4 * 4;
    if (plan.parts > 1) g.sums = (int*)workspace;
    switch (plan.tile) {
        case kI8Tile256: launch<256, 256, 2, 4, 2, true>(p, g, stream); break;
        case kI8Tile128: launch<128, 128, 2, 2, 2, true>(p, g, stream); break;
        case kI8Tile128Deep: launch<128, 128, 2, 4, 4, true>(p, g, stream); break;
        case kI8Tile64: launch<64, 128, 1, 4, 3, true>(p, g, stream); break;
        case kI8Tile32: launch<32, 128, 1, 4, 3, true>(p, g, stream); break;
        case kI8Any128: launch<128, 128, 2, 2, 2, false>(p, g, stream); break;
        default: launch<32, 128, 1, 4, 2, false>(p, g, stream); break;
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || plan.parts == 1) return e;
    hipLaunchKernelGGL(matmul_i8_finish_kernel, dim3((unsigned)((p.n + 1023) / 1024), (unsigned)p.m), dim3(256), 0, stream, p, g.sums, g.sums_stride, g.parts);
    return hipGetLastError();
}

}  // namespace hipops
