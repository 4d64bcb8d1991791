// Rows as 8-bit codes with a scale each (hipops_quantize_rows): what stands ahead of an 8-bit projection, with the RMS norm or the
// GLU that the layer has there on the way, so that neither goes through memory in 16 bits.
//
// HBM-bound: x read once, a byte an element written.  A workgroup takes a row and keeps it in registers (eight elements to a
// chunk, kKeep chunks a lane) over its reductions: the norm's sum of squares, then the largest magnitude; from 1,024 rows on a wavefront takes
// one by itself where its registers hold it.  bf16 rows, us: 8,192 of 4,096 plain 16.8 (6.0 TB/s), behind a norm 20.1, 1,111 of 14,336 behind a
// GLU 20.1 (4.0 TB/s: the activation's instructions), 8,192 of them 116 (5.1 TB/s), 64 of 4,096 behind a norm 3.8, one 2.5.
#include "hipops_int8.h"
#include "ops/ops_common.hpp"
#include "ops/vec8.hpp"

namespace hipops {

namespace {

struct QuantizeParams {
    const void* x;
    const void* gamma;
    int8_t* codes;
    float* scales;
    int64_t rows, width, x_row_stride;
    int source, x_dtype, gamma_dtype, activation, gate_first;
    float eps;
};

constexpr int kMaxWaves = 16;
constexpr int64_t kByWaveRows = 1024;

__device__ __forceinline__ float scale_of_peak(float peak) {
    const float s = peak * (1.0f / 127.0f);
    return s < 1e-30f ? 0.0f : s;
}
__device__ __forceinline__ int code_of(float y, float inverse) { return (int)fminf(fmaxf(rintf(y * inverse), -127.0f), 127.0f); }

// 1 / rms of a row with this sum of squares; 0 where mean square and eps are both 0, so that a row of zeros stays one (and not 0 times infinity)
__device__ __forceinline__ float inverse_rms(const QuantizeParams& p, float sq) {
    const float square = sq / (float)p.width + p.eps;
    // (every lane has the same sum: a scalar choice, 8,192 rows of 4,097 104.4 us, 106.9 with one in each lane)
    return __builtin_amdgcn_readfirstlane(square == 0.0f) ? 0.0f : 1.0f / sqrtf(square);
}

// over all lanes of the workgroup; `partial` is free again after the next barrier
template <bool kMax>
__device__ __forceinline__ float reduce(float x, float* partial) {
    x = kMax ? wave_max(x) : wave_sum(x);
    const int waves = (int)blockDim.x >> 6;
    if (waves == 1) return x;
    if ((threadIdx.x & 63) == 0) partial[threadIdx.x >> 6] = x;
    __syncthreads();
    x = partial[0];
    for (int w = 1; w < waves; w++) x = kMax ? fmaxf(x, partial[w]) : x + partial[w];
    return x;
}

// The activations of a GLU.  (Swish with the reciprocal instruction, good to a unit in the last place, instead of a division of ten
// operations: with the codes' conversion it is what a row of a GLU costs beside its bytes.)
__device__ __forceinline__ float gated(float x, int activation) {
    if (activation == HIPOPS_GLU_SWISH) return x * __builtin_amdgcn_rcpf(1.0f + __expf(-x));
    return activate(x, activation, 1.0f);
}

// kKeep chunks of a row as floats, zeros behind its end.  All loads of a type stand in one run of code, ahead of what converts them:
// a choice of the type at each would have every one waited for before the next (8,192 rows of 4,096 behind a norm 28 us against 20).
template <int kKeep>
struct RawChunks {
    uint4_t lo[kKeep], up[kKeep];  // (up: the second half of eight floats)
};
template <int kKeep>
__device__ __forceinline__ void load_chunks(RawChunks<kKeep>& r, const void* base, int64_t at, int dtype, int lane, int lanes, int chunks) {
#pragma unroll
    for (int c = 0; c < kKeep; c++) r.lo[c] = r.up[c] = (uint4_t){0u, 0u, 0u, 0u};
    if (dtype == HIPATTN_F32) {
#pragma unroll
        for (int c = 0; c < kKeep; c++) {
            const int chunk = lane + c * lanes;
            if (chunk < chunks) {
                r.lo[c] = *(const uint4_t*)((const float*)base + at + 8 * (int64_t)chunk);
                r.up[c] = *(const uint4_t*)((const float*)base + at + 8 * (int64_t)chunk + 4);
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < kKeep; c++) {
            const int chunk = lane + c * lanes;
            if (chunk < chunks) r.lo[c] = *(const uint4_t*)((const uint16_t*)base + at + 8 * (int64_t)chunk);
        }
    }
}
template <int kKeep>
__device__ __forceinline__ void floats_of(const RawChunks<kKeep>& r, int dtype, Float8 (&x)[kKeep]) {
    if (dtype == HIPATTN_F32) {
#pragma unroll
        for (int c = 0; c < kKeep; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[c].v[e] = __uint_as_float(e < 4 ? r.lo[c][e] : r.up[c][e - 4]);
    } else if (dtype == HIPATTN_F16) {
#pragma unroll
        for (int c = 0; c < kKeep; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[c].v[e] = f16_bits_to_float((uint16_t)(r.lo[c][e >> 1] >> (16 * (e & 1))));
    } else {
#pragma unroll
        for (int c = 0; c < kKeep; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) x[c].v[e] = bf16_bits_to_float((uint16_t)(r.lo[c][e >> 1] >> (16 * (e & 1))));
    }
}

// A row by `lanes` lanes of a workgroup, of which this is number `lane`; `over` reduces (sum of squares, largest magnitude) over them.
// Behind a norm y = (x gamma) / rms(x): the largest |x gamma| is found together with the sum of squares, so that one reduction does,
// and the codes are x gamma times one number.
template <int kSource, int kKeep, typename Reduce>
__device__ __forceinline__ void quantize_row(const QuantizeParams& p, int64_t row, int lane, int lanes, const Reduce& over) {
    const int64_t at = row * p.x_row_stride;
    const int chunks = (int)(p.width / 8);
    Float8 y[kKeep];
    float sq = 0.0f, peak = 0.0f;
    RawChunks<kKeep> raw, other;
    load_chunks(raw, p.x, at + (kSource == HIPOPS_QUANTIZE_GLU && !p.gate_first ? p.width : 0), p.x_dtype, lane, lanes, chunks);
    if constexpr (kSource == HIPOPS_QUANTIZE_GLU) load_chunks(other, p.x, at + (p.gate_first ? p.width : 0), p.x_dtype, lane, lanes, chunks);
    const bool weighed = kSource == HIPOPS_QUANTIZE_RMS_NORM && p.gamma != nullptr;
    if (weighed) load_chunks(other, p.gamma, 0, p.gamma_dtype, lane, lanes, chunks);
    floats_of(raw, p.x_dtype, y);
    if constexpr (kSource == HIPOPS_QUANTIZE_GLU) {
        Float8 up[kKeep];
        floats_of(other, p.x_dtype, up);
#pragma unroll
        for (int c = 0; c < kKeep; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) y[c].v[e] = gated(y[c].v[e], p.activation) * up[c].v[e];
    }
    if constexpr (kSource == HIPOPS_QUANTIZE_RMS_NORM) {
#pragma unroll
        for (int c = 0; c < kKeep; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) sq = fmaf(y[c].v[e], y[c].v[e], sq);
        if (weighed) {
            Float8 g[kKeep];
            floats_of(other, p.gamma_dtype, g);
#pragma unroll
            for (int c = 0; c < kKeep; c++)
#pragma unroll
                for (int e = 0; e < 8; e++) y[c].v[e] *= g[c].v[e];
        }
    }
#pragma unroll
    for (int c = 0; c < kKeep; c++)
#pragma unroll
        for (int e = 0; e < 8; e++) peak = fmaxf(peak, fabsf(y[c].v[e]));
    over(sq, peak);
    const float inv = kSource == HIPOPS_QUANTIZE_RMS_NORM ? inverse_rms(p, sq) : 1.0f;
    const float scale = scale_of_peak(peak * inv);
    const float inverse = scale > 0.0f ? inv * (1.0f / scale) : 0.0f;
    if (lane == 0) p.scales[row] = scale;
#pragma unroll
    for (int c = 0; c < kKeep; c++) {
        const int chunk = lane + c * lanes;
        if (chunk >= chunks) break;
        const float* const v = y[c].v;
        *(uint2*)(p.codes + row * p.width + 8 * (int64_t)chunk) = make_uint2(codes4(v[0], v[1], v[2], v[3], inverse), codes4(v[4], v[5], v[6], v[7], inverse));
    }
}

template <int kSource, int kKeep>
__global__ __launch_bounds__(64 * kMaxWaves) void quantize_rows_kernel(QuantizeParams p) {
    __shared__ float2 partial[kMaxWaves];
    quantize_row<kSource, kKeep>(p, blockIdx.x, threadIdx.x, blockDim.x, [&](float& sq, float& peak) {
        if (kSource == HIPOPS_QUANTIZE_RMS_NORM) sq = wave_sum(sq);
        peak = wave_max(peak);
        const int waves = (int)blockDim.x >> 6;
        if (waves == 1) return;
        if ((threadIdx.x & 63) == 0) partial[threadIdx.x >> 6] = make_float2(sq, peak);
        __syncthreads();
        sq = 0.0f;
        for (int w = 0; w < waves; w++) {
            sq += partial[w].x;
            peak = fmaxf(peak, partial[w].y);
        }
    });
}

// Many rows of up to 4,096: a wavefront to a row, and no barrier.
constexpr int kRowsPerGroup = 4;
template <int kSource, int kKeep>
__global__ __launch_bounds__(64 * kRowsPerGroup) void quantize_rows_by_wave_kernel(QuantizeParams p) {
    const int64_t row = (int64_t)blockIdx.x * kRowsPerGroup + (threadIdx.x >> 6);
    if (row >= p.rows) return;
    quantize_row<kSource, kKeep>(p, row, threadIdx.x & 63, 64, [&](float& sq, float& peak) {
        if (kSource == HIPOPS_QUANTIZE_RMS_NORM) sq = wave_sum(sq);
        peak = wave_max(peak);
    });
}

// Any width, stride and alignment: the row is read again for every pass.
template <int kSource>
__device__ __forceinline__ float value1(const QuantizeParams& p, int64_t at, int64_t i) {
    if constexpr (kSource != HIPOPS_QUANTIZE_GLU) return load_scalar(p.x, at + i, p.x_dtype);
    return activate(load_scalar(p.x, at + (p.gate_first ? 0 : p.width) + i, p.x_dtype), p.activation, 1.0f) *
           load_scalar(p.x, at + (p.gate_first ? p.width : 0) + i, p.x_dtype);
}
template <int kSource>
__global__ __launch_bounds__(256) void quantize_rows_scalar_kernel(QuantizeParams p) {
    __shared__ float sums[kMaxWaves], peaks[kMaxWaves];
    const int64_t row = blockIdx.x, at = row * p.x_row_stride;
    float inv = 1.0f, peak = 0.0f;
    if constexpr (kSource == HIPOPS_QUANTIZE_RMS_NORM) {
        float sq = 0.0f;
        for (int64_t i = threadIdx.x; i < p.width; i += blockDim.x) {
            const float x = value1<kSource>(p, at, i);
            sq = fmaf(x, x, sq);
        }
        inv = inverse_rms(p, reduce<false>(sq, sums));
    }
    const auto value = [&](int64_t i) {
        float y = value1<kSource>(p, at, i);
        if constexpr (kSource == HIPOPS_QUANTIZE_RMS_NORM) {
            y *= inv;
            if (p.gamma != nullptr) y *= load_scalar(p.gamma, i, p.gamma_dtype);
        }
        return y;
    };
    for (int64_t i = threadIdx.x; i < p.width; i += blockDim.x) peak = fmaxf(peak, fabsf(value(i)));
    const float scale = scale_of_peak(reduce<true>(peak, peaks));
    const float inverse = scale > 0.0f ? 1.0f / scale : 0.0f;
    if (threadIdx.x == 0) p.scales[row] = scale;
    for (int64_t i = threadIdx.x; i < p.width; i += blockDim.x) p.codes[row * p.width + i] = (int8_t)code_of(value(i), inverse);
}

// `rows_per_group` rows to a workgroup of `lanes`.  A launch of 2^32 threads or more runs modulo 2^32 of them, without an error (a row of
// three elements to 256 lanes: from 16.8 million rows on): more rows go in several.
template <typename Kernel>
void launch_in_runs(Kernel kernel, const QuantizeParams& all, int64_t rows_per_group, int lanes, hipStream_t stream) {
    const int64_t most = (0xffffffffLL / lanes) * rows_per_group;
    for (int64_t first = 0; first < all.rows; first += most) {
        QuantizeParams p = all;
        p.rows = all.rows - first < most ? all.rows - first : most;
        p.x = (const uint8_t*)all.x + first * all.x_row_stride * (all.x_dtype == HIPATTN_F32 ? 4 : 2);
        p.codes += first * all.width;
        p.scales += first;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((p.rows + rows_per_group - 1) / rows_per_group)), dim3((unsigned)lanes), 0, stream, p);
    }
}

template <int kSource>
void launch(const QuantizeParams& p, bool vector, hipStream_t stream) {
    if (!vector) {
        launch_in_runs(quantize_rows_scalar_kernel<kSource>, p, 1, 256, stream);
        return;
    }
    const int64_t chunks = p.width / 8;
    if (chunks <= 512 && p.rows >= kByWaveRows) {
        const auto by_wave = [&](auto kernel) { launch_in_runs(kernel, p, kRowsPerGroup, 64 * kRowsPerGroup, stream); };
        if (chunks <= 64)
            by_wave(quantize_rows_by_wave_kernel<kSource, 1>);
        else if (chunks <= 128)
            by_wave(quantize_rows_by_wave_kernel<kSource, 2>);
        else if (chunks <= 256)
            by_wave(quantize_rows_by_wave_kernel<kSource, 4>);
        else
            by_wave(quantize_rows_by_wave_kernel<kSource, 8>);
        return;
    }
    // one chunk a lane up to 512 lanes, then more chunks.  A GLU has more lanes instead of a fourth chunk (8,192 rows of 14,336 122 -> 116
    // us, 128 rows 6.0 -> 5.1)
    const int keep = chunks <= 512 ? 1 : chunks <= (kSource == HIPOPS_QUANTIZE_GLU ? 2048 : 1024) ? 2 : 4;
    const int lanes = (int)((chunks + 64 * keep - 1) / (64 * keep) * 64);
    if (keep == 1)
        launch_in_runs(quantize_rows_kernel<kSource, 1>, p, 1, lanes, stream);
    else if (keep == 2)
        launch_in_runs(quantize_rows_kernel<kSource, 2>, p, 1, lanes, stream);
    else
        launch_in_runs(quantize_rows_kernel<kSource, 4>, p, 1, lanes, stream);
}

bool float_dtype(int d) { return d == HIPATTN_F32 || d == HIPATTN_F16 || d == HIPATTN_BF16; }

}  // namespace

hipattn_status quantize_rows(const hipops_quantize_desc* d, const void* x, const void* gamma, int8_t* codes, float* scales, hipStream_t stream) {
    if (!d) return fail(HIPATTN_INVALID_ARGUMENT, "quantize_rows: null descriptor");
    if (d->source < HIPOPS_QUANTIZE_PLAIN || d->source > HIPOPS_QUANTIZE_GLU) return fail(HIPATTN_INVALID_ARGUMENT, "quantize_rows: source %d", d->source);
    const bool norm = d->source == HIPOPS_QUANTIZE_RMS_NORM, glu = d->source == HIPOPS_QUANTIZE_GLU;
    if (d->rows < 0 || d->width <= 0 || d->width > (int64_t)1 << 40)
        return fail(HIPATTN_INVALID_ARGUMENT, "quantize_rows: rows %lld width %lld", (long long)d->rows, (long long)d->width);
    if (!float_dtype(d->x_dtype) || (norm && gamma && !float_dtype(d->gamma_dtype)))
        return fail(HIPATTN_UNSUPPORTED, "quantize_rows: types must be f32, f16 or bf16");
    if (glu && (d->glu_activation < HIPOPS_GLU_SWISH || d->glu_activation > HIPOPS_GLU_GELU_TANH))
        return fail(HIPATTN_INVALID_ARGUMENT, "quantize_rows: activation %d", d->glu_activation);
    if (norm && !(d->eps >= 0.0f)) return fail(HIPATTN_INVALID_ARGUMENT, "quantize_rows: eps must be >= 0");
    const int64_t taken = glu ? 2 * d->width : d->width;
    if (d->x_row_stride != 0 && d->x_row_stride < taken)
        return fail(HIPATTN_INVALID_ARGUMENT, "quantize_rows: rows of %lld elements, %lld apart", (long long)taken, (long long)d->x_row_stride);
    if (d->rows == 0) return HIPATTN_OK;
    if (!x || !codes || !scales) return fail(HIPATTN_INVALID_ARGUMENT, "quantize_rows: null pointer");
    if (d->rows > 0x7fffffffLL) return fail(HIPATTN_UNSUPPORTED, "quantize_rows: too many rows");
    QuantizeParams p{x, gamma, codes, scales, d->rows, d->width, d->x_row_stride ? d->x_row_stride : taken, d->source, d->x_dtype, d->gamma_dtype,
                     d->glu_activation, d->glu_gate_first, d->eps};
    const auto aligned = [](const void* a, uintptr_t n) { return ((uintptr_t)a & (n - 1)) == 0; };
    const bool vector = d->width % 8 == 0 && d->width <= 32768 && p.x_row_stride % 8 == 0 && aligned(x, 16) && aligned(codes, 8) &&
                        (!norm || !gamma || aligned(gamma, 16));
    if (norm)
        launch<HIPOPS_QUANTIZE_RMS_NORM>(p, vector, stream);
    else if (glu)
        launch<HIPOPS_QUANTIZE_GLU>(p, vector, stream);
    else
        launch<HIPOPS_QUANTIZE_PLAIN>(p, vector, stream);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return fail(HIPATTN_HIP_ERROR, "quantize_rows: %s", hipGetErrorString(e));
    return HIPATTN_OK;
}

}  // namespace hipops
