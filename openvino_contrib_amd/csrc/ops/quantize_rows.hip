// Rows as 8-bit codes with a scale each (hipops_quantize_rows): what stands ahead of an 8-bit projection, with the RMS norm or the
// GLU that the layer has there on the way, so that neither goes through memory in 16 bits.
//
// HBM-bound: x read once, a byte an element written.  A workgroup takes a row and keeps it in registers (eight elements to a
// chunk, kKeep chunks a lane) over its reductions: the norm's sum of squares, then the largest magnitude.
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

__device__ __forceinline__ float scale_of_peak(float peak) {
    const float s = peak * (1.0f / 127.0f);
    return s < 1e-30f ? 0.0f : s;
}
__device__ __forceinline__ int code_of(float y, float inverse) { return (int)fminf(fmaxf(rintf(y * inverse), -127.0f), 127.0f); }

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

template <int kSource>
__device__ __forceinline__ Float8 values8(const QuantizeParams& p, int64_t at, int64_t i) {
    if constexpr (kSource != HIPOPS_QUANTIZE_GLU) {
        return load8(p.x, at + i, p.x_dtype);
    } else {
        const Float8 gate = load8(p.x, at + (p.gate_first ? 0 : p.width) + i, p.x_dtype), up = load8(p.x, at + (p.gate_first ? p.width : 0) + i, p.x_dtype);
        Float8 y;
#pragma unroll
        for (int e = 0; e < 8; e++) y.v[e] = activate(gate.v[e], p.activation, 1.0f) * up.v[e];
        return y;
    }
}

template <int kSource, int kKeep>
__global__ __launch_bounds__(64 * kMaxWaves) void quantize_rows_kernel(QuantizeParams p) {
    __shared__ float sums[kMaxWaves], peaks[kMaxWaves];
    const int64_t row = blockIdx.x, at = row * p.x_row_stride;
    const int chunks = (int)(p.width / 8);
    Float8 y[kKeep];
    float sq = 0.0f, peak = 0.0f;
#pragma unroll
    for (int c = 0; c < kKeep; c++) {
        const int chunk = (int)threadIdx.x + c * (int)blockDim.x;
        if (chunk < chunks) {
            y[c] = values8<kSource>(p, at, 8 * (int64_t)chunk);
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++) y[c].v[e] = 0.0f;
        }
    }
    if constexpr (kSource == HIPOPS_QUANTIZE_RMS_NORM) {
#pragma unroll
        for (int c = 0; c < kKeep; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) sq = fmaf(y[c].v[e], y[c].v[e], sq);
        sq = reduce<false>(sq, sums);
        const float inv = 1.0f / sqrtf(sq / (float)p.width + p.eps);
#pragma unroll
        for (int c = 0; c < kKeep; c++) {
            const int chunk = (int)threadIdx.x + c * (int)blockDim.x;
            Float8 g;
            if (p.gamma != nullptr && chunk < chunks) g = load8(p.gamma, 8 * (int64_t)chunk, p.gamma_dtype);
#pragma unroll
            for (int e = 0; e < 8; e++) y[c].v[e] *= inv;
            if (p.gamma != nullptr && chunk < chunks) {
#pragma unroll
                for (int e = 0; e < 8; e++) y[c].v[e] *= g.v[e];
            }
        }
    }
#pragma unroll
    for (int c = 0; c < kKeep; c++)
#pragma unroll
        for (int e = 0; e < 8; e++) peak = fmaxf(peak, fabsf(y[c].v[e]));
    const float scale = scale_of_peak(reduce<true>(peak, peaks));
    const float inverse = scale > 0.0f ? 1.0f / scale : 0.0f;
    if (threadIdx.x == 0) p.scales[row] = scale;
#pragma unroll
    for (int c = 0; c < kKeep; c++) {
        const int chunk = (int)threadIdx.x + c * (int)blockDim.x;
        if (chunk >= chunks) break;
        uint32_t w[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            int q[4];
#pragma unroll
            for (int e = 0; e < 4; e++) q[e] = code_of(y[c].v[4 * h + e], inverse);
            w[h] = (uint32_t)(q[0] & 255) | ((uint32_t)(q[1] & 255) << 8) | ((uint32_t)(q[2] & 255) << 16) | ((uint32_t)q[3] << 24);
        }
        *(uint2*)(p.codes + row * p.width + 8 * (int64_t)chunk) = make_uint2(w[0], w[1]);
    }
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
        inv = 1.0f / sqrtf(reduce<false>(sq, sums) / (float)p.width + p.eps);
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

template <int kSource>
void launch(const QuantizeParams& p, bool vector, hipStream_t stream) {
    const dim3 grid((unsigned)p.rows);
    if (!vector) {
        hipLaunchKernelGGL(quantize_rows_scalar_kernel<kSource>, grid, dim3(256), 0, stream, p);
        return;
    }
    // one chunk a lane up to 512 lanes, then more chunks
    const int64_t chunks = p.width / 8;
    const int keep = chunks <= 512 ? 1 : chunks <= 1024 ? 2 : 4;
    const dim3 block((unsigned)((chunks + 64 * keep - 1) / (64 * keep) * 64));
    if (keep == 1)
        hipLaunchKernelGGL((quantize_rows_kernel<kSource, 1>), grid, block, 0, stream, p);
    else if (keep == 2)
        hipLaunchKernelGGL((quantize_rows_kernel<kSource, 2>), grid, block, 0, stream, p);
    else
        hipLaunchKernelGGL((quantize_rows_kernel<kSource, 4>), grid, block, 0, stream, p);
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
