// Rows as e4m3 codes with a scale for each 128 columns (hipops_quantize_fp8): what stands ahead of a projection in 8-bit floating point,
// with the RMS norm or the GLU that the layer has there on the way.
//
// HBM-bound: x read once, a byte an element and four a block written.  Eight elements to a lane, so sixteen lanes share a block and its
// largest magnitude.  Without a norm a block is all that a code depends on: a wavefront takes 512 columns of some rows.  Behind a norm a
// row's lanes hold it in registers over the sum of its squares.
// Measured: 8,192 x 4,096 plain 17.5 us (5.8 TB/s), the GLU of 18,006 x 2 x 2,048 37 (5.0 TB/s); two or four rows to a wavefront 41 and 54.  One row behind a norm
// 2.7: a launch and a chain of load, sum, largest magnitude and store.  Widths that are no whole eights: 4,000 x 4,097 12.1 (4,096 columns: 10.2), a block to a
// wavefront's two elements a lane 24.6.
#include <type_traits>

#include "ops/fp8.hpp"

namespace hipops {

namespace {

__device__ __forceinline__ float scale_of_peak(float peak) {
    const float s = peak * (1.0f / kFp8Largest);
    return s < 1e-30f ? 0.0f : s;
}
__device__ __forceinline__ float clamped(float y) { return __builtin_amdgcn_fmed3f(y, -kFp8Largest, kFp8Largest); }
// four codes, to nearest even (the conversion does not saturate: its operands are clamped)
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inverse) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(clamped(a * inverse), clamped(b * inverse), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(clamped(c * inverse), clamped(d * inverse), w, true);
}
__device__ __forceinline__ float inverse_rms(const QuantizeFp8Params& p, float sq) {
    const float square = sq / (float)p.width + p.eps;
    return square == 0.0f ? 0.0f : 1.0f / sqrtf(square);
}
__device__ __forceinline__ bool real_row(const QuantizeFp8Params& p, int64_t row) {
    if (row >= p.rows) return false;
    return p.row_limit == nullptr || (p.row_first + row >= (int64_t)*p.row_begin && p.row_first + row < (int64_t)*p.row_limit);
}
// another lane's number, without the way through LDS that a shuffle takes; 0 in rows of lanes that the control leaves out
template <int kControl, int kRows>
__device__ __forceinline__ float from_lane(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), kControl, kRows, 0xf, false));
}
// the largest of sixteen neighbouring lanes (turned by eight, four, two, one)
__device__ __forceinline__ float max_of_16(float v) {
    v = fmaxf(v, from_lane<0x128, 0xf>(v));
    v = fmaxf(v, from_lane<0x124, 0xf>(v));
    v = fmaxf(v, from_lane<0x122, 0xf>(v));
    return fmaxf(v, from_lane<0x121, 0xf>(v));
}
// the sum of all lanes (from one, two, four, eight lanes below within sixteen, then from the end of the sixteen below, and of the 32)
__device__ __forceinline__ float sum_of_64(float v) {
    v += from_lane<0x111, 0xf>(v);
    v += from_lane<0x112, 0xf>(v);
    v += from_lane<0x114, 0xf>(v);
    v += from_lane<0x118, 0xf>(v);
    v += from_lane<0x142, 0xa>(v);
    v += from_lane<0x143, 0xc>(v);
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}
__device__ __forceinline__ float peak_of(const Float8& y) {
    float peak = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) peak = fmaxf(peak, fabsf(y.v[e]));
    return peak;
}
// eight elements, or (kRest: widths that are no whole eights, which cost others 3 %) the `count` that are left of a row, and zeros
template <bool kRest>
__device__ __forceinline__ Raw8 load_some8(const void* base, int64_t idx, int dtype, int64_t count) {
    if (!kRest || count >= 8) return load_raw8(base, idx, dtype);
    Raw8 r = {};
#pragma unroll
    for (int e = 0; e < 7; e++) {
        if (e >= count) break;
        if (dtype == HIPATTN_F32) {
            const uint32_t v = ((const uint32_t*)base)[idx + e];
            e < 4 ? r.lo[e & 3] = v : r.hi[e & 3] = v;
        } else {
            r.lo[e >> 1] |= (uint32_t)((const uint16_t*)base)[idx + e] << (16 * (e & 1));
        }
    }
    return r;
}
// the codes of one chunk of eight, and the block's scale by the lane that has its first
template <bool kRest>
__device__ __forceinline__ void store_chunk(const QuantizeFp8Params& p, int64_t row, int64_t chunk, const Float8& y, float scale, float inverse) {
    const float* const v = y.v;
    const uint32_t codes[2] = {codes4(v[0], v[1], v[2], v[3], inverse), codes4(v[4], v[5], v[6], v[7], inverse)};
    uint8_t* const to = p.codes + row * p.width + 8 * chunk;
    const int64_t count = p.width - 8 * chunk;
    if (!kRest || count >= 8) {
        __builtin_memcpy(to, codes, 8);
    } else {
#pragma unroll
        for (int e = 0; e < 7; e++)
            if (e < count) to[e] = (uint8_t)(codes[e >> 2] >> (8 * (e & 3)));
    }
    if ((chunk & 15) == 0) p.scales[row * p.scale_row + (chunk >> 4) * p.scale_block] = scale;
}

// Without a norm: 64 chunks of a row to a wavefront, four rows to a workgroup.  Rows at any address, of any width (the last chunk's elements one by one).
template <int kSource, bool kRest>
__global__ __launch_bounds__(256) void quantize_fp8_kernel(QuantizeFp8Params p) {
    const int64_t row = 4 * (int64_t)blockIdx.x + (threadIdx.x >> 6), chunk = 64 * (int64_t)blockIdx.y + (threadIdx.x & 63);
    if (!real_row(p, row)) return;
    const bool there = 8 * chunk < p.width;
    Float8 y = {};
    if (there) {
        const int64_t at = row * p.x_row_stride + 8 * chunk, count = p.width - 8 * chunk;
        if constexpr (kSource == HIPOPS_QUANTIZE_GLU) {
            const Raw8 gate = load_some8<kRest>(p.x, at + (p.gate_first ? 0 : p.width), p.x_dtype, count), up = load_some8<kRest>(p.x, at + (p.gate_first ? p.width : 0), p.x_dtype, count);
            const Float8 g = float8_of(gate, p.x_dtype), u = float8_of(up, p.x_dtype);
#pragma unroll
            for (int e = 0; e < 8; e++) y.v[e] = gated(g.v[e], p.activation) * u.v[e];
        } else {
            y = float8_of(load_some8<kRest>(p.x, at, p.x_dtype, count), p.x_dtype);
        }
    }
    const float scale = scale_of_peak(max_of_16(peak_of(y)));
    if (there) store_chunk<kRest>(p, row, chunk, y, scale, scale > 0.0f ? 1.0f / scale : 0.0f);
}

// Behind a norm: a row to a workgroup, kKeep chunks a lane.  y = (x gamma) / rms(x): the codes are x gamma times one number a block.
constexpr int kMaxWaves = 16;
template <int kKeep, bool kRest>
__global__ __launch_bounds__(64 * kMaxWaves) void quantize_fp8_norm_kernel(QuantizeFp8Params p) {
    __shared__ float partial[kMaxWaves];
    const int64_t row = blockIdx.x;
    if (!real_row(p, row)) return;
    const int lane = threadIdx.x, lanes = blockDim.x, chunks = (int)((p.width + 7) / 8), waves = lanes >> 6;
    Float8 y[kKeep];
    Raw8 x[kKeep], gamma[kKeep];
    float sq = 0.0f;
#pragma unroll
    for (int c = 0; c < kKeep; c++) {
        const int chunk = lane + c * lanes;
        x[c] = gamma[c] = Raw8{};  // (zeros of any type)
        if (chunk < chunks) x[c] = load_some8<kRest>(p.x, row * p.x_row_stride + 8 * (int64_t)chunk, p.x_dtype, p.width - 8 * (int64_t)chunk);
        if (p.gamma != nullptr && chunk < chunks) gamma[c] = load_some8<kRest>(p.gamma, 8 * (int64_t)chunk, p.gamma_dtype, p.width - 8 * (int64_t)chunk);
    }
#pragma unroll
    for (int c = 0; c < kKeep; c++) {
        y[c] = float8_of(x[c], p.x_dtype);
#pragma unroll
        for (int e = 0; e < 8; e++) sq = fmaf(y[c].v[e], y[c].v[e], sq);
        if (p.gamma != nullptr) {
            const Float8 g = float8_of(gamma[c], p.gamma_dtype);
#pragma unroll
            for (int e = 0; e < 8; e++) y[c].v[e] *= g.v[e];
        }
    }
    sq = sum_of_64(sq);
    float peak[kKeep];
#pragma unroll
    for (int c = 0; c < kKeep; c++) peak[c] = max_of_16(peak_of(y[c]));
    if (waves > 1) {
        if ((lane & 63) == 0) partial[lane >> 6] = sq;
        __syncthreads();
        sq = 0.0f;
        for (int w = 0; w < waves; w++) sq += partial[w];
    }
    const float inv = inverse_rms(p, sq);
#pragma unroll
    for (int c = 0; c < kKeep; c++) {
        const int chunk = lane + c * lanes;
        const float scale = scale_of_peak(peak[c] * inv);
        if (chunk < chunks) store_chunk<kRest>(p, row, chunk, y[c], scale, scale > 0.0f ? inv * (1.0f / scale) : 0.0f);
    }
}

// Rows that are too wide for these (behind a norm 32,768): a row to a workgroup, a block to a wavefront; behind a norm the row is read twice.
template <int kSource>
__device__ __forceinline__ float value1(const QuantizeFp8Params& p, int64_t at, int64_t i) {
    if constexpr (kSource != HIPOPS_QUANTIZE_GLU) return load_scalar(p.x, at + i, p.x_dtype);
    return gated(load_scalar(p.x, at + (p.gate_first ? 0 : p.width) + i, p.x_dtype), p.activation) *
           load_scalar(p.x, at + (p.gate_first ? p.width : 0) + i, p.x_dtype);
}
template <int kSource>
__global__ __launch_bounds__(256) void quantize_fp8_scalar_kernel(QuantizeFp8Params p) {
    __shared__ float partial[4];
    const int64_t row = blockIdx.x, at = row * p.x_row_stride;
    if (!real_row(p, row)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float inv = 1.0f;
    if constexpr (kSource == HIPOPS_QUANTIZE_RMS_NORM) {
        float sq = 0.0f;
        for (int64_t i = threadIdx.x; i < p.width; i += 256) {
            const float x = value1<kSource>(p, at, i);
            sq = fmaf(x, x, sq);
        }
        sq = wave_sum(sq);
        if (lane == 0) partial[wave] = sq;
        __syncthreads();
        inv = inverse_rms(p, partial[0] + partial[1] + partial[2] + partial[3]);
    }
    const int64_t blocks = (p.width + kFp8Block - 1) / kFp8Block;
    for (int64_t b = wave; b < blocks; b += 4) {
        float y[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int64_t i = b * kFp8Block + 64 * e + lane;
            y[e] = i < p.width ? value1<kSource>(p, at, i) : 0.0f;
            if constexpr (kSource == HIPOPS_QUANTIZE_RMS_NORM)
                if (p.gamma != nullptr && i < p.width) y[e] *= load_scalar(p.gamma, i, p.gamma_dtype);
        }
        const float scale = scale_of_peak(wave_max(fmaxf(fabsf(y[0]), fabsf(y[1]))) * inv);
        const float inverse = scale > 0.0f ? inv * (1.0f / scale) : 0.0f;
        if (lane == 0) p.scales[row * p.scale_row + b * p.scale_block] = scale;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int64_t i = b * kFp8Block + 64 * e + lane;
            if (i < p.width) p.codes[row * p.width + i] = (uint8_t)codes4(y[e], 0.0f, 0.0f, 0.0f, inverse);
        }
    }
}

// `per_group` rows to a workgroup of `lanes`, `columns` workgroups to a row.  A launch of 2^32 threads or more runs modulo 2^32 of them,
// without an error: more rows go in several.
template <typename Kernel>
void launch_in_runs(Kernel kernel, const QuantizeFp8Params& all, int64_t per_group, int lanes, int64_t columns, hipStream_t stream) {
    const int64_t most = (0xffffffffLL / (lanes * columns)) * per_group;
    for (int64_t first = 0; first < all.rows; first += most) {
        QuantizeFp8Params p = all;
        p.rows = all.rows - first < most ? all.rows - first : most;
        p.x = (const uint8_t*)all.x + first * all.x_row_stride * (all.x_dtype == HIPATTN_F32 ? 4 : 2);
        p.codes += first * all.width;
        p.scales += first * all.scale_row;
        p.row_first += first;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((p.rows + per_group - 1) / per_group), (unsigned)columns), dim3((unsigned)lanes), 0, stream, p);
    }
}

bool float_dtype(int d) { return d == HIPATTN_F32 || d == HIPATTN_F16 || d == HIPATTN_BF16; }

}  // namespace

hipError_t launch_quantize_fp8(int source, const QuantizeFp8Params& p, hipStream_t stream) {
    const bool norm = source == HIPOPS_QUANTIZE_RMS_NORM;
    const bool vector = p.width <= (norm ? 32768 : (int64_t)1 << 24);
    const int64_t chunks = (p.width + 7) / 8;
    if (!vector) {
        if (norm)
            launch_in_runs(quantize_fp8_scalar_kernel<HIPOPS_QUANTIZE_RMS_NORM>, p, 1, 256, 1, stream);
        else if (source == HIPOPS_QUANTIZE_GLU)
            launch_in_runs(quantize_fp8_scalar_kernel<HIPOPS_QUANTIZE_GLU>, p, 1, 256, 1, stream);
        else
            launch_in_runs(quantize_fp8_scalar_kernel<HIPOPS_QUANTIZE_PLAIN>, p, 1, 256, 1, stream);
        return hipGetLastError();
    }
    const auto launch = [&](auto rest) {
        constexpr bool kRest = decltype(rest)::value != 0;
        const int64_t columns = (chunks + 63) / 64;
        if (source == HIPOPS_QUANTIZE_GLU) {
            launch_in_runs(quantize_fp8_kernel<HIPOPS_QUANTIZE_GLU, kRest>, p, 4, 256, columns, stream);
        } else if (!norm) {
            launch_in_runs(quantize_fp8_kernel<HIPOPS_QUANTIZE_PLAIN, kRest>, p, 4, 256, columns, stream);
        } else {
            const int keep = chunks <= 512 ? 1 : chunks <= 1024 ? 2 : 4;
            const int lanes = (int)((chunks + 64 * keep - 1) / (64 * keep) * 64);
            if (keep == 1)
                launch_in_runs(quantize_fp8_norm_kernel<1, kRest>, p, 1, lanes, 1, stream);
            else if (keep == 2)
                launch_in_runs(quantize_fp8_norm_kernel<2, kRest>, p, 1, lanes, 1, stream);
            else
                launch_in_runs(quantize_fp8_norm_kernel<4, kRest>, p, 1, lanes, 1, stream);
        }
    };
    if (p.width % 8)
        launch(std::true_type{});
    else
        launch(std::false_type{});
    return hipGetLastError();
}

hipattn_status quantize_fp8(const hipops_quantize_fp8_desc* d, const void* x, const void* gamma, uint8_t* codes, float* scales, hipStream_t stream) {
    if (!d) return fail(HIPATTN_INVALID_ARGUMENT, "quantize_fp8: null descriptor");
    if (d->source < HIPOPS_QUANTIZE_PLAIN || d->source > HIPOPS_QUANTIZE_GLU) return fail(HIPATTN_INVALID_ARGUMENT, "quantize_fp8: source %d", d->source);
    const bool norm = d->source == HIPOPS_QUANTIZE_RMS_NORM, glu = d->source == HIPOPS_QUANTIZE_GLU;
    if (d->rows < 0 || d->width <= 0 || d->width > (int64_t)1 << 28)
        return fail(HIPATTN_INVALID_ARGUMENT, "quantize_fp8: rows %lld width %lld", (long long)d->rows, (long long)d->width);
    if (d->rows > 0x7fffffffLL) return fail(HIPATTN_UNSUPPORTED, "quantize_fp8: too many rows");
    if (!float_dtype(d->x_dtype) || (norm && gamma && !float_dtype(d->gamma_dtype)))
        return fail(HIPATTN_UNSUPPORTED, "quantize_fp8: types must be f32, f16 or bf16");
    if (glu && (d->glu_activation < HIPOPS_GLU_SWISH || d->glu_activation > HIPOPS_GLU_GELU_TANH))
        return fail(HIPATTN_INVALID_ARGUMENT, "quantize_fp8: activation %d", d->glu_activation);
    if (norm && !(d->eps >= 0.0f)) return fail(HIPATTN_INVALID_ARGUMENT, "quantize_fp8: eps must be >= 0");
    const int64_t taken = glu ? 2 * d->width : d->width, blocks = (d->width + kFp8Block - 1) / kFp8Block;
    if (d->x_row_stride != 0 && d->x_row_stride < taken)
        return fail(HIPATTN_INVALID_ARGUMENT, "quantize_fp8: rows of %lld elements, %lld apart", (long long)taken, (long long)d->x_row_stride);
    const int64_t row = d->scale_row_stride, block = d->scale_block_stride;
    if (row > (int64_t)1 << 40 || block > (int64_t)1 << 40) return fail(HIPATTN_UNSUPPORTED, "quantize_fp8: scales %lld and %lld apart", (long long)row, (long long)block);
    if (row < 0 || block < 0 || ((row == 0) != (block == 0)) || (row && !(row >= blocks * block || block / row >= d->rows)))
        return fail(HIPATTN_INVALID_ARGUMENT, "quantize_fp8: scales of %lld rows and %lld blocks overlap, %lld and %lld apart", (long long)d->rows, (long long)blocks,
                    (long long)row, (long long)block);
    if (d->rows == 0) return HIPATTN_OK;
    if (!x || !codes || !scales) return fail(HIPATTN_INVALID_ARGUMENT, "quantize_fp8: null pointer");
    const QuantizeFp8Params p{x, gamma, codes, scales, d->rows, d->width, d->x_row_stride ? d->x_row_stride : taken, row ? row : 1, row ? block : d->rows,
                              d->x_dtype, d->gamma_dtype, d->glu_activation, d->glu_gate_first, d->eps, nullptr, nullptr, 0};
    if (const hipError_t e = launch_quantize_fp8(d->source, p, stream); e != hipSuccess) return fail(HIPATTN_HIP_ERROR, "quantize_fp8: %s", hipGetErrorString(e));
    return HIPATTN_OK;
}

}  // namespace hipops
