// Routing to experts and the sum over a token's experts (hipops_route_experts, hipops_combine_experts).
#include <algorithm>
#include <cmath>

#include "ops/fp8.hpp"

namespace hipops {

namespace {

// ---- routing -----------------------------------------------------------------------------------------
// Bound by latency: a token is a kilobyte of logits, and then a chain of reductions, one for each choice.  A wavefront takes a token, kEach experts a
// lane (expert 64 i + lane).  Choices are compared as whole numbers in the order of the fp64 values, upper halves first: a reduction of 32 bits over the
// lanes, and a second one where several lanes share the upper half.  A softmax's scores without a bias (and without sums of two) have the order of the
// logits, and no exponential stands in front of it.
// Measured: one token of 64 experts 4.6 us, 64 tokens of 256 experts in groups (8 of them, sigmoid) 8.4 and 4.4 for the lists, 8,192 tokens 21.3 and 8.7: by then some 940
// vector instructions a token at four wavefronts a SIMD, which wait half of their time on one another's results.
struct RouteParams {
    const void* logits;
    const float* bias;
    int32_t* indices;
    float* weights;
    int32_t* begins;
    int32_t* order;
    int32_t* slots;
    uint8_t* counts;  // [runs][count_stride]: the pairs of each expert in a run
    int64_t tokens, row_stride;
    int run;  // tokens of a workgroup
    int count_stride;
    int dtype, score, renormalise, experts, top_k, groups, kept, group_top;
    float scale;
};
constexpr double kNoScore = -745.2;  // (exponentials below this are 0 in fp64)
constexpr int kRouteWaves = 16, kMostExperts = 1024, kMaskTokens = 32;

// a number whose order is that of the values (which are no NaN); zeros are alike
__device__ __forceinline__ uint64_t key_of(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
template <int kControl, int kRows>
__device__ __forceinline__ uint32_t max_with(uint32_t v) {
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kControl, kRows, 0xf, false));
}
// the largest of all lanes
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    v = max_with<0x111, 0xf>(v);  // from one, two, four, eight lanes below, within sixteen
    v = max_with<0x112, 0xf>(v);
    v = max_with<0x114, 0xf>(v);
    v = max_with<0x118, 0xf>(v);
    v = max_with<0x142, 0xa>(v);  // from the end of the sixteen below, and of the 32
    v = max_with<0x143, 0xc>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// One token by a wavefront: lane j < top_k returns its j-th expert and writes it and its weight.  `scratch`: a double for each expert, of this wavefront.
template <int kEach>
__device__ __forceinline__ int route_token(const RouteParams& p, int64_t token, int lane, double* scratch) {
    const double lowest = -INFINITY;
    const bool by_logits = p.score == HIPOPS_ROUTE_SOFTMAX && p.bias == nullptr && (p.groups == 1 || p.group_top == 1);  // (the same for all)
    double logit[kEach], score[kEach];
    uint64_t key[kEach];  // 0: not to be had
    // (all loads of a type in one run of code: a choice of the type at each would have every one waited for before the next)
    float x[kEach], bias[kEach];
    const int64_t row = token * p.row_stride;
#pragma unroll
    for (int i = 0; i < kEach; i++) x[i] = -INFINITY, bias[i] = 0.0f;
    if (p.bias != nullptr) {
#pragma unroll
        for (int i = 0; i < kEach; i++)
            if (64 * i + lane < p.experts) bias[i] = p.bias[64 * i + lane];
    }
    if (p.dtype == HIPATTN_F32) {
#pragma unroll
        for (int i = 0; i < kEach; i++)
            if (64 * i + lane < p.experts) x[i] = ((const float*)p.logits)[row + 64 * i + lane];
    } else {
        uint16_t raw[kEach];
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            raw[i] = 0;
            if (64 * i + lane < p.experts) raw[i] = ((const uint16_t*)p.logits)[row + 64 * i + lane];
        }
#pragma unroll
        for (int i = 0; i < kEach; i++)
            if (64 * i + lane < p.experts) x[i] = p.dtype == HIPATTN_F16 ? f16_bits_to_float(raw[i]) : bf16_bits_to_float(raw[i]);
    }
    uint32_t highest = 0;
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        x[i] = x[i] == x[i] ? fminf(x[i], 3.4028234663852886e38f) : -INFINITY;
        logit[i] = (double)x[i];
        const uint32_t u = __float_as_uint(x[i]);
        highest = max(highest, u >> 31 ? ~u : u | 0x80000000u);
    }
    double most = 0.0, total = 1.0;
    if (p.score == HIPOPS_ROUTE_SOFTMAX) {
        const uint32_t u = wave_max_u32(highest);
        most = (double)__uint_as_float(u >> 31 ? u & 0x7fffffffu : ~u);
    }
    const auto score_of = [&](double x) __attribute__((always_inline)) -> double {  // before the division by the total
        if (p.score == HIPOPS_ROUTE_SIGMOID) return 1.0 / (1.0 + exp(-x));
        return x == lowest ? 0.0 : exp(x - most);
    };
    if (by_logits) {
        if (!p.renormalise) {
            total = 0.0;  // (a sum of fp32 exponentials: the weights are fp32)
#pragma unroll
            for (int i = 0; i < kEach; i++) total += logit[i] == lowest ? 0.0 : (double)expf((float)(logit[i] - most));
            total = wave_sum64(total);
        }
#pragma unroll
        for (int i = 0; i < kEach; i++) score[i] = logit[i] - most < kNoScore ? lowest : logit[i];
    } else {
#pragma unroll
        for (int i = 0; i < kEach; i++) score[i] = score_of(logit[i]);
        if (p.score == HIPOPS_ROUTE_SOFTMAX) {
            total = 0.0;
#pragma unroll
            for (int i = 0; i < kEach; i++) total += score[i];
            total = wave_sum64(total);
#pragma unroll
            for (int i = 0; i < kEach; i++) score[i] = total > 0.0 ? score[i] / total : 0.0;
        }
    }
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        const int e = 64 * i + lane;
        double choice = score[i];
        if (p.bias != nullptr) choice += (double)bias[i];
        key[i] = e < p.experts ? key_of(choice == choice ? choice : lowest) : 0;
        scratch[e] = by_logits || p.groups == 1 ? score[i] : choice == choice ? choice : lowest;
    }
    __builtin_amdgcn_wave_barrier();
    if (p.groups > 1) {
        // a group's best two by some lanes each, a power of two of them
        const int size = p.experts / p.groups, parts = 1 << (31 - __builtin_clz(64 / p.groups));
        const int group = lane / parts, part = lane & (parts - 1);
        double first = lowest, second = lowest;
        if (group < p.groups) {
            for (int j = part; j < size; j += parts) {
                const double c = scratch[group * size + j];
                second = fmax(second, fmin(first, c));
                first = fmax(first, c);
            }
        }
        for (int off = 1; off < parts; off <<= 1) {
            const double a = __shfl_xor(first, off, 64), b = __shfl_xor(second, off, 64);
            second = fmax(fmin(first, a), fmax(second, b));
            first = fmax(first, a);
        }
        double best = p.group_top == 2 && size > 1 ? first + second : first;
        if (!(best == best)) best = lowest;  // (infinities of both signs)
        const uint64_t mine = key_of(best);
        int ahead = 0;
        for (int g = 0; g < p.groups; g++) {
            const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), g * parts) << 32 |
                                   (uint32_t)__builtin_amdgcn_readlane((int)mine, g * parts);
            ahead += other > mine || (other == mine && g < group);
        }
        const uint64_t kept = __ballot(part == 0 && group < p.groups && ahead < p.kept);
#pragma unroll
        for (int i = 0; i < kEach; i++)
            if (key[i] != 0 && !(kept >> ((64 * i + lane) / size * parts) & 1)) key[i] = 0;
        if (!by_logits) {  // the scores, for the choices that stood there
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int i = 0; i < kEach; i++) scratch[64 * i + lane] = score[i];
            __builtin_amdgcn_wave_barrier();
        }
    }
    int taken = 0;
    for (int j = 0; j < p.top_k; j++) {
        uint64_t head = key[0];
        int at = lane;
#pragma unroll
        for (int i = 1; i < kEach; i++)
            if (key[i] > head) head = key[i], at = 64 * i + lane;
        const uint32_t upper = (uint32_t)(head >> 32), largest = wave_max_u32(upper);
        uint64_t among = __ballot(upper == largest);
        if (__popcll(among) > 1) {
            const uint32_t lower = upper == largest ? (uint32_t)head : 0u, of_those = wave_max_u32(lower);
            among = __ballot(upper == largest && lower == of_those);
        }
        int found;
        if (__popcll(among) == 1) {
            found = __builtin_amdgcn_readlane(at, __builtin_ctzll(among));
        } else {  // equal choices: the lowest index
            found = (int)(0x7fffffffu - wave_max_u32(among >> lane & 1 ? 0x7fffffffu - (uint32_t)at : 0u));
        }
        if (lane == j) taken = found;
#pragma unroll
        for (int i = 0; i < kEach; i++)
            if (found == 64 * i + lane) key[i] = 0;
    }
    double mine = 0.0;
    if (lane < p.top_k) mine = by_logits ? score_of(scratch[taken]) : scratch[taken];
    if (by_logits && !p.renormalise) mine = total > 0.0 ? mine / total : 0.0;
    double sum = 1.0;
    if (p.renormalise) {
        sum = 0.0;
        for (int j = 0; j < p.top_k; j++) {
            const uint64_t u = (uint64_t)__double_as_longlong(mine);
            sum += __longlong_as_double((long long)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), j) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)u, j)));
        }
    }
    if (lane < p.top_k) {
        p.indices[token * p.top_k + lane] = taken;
        p.weights[token * p.top_k + lane] = sum > 0.0 ? (float)(mine / sum * (double)p.scale) : 0.0f;
    }
    return taken;
}

// ---- the lists ---------------------------------------------------------------------------------------
// The pairs of up to 32 tokens from token t0 on, pair threadIdx.x + blockDim.x i of theirs with expert expert[i]; `next[e]` is the place of expert e's
// first.  A token has an expert once at most, so a mask of the tokens for each expert has a pair's rank among them; masks, as counts, do not mind the
// order in which they are made.
constexpr int kMostPairs = 64 * kMaskTokens;
template <int kPairs>
__device__ __forceinline__ void place_pairs(const RouteParams& p, int64_t t0, int pairs, const int (&expert)[kPairs], int* next, uint32_t* masks) {
    const int threads = (int)blockDim.x, thread = threadIdx.x;
    for (int e = thread; e < p.experts; e += threads) masks[e] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPairs; i++)
        if (thread + i * threads < pairs) atomicOr(&masks[expert[i]], 1u << ((thread + i * threads) / p.top_k));
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPairs; i++) {
        const int at = thread + i * threads;
        if (at >= pairs) break;
        const int64_t pair = t0 * p.top_k + at;
        const int to = next[expert[i]] + __popc(masks[expert[i]] & ((1u << (at / p.top_k)) - 1));
        p.order[to] = (int32_t)pair;
        p.slots[pair] = to;
    }
}
template <int kControl, int kRows>
__device__ __forceinline__ int add_with(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, kControl, kRows, 0xf, false);
}
// next[e] += the pairs of the experts before e, of which all[] has the numbers; the first workgroup writes them down as begins
__device__ __forceinline__ void scan_experts(const RouteParams& p, const int* all, int* next) {
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x, each = (p.experts + 63) >> 6;
        int sum = 0;
        for (int i = 0; i < each; i++) sum += lane * each + i < p.experts ? all[lane * each + i] : 0;
        int until = add_with<0x111, 0xf>(sum);
        until = add_with<0x112, 0xf>(until);
        until = add_with<0x114, 0xf>(until);
        until = add_with<0x118, 0xf>(until);
        until = add_with<0x142, 0xa>(until);
        until = add_with<0x143, 0xc>(until);
        int before = until - sum;
        for (int i = 0; i < each; i++) {
            const int e = lane * each + i;
            if (e >= p.experts) break;
            next[e] += before;
            if (blockIdx.x == 0) p.begins[e] = before;
            before += all[e];
        }
        if (blockIdx.x == 0 && lane == 63) p.begins[p.experts] = until;
    }
    __syncthreads();
}

// A workgroup takes a run of tokens and counts its pairs; with one run, and lists wanted, it makes them too.
template <int kEach>
__global__ __launch_bounds__(64 * kRouteWaves) void route_kernel(RouteParams p) {
    __shared__ double scratch[kRouteWaves][64 * kEach];
    __shared__ int count[64 * kEach], next[64 * kEach], chosen[64 * kRouteWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = (int)blockDim.x >> 6;
    const int64_t first = (int64_t)blockIdx.x * p.run, last = min(first + p.run, p.tokens);
    const bool lists = p.begins != nullptr, alone = gridDim.x == 1;
    if (lists) {
        for (int e = threadIdx.x; e < p.experts; e += (int)blockDim.x) count[e] = next[e] = 0;
        __syncthreads();
    }
    for (int64_t token = first + wave; token < last; token += waves) {
        const int taken = route_token<kEach>(p, token, lane, scratch[wave]);
        if (lists && lane < p.top_k) {
            atomicAdd(&count[taken], 1);
            if (alone) chosen[token * p.top_k + lane] = taken;  // (a run that is alone has a wavefront for each token)
        }
        __builtin_amdgcn_wave_barrier();
    }
    if (!lists) return;
    __syncthreads();
    if (alone) {
        scan_experts(p, count, next);
        const int pairs = (int)p.tokens * p.top_k;
        const int expert[1] = {(int)threadIdx.x < pairs ? chosen[threadIdx.x] : 0};
        place_pairs<1>(p, 0, pairs, expert, next, (uint32_t*)count);
    } else {
        for (int e = threadIdx.x; e < p.count_stride; e += (int)blockDim.x) p.counts[(int64_t)blockIdx.x * p.count_stride + e] = e < p.experts ? (uint8_t)count[e] : 0;
    }
}

// A workgroup adds up every expert's pairs in all runs and in those before its own, which together say where its own pairs go.
constexpr int kListThreads = 1024;
__global__ __launch_bounds__(kListThreads) void expert_lists_kernel(RouteParams p) {
    __shared__ int all[kMostExperts], next[kMostExperts];
    constexpr int kPairs = kMostPairs / kListThreads;
    const int thread = threadIdx.x, lane = thread & 63, wave = thread >> 6, waves = kListThreads / 64;
    const int64_t first = (int64_t)blockIdx.x * p.run, last = min(first + p.run, p.tokens);
    int expert[kPairs], pairs = 0;
    const auto fetch = [&](int64_t t0) __attribute__((always_inline)) {
        pairs = (int)min((int64_t)kMaskTokens, last - t0) * p.top_k;
#pragma unroll
        for (int i = 0; i < kPairs; i++) expert[i] = thread + i * kListThreads < pairs ? p.indices[t0 * p.top_k + thread + i * kListThreads] : 0;
    };
    fetch(first);
    for (int e = thread; e < p.experts; e += kListThreads) all[e] = next[e] = 0;
    __syncthreads();
    const int runs = (int)gridDim.x, words = p.count_stride / 4;
    for (int w = lane; w < words; w += 64) {
        int sum[4] = {0, 0, 0, 0}, before[4] = {0, 0, 0, 0};
#pragma unroll 8
        for (int r = wave; r < runs; r += waves) {
            const uint32_t four = *(const uint32_t*)(p.counts + (int64_t)r * p.count_stride + 4 * w);
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const int n = (int)(four >> (8 * b) & 255u);
                sum[b] += n;
                before[b] += r < (int)blockIdx.x ? n : 0;
            }
        }
#pragma unroll
        for (int b = 0; b < 4; b++)
            if (4 * w + b < p.experts) {
                atomicAdd(&all[4 * w + b], sum[b]);
                atomicAdd(&next[4 * w + b], before[b]);
            }
    }
    __syncthreads();
    scan_experts(p, all, next);
    uint32_t* const masks = (uint32_t*)all;
    for (int64_t t0 = first;;) {
        place_pairs(p, t0, pairs, expert, next, masks);
        t0 += kMaskTokens;
        if (t0 >= last) break;
        __syncthreads();
        for (int e = thread; e < p.experts; e += kListThreads) next[e] += __popc(masks[e]);
        fetch(t0);
        __syncthreads();
    }
}

// ---- the sum over a token's experts ----------------------------------------------------------------------
struct CombineParams {
    const void* y;
    const float* weights;
    const int32_t* slots;
    const void* residual;
    void* out;
    int64_t tokens, rows, n;
    int top_k, y_dtype, out_dtype;
};

// HBM-bound: 8,192 tokens of 8 rows of 4,096 in 131 us, 5.1 TB/s; 64 tokens 4.2, a launch and three loads one behind the other.
// Eight columns a lane, rows at any address (the hardware loads 16 bytes from there), and a lane for each of the columns that are left: 4,096 tokens of 4,097
// columns 77 us, a column a lane 264.  kSize: bytes of an element of y.  kRest: there are such (more registers: 138 us in place of 131).
template <int kSize, bool kRest>
__global__ __launch_bounds__(256) void combine_kernel(CombineParams p) {
    constexpr int kAtOnce = 16 / kSize;
    const int64_t eights = p.n / 8, units = eights + p.n % 8, at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t token = at / units, unit = at - token * units, column = unit < eights ? 8 * unit : unit + 7 * eights;
    if (token >= p.tokens) return;
    const int64_t to = token * p.n + column;
    const int32_t* const slots = p.slots + token * p.top_k;
    const float* const weights = p.weights + token * p.top_k;
    const bool eight = !kRest || unit < eights;
    float sum[8];
#pragma unroll
    for (int e = 0; e < 8; e++) sum[e] = 0.0f;
    Raw8 other = {};
    if (p.residual != nullptr && eight) other = load_raw8(p.residual, to, p.out_dtype);
    for (int j0 = 0; j0 < p.top_k; j0 += kAtOnce) {  // (rows of some experts on their way at a time)
        int slot[kAtOnce];
        float w[kAtOnce];
        uint4_t y[kAtOnce][kSize / 2];
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {
            slot[u] = -1, w[u] = 0.0f;
            if (j0 + u < p.top_k) slot[u] = slots[j0 + u], w[u] = weights[j0 + u];
        }
        if (eight) {
#pragma unroll
            for (int u = 0; u < kAtOnce; u++) {
                if (slot[u] < 0 || slot[u] >= p.rows) continue;
                __builtin_memcpy(y[u], (const uint8_t*)p.y + kSize * (slot[u] * p.n + column), 8 * kSize);
            }
        } else {
#pragma unroll
            for (int u = 0; u < kAtOnce; u++) {
                if (slot[u] < 0 || slot[u] >= p.rows) continue;
                const int64_t from = slot[u] * p.n + column;
                y[u][0][0] = kSize == 4 ? ((const uint32_t*)p.y)[from] : ((const uint16_t*)p.y)[from];
            }
        }
#pragma unroll
        for (int u = 0; u < kAtOnce; u++) {  // (a lane with one column has seven more sums that nobody looks at)
            if (slot[u] < 0 || slot[u] >= p.rows) continue;
            const Float8 values = float8_of({y[u][0], y[u][kSize / 2 - 1]}, p.y_dtype);
#pragma unroll
            for (int e = 0; e < 8; e++) sum[e] = fmaf(w[u], values.v[e], sum[e]);
        }
    }
    if (!eight) {
        if (p.residual != nullptr) sum[0] += load_scalar(p.residual, to, p.out_dtype);
        store_scalar(p.out, to, p.out_dtype, sum[0]);
        return;
    }
    Float8 r = {};
    if (p.residual != nullptr) r = float8_of(other, p.out_dtype);
#pragma unroll
    for (int e = 0; e < 8; e++) r.v[e] += sum[e];
    store_loose8(p.out, to, p.out_dtype, r.v);
}

bool float_dtype(int d) { return d == HIPATTN_F32 || d == HIPATTN_F16 || d == HIPATTN_BF16; }

hipattn_status checked(const hipops_route_desc* d) {
    if (!d) return fail(HIPATTN_INVALID_ARGUMENT, "route_experts: null descriptor");
    if (!float_dtype(d->logits_dtype)) return fail(HIPATTN_UNSUPPORTED, "route_experts: logits must be f32, f16 or bf16");
    if (d->score != HIPOPS_ROUTE_SOFTMAX && d->score != HIPOPS_ROUTE_SIGMOID) return fail(HIPATTN_INVALID_ARGUMENT, "route_experts: score %d", d->score);
    if (d->tokens < 0 || d->experts < 1 || d->top_k < 1)
        return fail(HIPATTN_INVALID_ARGUMENT, "route_experts: %lld tokens, %d of %d experts", (long long)d->tokens, d->top_k, d->experts);
    if (d->experts > kMostExperts || d->top_k > 64 || d->tokens * d->top_k > 0x7fffffffLL || d->tokens > 0x7fffffffLL)
        return fail(HIPATTN_UNSUPPORTED, "route_experts: more than %d experts, 64 choices or 2^31 - 1 pairs", kMostExperts);
    int64_t reachable = d->experts;
    if (d->groups < 0) return fail(HIPATTN_INVALID_ARGUMENT, "route_experts: %d groups", d->groups);
    if (d->groups > 1) {
        if (d->groups > 64) return fail(HIPATTN_UNSUPPORTED, "route_experts: %d groups are more than 64", d->groups);
        if (d->experts % d->groups || d->kept_groups < 1 || d->kept_groups > d->groups || d->group_top < 1 || d->group_top > 2)
            return fail(HIPATTN_INVALID_ARGUMENT, "route_experts: %d of %d groups of %d experts by their best %d", d->kept_groups, d->groups, d->experts, d->group_top);
        reachable = (int64_t)d->experts / d->groups * d->kept_groups;
    }
    if (d->top_k > reachable) return fail(HIPATTN_INVALID_ARGUMENT, "route_experts: %d of %lld experts", d->top_k, (long long)reachable);
    if (d->logits_row_stride && d->logits_row_stride < d->experts)
        return fail(HIPATTN_INVALID_ARGUMENT, "route_experts: rows of %d logits, %lld apart", d->experts, (long long)d->logits_row_stride);
    return HIPATTN_OK;
}

}  // namespace

// Tokens of a run: one workgroup's; a byte counts its pairs of an expert.  Up to eight need no second launch (one token of 64 experts 5.0 us).
// A few tokens are spread out, four to a workgroup: 64 of 256 experts 12.1 us, 15.7 in a run of 16.  From 4,096 on compute units take whole
// rounds of workgroups, of which each holds one (sixteen wavefronts of 101 registers): as few rounds as leave a run at 128 tokens.  us in runs of 16, 32, 64,
// 128 and 224 tokens: 8,192 tokens 38.6, 30.0, 44.0, -, -; 16,384 87.6, 54.3, 47.2, -, -; 60,000 584, -, 183, 155, 246.  Every workgroup of the lists adds up the
// counts of all runs, so very many tokens go in the longest runs.  That grows with the square of the tokens all the same: the lists of 2^20 tokens of 256 experts
// 0.8 ms of 2.5, of 2^24 221 of 246, of 2^26 tokens of 8 experts 2,360 of 2,390.  More than 2^26 get no lists.
static constexpr int64_t kMostListTokens = (int64_t)1 << 26;
static int run_of(int64_t tokens) {
    if (tokens <= 8) return (int)std::max<int64_t>(tokens, 1);
    if (tokens <= 1024) return 4;
    if (tokens <= 4096) return 16;
    if (tokens > 1 << 18) return 224;
    const int64_t round = 4096 * ((tokens + 32767) / 32768);
    return (int)(16 * ((tokens + round - 1) / round));
}
static int count_stride_of(int experts) { return (experts + 3) / 4 * 4; }

hipattn_status route_experts_workspace_size(const hipops_route_desc* d, size_t* bytes) {
    if (!bytes) return fail(HIPATTN_INVALID_ARGUMENT, "route_experts_workspace_size: null output");
    *bytes = 0;
    if (const hipattn_status st = checked(d)) return st;
    const int64_t run = run_of(d->tokens), runs = (d->tokens + run - 1) / run;
    if (runs > 1) *bytes = (size_t)(runs * count_stride_of(d->experts));
    return HIPATTN_OK;
}

hipattn_status route_experts(const hipops_route_desc* d, const void* logits, const float* bias, int32_t* indices, float* weights, int32_t* begins, int32_t* order,
                             int32_t* slots, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (const hipattn_status st = checked(d)) return st;
    const bool lists = begins || order || slots;
    if (lists && (!begins || (d->tokens > 0 && (!order || !slots)))) return fail(HIPATTN_INVALID_ARGUMENT, "route_experts: begins, order and slots come together");
    if (d->tokens > 0 && (!logits || !indices || !weights)) return fail(HIPATTN_INVALID_ARGUMENT, "route_experts: null pointer");
    if (lists && d->tokens > kMostListTokens) return fail(HIPATTN_UNSUPPORTED, "route_experts: lists of %lld tokens, more than 2^26", (long long)d->tokens);
    if (d->tokens == 0 && !lists) return HIPATTN_OK;
    RouteParams p{logits, bias, indices, weights, begins, order, slots, nullptr, d->tokens, d->logits_row_stride ? d->logits_row_stride : d->experts, run_of(d->tokens),
                  count_stride_of(d->experts), d->logits_dtype, d->score, d->renormalise, d->experts, d->top_k, std::max(d->groups, 1), d->kept_groups, d->group_top, d->scale};
    const int64_t runs = std::max<int64_t>(1, (d->tokens + p.run - 1) / p.run);
    if (lists && runs > 1) {
        size_t need = 0;
        if (const hipattn_status st = route_experts_workspace_size(d, &need)) return st;
        if (!workspace || workspace_bytes < need) return fail(HIPATTN_WORKSPACE_TOO_SMALL, "route_experts: %zu bytes of workspace, %zu needed", workspace_bytes, need);
        if ((uintptr_t)workspace % 16) return fail(HIPATTN_INVALID_ARGUMENT, "route_experts: workspace must be 16-byte aligned");
        p.counts = (uint8_t*)workspace;
    }
    // (a launch of 2^32 threads or more would run modulo 2^32 of them, without an error: so many tokens, which get no lists, go in several)
    const unsigned lanes = 64 * std::min(p.run, kRouteWaves);
    const int64_t most = std::min<int64_t>(runs, 0xffffffffu / lanes);
    for (int64_t first = 0; first < runs; first += most) {
        const int64_t token = first * p.run, here = std::min(runs - first, most);
        RouteParams q = p;
        q.logits = (const uint8_t*)logits + token * p.row_stride * (d->logits_dtype == HIPATTN_F32 ? 4 : 2);
        q.indices += token * d->top_k, q.weights += token * d->top_k, q.tokens = std::min(d->tokens - token, here * p.run);
        const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)here), dim3(lanes), 0, stream, q); };
        if (d->experts <= 64)
            launch(route_kernel<1>);
        else if (d->experts <= 128)
            launch(route_kernel<2>);
        else if (d->experts <= 256)
            launch(route_kernel<4>);
        else if (d->experts <= 512)
            launch(route_kernel<8>);
        else
            launch(route_kernel<16>);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return fail(HIPATTN_HIP_ERROR, "route_experts: %s", hipGetErrorString(e));
    }
    if (lists && runs > 1) hipLaunchKernelGGL(expert_lists_kernel, dim3((unsigned)runs), dim3(kListThreads), 0, stream, p);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return fail(HIPATTN_HIP_ERROR, "route_experts: %s", hipGetErrorString(e));
    return HIPATTN_OK;
}

hipattn_status combine_experts(const hipops_combine_desc* d, const void* y, const float* weights, const int32_t* slots, const void* residual, void* out,
                               hipStream_t stream) {
    if (!d) return fail(HIPATTN_INVALID_ARGUMENT, "combine_experts: null descriptor");
    if (!float_dtype(d->y_dtype) || !float_dtype(d->out_dtype)) return fail(HIPATTN_UNSUPPORTED, "combine_experts: types must be f32, f16 or bf16");
    if (d->top_k < 1 || d->tokens < 0 || d->rows < 0 || d->n < 0)
        return fail(HIPATTN_INVALID_ARGUMENT, "combine_experts: %lld tokens of %d rows, %lld x %lld", (long long)d->tokens, d->top_k, (long long)d->rows, (long long)d->n);
    if (d->tokens > 0x7fffffffLL || d->n > 0x7fffffffLL) return fail(HIPATTN_UNSUPPORTED, "combine_experts: more than 2^31 - 1 tokens or columns");
    if (d->tokens == 0 || d->n == 0) return HIPATTN_OK;
    if (!weights || !slots || !out || (d->rows > 0 && !y)) return fail(HIPATTN_INVALID_ARGUMENT, "combine_experts: null pointer");
    CombineParams p{y, weights, slots, residual, out, 0, d->rows, d->n, d->top_k, d->y_dtype, d->out_dtype};
    const int64_t units = d->n / 8 + d->n % 8, most = std::max<int64_t>(1, 0xffffff00LL / units - 1), size = d->out_dtype == HIPATTN_F32 ? 4 : 2;
    for (int64_t first = 0; first < d->tokens; first += most) {  // (fewer than 2^32 threads to a launch)
        p.tokens = std::min(d->tokens - first, most);
        const dim3 grid((unsigned)((p.tokens * units + 255) / 256));
        const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, p); };
        if (p.y_dtype == HIPATTN_F32)
            d->n % 8 ? launch(combine_kernel<4, true>) : launch(combine_kernel<4, false>);
        else
            d->n % 8 ? launch(combine_kernel<2, true>) : launch(combine_kernel<2, false>);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return fail(HIPATTN_HIP_ERROR, "combine_experts: %s", hipGetErrorString(e));
        p.weights += most * d->top_k, p.slots += most * d->top_k, p.out = (uint8_t*)p.out + size * most * d->n;
        if (p.residual) p.residual = (const uint8_t*)p.residual + size * most * d->n;
    }
    return HIPATTN_OK;
}

}  // namespace hipops
