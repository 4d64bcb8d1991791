// New keys and values into a paged cache with the rotary position embedding applied on the way, and the
// queries rotated beside them: what stands between a decoder layer's q / k / v projection and its attention, in
// one launch.  HBM-bound byte moving: every row is read once and written once; a table row is read once per
// wavefront and token and kept in registers over the token's heads.
//
//   rotate-half:  y[i] = x[i] cos[i] - x[i + h] sin[i],  y[i + h] = x[i + h] cos[i + h] + x[i] sin[i + h],  h = rotary / 2
//   interleaved:  the same on the pairs (2i, 2i + 1) with cos[i], sin[i]
// fp32, no product fused with the sum: the stored codes are then defined to the bit.
//
// Two kinds of work, chosen by wavefront number:
//  * rows: the heads of one token (queries; with 16-bit, fp32 and u8 caches also its key and value heads);
//  * blocks (i8 caches): the new rows of one cache block for one kv head of K or V.  The block's scale follows from
//    all rows that the call puts there, so the wavefront that owns the block-head reads them, finds the largest magnitude,
//    and only then stores codes; where the scale grew it also scales the codes that were there.  No atomics, no
//    second launch: a block belongs to one sequence, and one wavefront owns each (block, kv head, K or V).
//
// A work item of 16 elements is what a lane holds: eight at d and eight at d + h (rotate-half), or sixteen side by side
// (interleaved, and the part that is not rotated), so that both partners of a pair are in one lane and memory is
// accessed sixteen bytes at a time.  No counterpart in the reference.
#include "kv_cache_write.hpp"

namespace hipattn {

namespace {

constexpr int kWavesPerGroup = 4;

// Slots of the block items: sequence s owns those from slot_base(s) on, which is enough for its new tokens n wherever in a
// block they begin: floor((b + n) / size) - floor(b / size) + 2 >= floor((n - 1) / size) + 2.
__host__ __device__ __forceinline__ int64_t slot_base(int64_t begin, int s, int block_size) { return begin / block_size + 2 * (int64_t)s; }

__device__ __forceinline__ float scale_of_peak(float peak) {
    const float s = peak / 127.0f;
    return s < 1e-30f ? 0.0f : s;
}
__device__ __forceinline__ int code_of(float x, float inverse) { return (int)fminf(fmaxf(rintf(x * inverse), -127.0f), 127.0f); }
__device__ __forceinline__ uint32_t pack_codes(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | ((uint32_t)(b & 255) << 8) | ((uint32_t)(c & 255) << 16) | ((uint32_t)d << 24);
}

__device__ __forceinline__ void rotate_pair(float& a, float& b, float ca, float sa, float cb, float sb) {
#pragma clang fp contract(off)
    const float x = a, y = b;
    a = x * ca - y * sa;
    b = y * cb + x * sb;
}

// row of the table for a token, -1: not rotated
__device__ __forceinline__ int64_t table_row(const RopeAppendParams& p, int t, int position) {
    const int row = p.positions ? p.positions[t] : position;
    return row >= 0 && row < p.table_rows ? row : -1;
}

struct Slot {
    int sequence;  // -1: a token outside every sequence
    int position;
    int block;     // -1: nowhere to store it
};
__device__ __forceinline__ Slot slot_of_token(const RopeAppendParams& p, int t, int lane) {
    Slot r{-1, -1, -1};
    if (t < p.subsequence_begins[0] || t >= p.subsequence_begins[p.num_seqs]) return r;
    r.sequence = locate_sequence(p.subsequence_begins, p.num_seqs, t, lane);
    r.position = p.past_lens[r.sequence] + (t - p.subsequence_begins[r.sequence]);
    if (r.position < 0) return r;
    const int tb = p.block_indices_begins[r.sequence], entry = r.position / p.block_size;
    if (entry >= p.block_indices_begins[r.sequence + 1] - tb) return r;
    const int block = p.block_indices[tb + entry];
    if (block >= 0 && block < p.num_blocks) r.block = block;
    return r;
}

// ---- scalar form: any types, sizes and strides --------------------------------------------------------------
// Element d of a head with its partner's: the pairs of the rotated part come first, then single elements.
__device__ __forceinline__ void load_pair(const RopeAppendParams& p, const void* src, int64_t at, int dtype, int i, int64_t row, float& a, float& b,
                                          int& da, int& db) {
    const int h = p.rotary / 2;
    if (i < h) {
        da = p.interleaved ? 2 * i : i;
        db = p.interleaved ? 2 * i + 1 : i + h;
        a = load_scalar(src, at + da, dtype);
        b = load_scalar(src, at + db, dtype);
        if (row >= 0) {
            const int64_t ta = row * p.table_row_stride + i, tb = ta + (p.interleaved ? 0 : h);
            rotate_pair(a, b, load_scalar(p.cos, ta, p.table_dtype), load_scalar(p.sin, ta, p.table_dtype), load_scalar(p.cos, tb, p.table_dtype),
                        load_scalar(p.sin, tb, p.table_dtype));
        }
    } else {
        da = db = i + h;
        a = b = load_scalar(src, at + da, dtype);
    }
}

// One row by one wavefront, into an array or a cache row that is not i8.
constexpr int kMaxPairs = 8;  // head sizes up to 512, rotated or not
__device__ __forceinline__ void move_row(const RopeAppendParams& p, const void* src, int64_t at, int src_dtype, bool rotated, int64_t row, void* dst,
                                         int64_t to, int dst_dtype, int lane) {
    RopeAppendParams r = p;
    if (!rotated) r.rotary = 0;
    const int items = p.head_dim - r.rotary / 2;
    if (dst_dtype != HIPATTN_U8) {
        for (int i = lane; i < items; i += 64) {
            float a, b;
            int da, db;
            load_pair(r, src, at, src_dtype, i, row, a, b, da, db);
            store_scalar(dst, to + da, dst_dtype, a);
            if (db != da) store_scalar(dst, to + db, dst_dtype, b);
        }
        return;
    }
    float a[kMaxPairs], b[kMaxPairs];
    int da[kMaxPairs], db[kMaxPairs];
    float mn = 3.402823466e+38f, mx = -3.402823466e+38f;
#pragma unroll
    for (int u = 0; u < kMaxPairs; u++) {
        const int i = lane + 64 * u;
        if (i >= items) break;
        load_pair(r, src, at, src_dtype, i, row, a[u], b[u], da[u], db[u]);
        mn = fminf(mn, fminf(a[u], b[u]));
        mx = fmaxf(mx, fmaxf(a[u], b[u]));
    }
    mn = wave_min(mn);
    mx = wave_max(mx);
    float scale = (mx - mn) / 255.0f;
    if (scale == 0.0f) scale = 0.0001f;
    const float zp = -mn / scale + 0.0f;  // -0 becomes +0
    const float inv = 1.0f / scale;
    uint8_t* const bytes = (uint8_t*)dst + to;
    if (lane == 0) {
        ((float*)bytes)[0] = scale;
        ((float*)bytes)[1] = zp;
    }
    const auto quantised = [&](float x) { return (uint8_t)fminf(fmaxf(rintf(fmaf(x, inv, zp)), 0.0f), 255.0f); };
#pragma unroll
    for (int u = 0; u < kMaxPairs; u++) {
        if (lane + 64 * u >= items) break;
        bytes[8 + da[u]] = quantised(a[u]);
        if (db[u] != da[u]) bytes[8 + db[u]] = quantised(b[u]);
    }
}

// Head `head` of a token: queries first, then (caches that are not i8) keys and values.
__device__ __forceinline__ void row_scalar(const RopeAppendParams& p, int t, int head, const Slot& slot, int64_t row, int lane) {
    const int Hq = p.q ? p.num_heads_q : 0, Hkv = p.num_heads_kv;
    if (head < Hq) {
        move_row(p, p.q, t * p.q_token + head * p.q_head, p.q_dtype, true, row, p.q_out, t * p.out_token + head * p.out_head, p.q_dtype, lane);
        return;
    }
    if (slot.block < 0) return;
    const bool value = head - Hq >= Hkv;
    const int h = head - Hq - (value ? Hkv : 0);
    const int64_t cache_row = ((int64_t)slot.block * Hkv + h) * p.block_size + slot.position % p.block_size;
    const bool bytes = p.cache_dtype == HIPATTN_U8;
    move_row(p, value ? p.v_new : p.k_new, value ? t * p.v_token + h * p.v_head : t * p.k_token + h * p.k_head, p.kv_dtype, !value, row,
             value ? p.value_cache : p.key_cache, cache_row * (bytes ? p.head_dim + 8 : p.head_dim), p.cache_dtype, lane);
}

// Rows [r0, r1) of one i8 block-head, the tokens from t0 on.
__device__ __forceinline__ void block_scalar(const RopeAppendParams& p, bool value, int h, int block, int t0, int position0, int r0, int r1, int lane) {
    RopeAppendParams r = p;
    if (value) r.rotary = 0;
    const void* const src = value ? p.v_new : p.k_new;
    const int64_t token = value ? p.v_token : p.k_token, head = value ? p.v_head : p.k_head;
    const int items = p.head_dim - r.rotary / 2;
    const int64_t head_index = (int64_t)block * p.num_heads_kv + h;
    int8_t* const codes = (int8_t*)(value ? p.value_cache : p.key_cache) + head_index * p.block_size * p.head_dim;
    float* const scales = (value ? p.value_scales : p.key_scales) + head_index;
    float peak = 0.0f;
    for (int n = 0; n < r1 - r0; n++) {
        const int t = t0 + n;
        const int64_t row = r.rotary ? table_row(p, t, position0 + n) : -1;
        for (int i = lane; i < items; i += 64) {
            float a, b;
            int da, db;
            load_pair(r, src, t * token + h * head, p.kv_dtype, i, row, a, b, da, db);
            peak = fmaxf(peak, fmaxf(fabsf(a), fabsf(b)));
        }
    }
    const float before = r0 == 0 ? 0.0f : *scales;
    const float scale = fmaxf(before, scale_of_peak(wave_max(peak)));
    const float inverse = scale > 0.0f ? 1.0f / scale : 0.0f;
    if (scale > before) {
        const float ratio = before / scale;
        for (int64_t i = lane; i < (int64_t)r0 * p.head_dim; i += 64) codes[i] = (int8_t)rintf((float)codes[i] * ratio);
    }
    for (int n = 0; n < r1 - r0; n++) {
        const int t = t0 + n;
        const int64_t row = r.rotary ? table_row(p, t, position0 + n) : -1;
        int8_t* const out = codes + (int64_t)(r0 + n) * p.head_dim;
        for (int i = lane; i < items; i += 64) {
            float a, b;
            int da, db;
            load_pair(r, src, t * token + h * head, p.kv_dtype, i, row, a, b, da, db);
            out[da] = (int8_t)code_of(a, inverse);
            if (db != da) out[db] = (int8_t)code_of(b, inverse);
        }
    }
    if (lane == 0) *scales = scale;
}

__global__ __launch_bounds__(64 * kWavesPerGroup) void rope_append_scalar_kernel(RopeAppendParams p, int64_t block_items, int row_heads) {
    const int lane = threadIdx.x & 63;
    int64_t w = (int64_t)blockIdx.x * kWavesPerGroup + (threadIdx.x >> 6);
    if (w >= block_items) {  // a row
        w -= block_items;
        const int t = (int)(w / row_heads), head = (int)(w % row_heads);
        if (t >= p.num_tokens) return;
        const Slot slot = slot_of_token(p, t, lane);
        const int64_t row = p.rotary && slot.sequence >= 0 ? table_row(p, t, slot.position) : -1;
        row_scalar(p, t, head, slot, row, lane);
        return;
    }
    const int per_slot = 2 * p.num_heads_kv;
    const int64_t slot = w / per_slot;
    const int which = (int)(w % per_slot);
    // the last sequence whose slots begin at or before this one
    int lo = 0, hi = p.num_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (slot_base(p.subsequence_begins[mid], mid, p.block_size) <= slot)
            lo = mid;
        else
            hi = mid;
    }
    const int begin = p.subsequence_begins[lo], end = min(p.subsequence_begins[lo + 1], p.num_tokens), past = p.past_lens[lo];
    if (begin < 0 || past < 0 || end <= begin) return;
    const int64_t n = slot - slot_base(begin, lo, p.block_size);
    const int64_t entry = past / p.block_size + n;  // of the sequence's block table
    const int64_t first = entry * p.block_size, last = (int64_t)past + (end - begin);
    const int tb = p.block_indices_begins[lo];
    if (n < 0 || first >= last || entry >= p.block_indices_begins[lo + 1] - tb) return;
    const int block = p.block_indices[tb + entry];
    if (block < 0 || block >= p.num_blocks) return;
    const int r0 = (int)max((int64_t)past - first, (int64_t)0), r1 = (int)min(last - first, (int64_t)p.block_size);
    const int position0 = (int)(first + r0);
    block_scalar(p, which >= p.num_heads_kv, which % p.num_heads_kv, block, begin + (position0 - past), position0, r0, r1, lane);
}

}  // namespace

hipError_t launch_rope_append(const RopeAppendParams& p, hipStream_t stream) {
    if (p.num_tokens == 0 || p.num_seqs == 0) return hipSuccess;
    const bool blocks = p.cache_dtype == HIPATTN_I8;
    const int64_t block_items = blocks ? (p.num_tokens / p.block_size + 2 * (int64_t)p.num_seqs) * 2 * p.num_heads_kv : 0;
    const int row_heads = (p.q ? p.num_heads_q : 0) + (blocks ? 0 : 2 * p.num_heads_kv);
    const int64_t waves = block_items + (int64_t)p.num_tokens * row_heads;
    const int64_t groups = (waves + kWavesPerGroup - 1) / kWavesPerGroup;
    if (groups > 0x7fffffff) return hipErrorInvalidValue;
    hipLaunchKernelGGL(rope_append_scalar_kernel, dim3((unsigned)groups), dim3(64 * kWavesPerGroup), 0, stream, p, block_items, row_heads);
    return hipGetLastError();
}

}  // namespace hipattn
