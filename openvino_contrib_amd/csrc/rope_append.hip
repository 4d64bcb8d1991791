// New keys and values into a paged cache with the rotary position embedding applied on the way, and the
// queries rotated beside them: what stands between a decoder layer's q / k / v projection and its attention, in
// one launch.  HBM-bound byte moving: every row is read once and written once; a table row is read once by each
// wavefront of a token and kept in registers over its heads (32 of 128 elements: a token of more takes several wavefronts).
//
//   rotate-half:  y[i] = x[i] cos[i] - x[i + h] sin[i],  y[i + h] = x[i + h] cos[i + h] + x[i] sin[i + h],  h = rotary / 2
//   interleaved:  the same on the pairs (2i, 2i + 1) with cos[i], sin[i]
// fp32, no product fused with the sum: the stored codes are then defined to the bit.
//
// Two kinds of work, chosen by wavefront number:
//  * rows: heads of one token (queries; with 16-bit, fp32 and u8 caches also its key and value heads);
//  * blocks (i8 caches): the new rows of one cache block for one kv head of K or V.  The block's scale follows from
//    all rows that the call puts there, so the wavefront that owns the block-head reads them, finds the largest magnitude,
//    and only then stores codes; where the scale grew it also scales the codes that were there.  No atomics, no
//    second launch: a block belongs to one sequence, and one wavefront owns each (block, kv head, K or V).
//
// A work item of 16 elements is what a lane holds: eight at d and eight at d + h (rotate-half), or sixteen side by side
// (interleaved, and the part that is not rotated), so that both partners of a pair are in one lane and memory is
// accessed sixteen bytes at a time.  No counterpart in the reference.
//
// Measured: eight chunks of 400 to 512 tokens (64 heads on 8 of 128, bf16, a packed projection, i8 cache of blocks of 32) 34.9 us (154 MB, 4.4 TB/s; a
// large copy 5.1 to 5.9), 7,300 tokens of new prompts (32 heads on 8 of 64, neighbours turned, fp16 cache of blocks of 16) 21.2 us (87 MB, 4.1 TB/s);
// the scalar form takes 197 and 168 us for them.  128 single tokens into an i8 cache 8.5 us, one 4.3: a chain of the sequence's place, its
// block, that block's scale and its rows.
#include <algorithm>

#include "kv_cache_write.hpp"

namespace hipattn {

namespace {

constexpr int kWavesPerGroup = 4;

// Slots of the block items: sequence s owns those from slot_base(s) on, which is enough for its new tokens n wherever in a
// block they begin: floor((b + n) / size) - floor(b / size) + 2 >= floor((n - 1) / size) + 2.
__host__ __device__ __forceinline__ int64_t slot_base(int64_t begin, int s, int block_size) { return begin / block_size + 2 * (int64_t)s; }

__device__ __forceinline__ float scale_of_peak(float peak) {
    const float s = peak * (1.0f / 127.0f);
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
    if (p.num_seqs == 0 || t < p.subsequence_begins[0] || t >= p.subsequence_begins[p.num_seqs]) return r;
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

// What a block item works on; false: nothing.
struct BlockItem {
    int head, block, t0, position0, r0, r1;
    bool value;
};
__device__ __forceinline__ bool find_block_item(const RopeAppendParams& p, int64_t w, int lane, BlockItem& item) {
    const int per_slot = 2 * p.num_heads_kv;
    const int64_t slot = w / per_slot;
    const int which = (int)(w % per_slot);
    // the last sequence whose slots begin at or before this one, 64 of them a step
    int lo = 0, hi = p.num_seqs;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64, at = lo + lane * step;
        const bool ok = at < hi && slot_base(p.subsequence_begins[at], at, p.block_size) <= slot;
        const int k = max(__builtin_popcountll(__builtin_amdgcn_ballot_w64(ok)) - 1, 0);
        lo = lo + k * step;
        hi = min(hi, lo + step);
    }
    const int begin = p.subsequence_begins[lo], end = min(p.subsequence_begins[lo + 1], p.num_tokens), past = p.past_lens[lo];
    const int tb = p.block_indices_begins[lo], entries = p.block_indices_begins[lo + 1] - tb;
    if (begin < 0 || past < 0 || end <= begin) return false;
    const int64_t n = slot - slot_base(begin, lo, p.block_size);
    const int64_t entry = past / p.block_size + n;  // of the sequence's block table
    const int64_t first = entry * p.block_size, last = (int64_t)past + (end - begin);
    if (n < 0 || first >= last || entry >= entries) return false;
    item.block = p.block_indices[tb + entry];
    if (item.block < 0 || item.block >= p.num_blocks) return false;
    item.r0 = (int)max((int64_t)past - first, (int64_t)0);
    item.r1 = (int)min(last - first, (int64_t)p.block_size);
    item.position0 = (int)(first + item.r0);
    item.t0 = begin + (item.position0 - past);
    item.value = which >= p.num_heads_kv;
    item.head = which - (item.value ? p.num_heads_kv : 0);
    return true;
}

__global__ __launch_bounds__(64 * kWavesPerGroup) void rope_append_scalar_kernel(RopeAppendParams p, int64_t first_group, int64_t block_items,
                                                                                  int row_heads) {
    const int lane = threadIdx.x & 63;
    int64_t w = (first_group + blockIdx.x) * kWavesPerGroup + (threadIdx.x >> 6);
    if (w >= block_items) {  // a row
        w -= block_items;
        const int t = (int)(w / row_heads), head = (int)(w % row_heads);
        if (t >= p.num_tokens) return;
        const Slot slot = slot_of_token(p, t, lane);
        const int64_t row = p.rotary && slot.sequence >= 0 ? table_row(p, t, slot.position) : -1;
        row_scalar(p, t, head, slot, row, lane);
        return;
    }
    BlockItem i;
    if (find_block_item(p, w, lane, i)) block_scalar(p, i.value, i.head, i.block, i.t0, i.position0, i.r0, i.r1, lane);
}

// ---- vector form: 16-bit q, k and v of one type, head size and rotated part multiples of 16, everything 16-byte aligned ----
// Where the sixteen elements of unit u of a head lie: eight at d0 and eight at d1.
struct Unit {
    int d0, d1;
    bool rotated;
};
__device__ __forceinline__ Unit unit_of(const RopeAppendParams& p, int u, int rotary) {
    if (p.interleaved || 16 * u >= rotary) return {16 * u, 16 * u + 8, 16 * u < rotary};
    return {8 * u, 8 * u + rotary / 2, true};
}

// A unit's factors: of its first eight elements and (rotate-half) of its second eight.
struct Turn {
    float c0[8], s0[8], c1[8], s1[8];
};
__device__ __forceinline__ void load_row8(const void* base, int64_t at, int dtype, float (&x)[8]) {
    if (dtype == HIPATTN_F32) {
        const float4_t a = *(const float4_t*)((const float*)base + at), b = *(const float4_t*)((const float*)base + at + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = a[i], x[4 + i] = b[i];
    } else {
        const uint4_t w = *(const uint4_t*)((const uint16_t*)base + at);
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = bits16_to_float((w[i >> 1] >> (16 * (i & 1))) & 0xffffu, dtype);
    }
}
__device__ __forceinline__ void load_turn(const RopeAppendParams& p, const Unit& u, int64_t row, Turn& t) {
    const int64_t at = row * p.table_row_stride + (p.interleaved ? u.d0 / 2 : u.d0);
    load_row8(p.cos, at, p.table_dtype, t.c0);
    load_row8(p.sin, at, p.table_dtype, t.s0);
    if (!p.interleaved) {
        load_row8(p.cos, at + p.rotary / 2, p.table_dtype, t.c1);
        load_row8(p.sin, at + p.rotary / 2, p.table_dtype, t.s1);
    }
}

struct Raw {
    uint4_t lo, up;
};
template <bool kBf16>
__device__ __forceinline__ void floats_of(const Raw& r, float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        x[i] = bits16_to_float((r.lo[i >> 1] >> (16 * (i & 1))) & 0xffffu, kBf16 ? HIPATTN_BF16 : HIPATTN_F16);
        x[8 + i] = bits16_to_float((r.up[i >> 1] >> (16 * (i & 1))) & 0xffffu, kBf16 ? HIPATTN_BF16 : HIPATTN_F16);
    }
}
__device__ __forceinline__ void turn_unit(const RopeAppendParams& p, const Turn& t, float (&x)[16]) {
    if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < 8; i++) rotate_pair(x[2 * i], x[2 * i + 1], t.c0[i], t.s0[i], t.c0[i], t.s0[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) rotate_pair(x[i], x[8 + i], t.c0[i], t.s0[i], t.c1[i], t.s1[i]);
    }
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    typedef float float2_t __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    if constexpr (kBf16)
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2_t){lo, hi}, bf16x2_t));
    else
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2_t){lo, hi}, half2_t));
}
template <bool kBf16>
__device__ __forceinline__ Raw bits_of(const float (&x)[16]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        r.lo[i] = pack16<kBf16>(x[2 * i], x[2 * i + 1]);
        r.up[i] = pack16<kBf16>(x[8 + 2 * i], x[9 + 2 * i]);
    }
    return r;
}
__device__ __forceinline__ uint2_t pack_bytes(const int (&q)[8]) {
    return (uint2_t){pack_codes(q[0], q[1], q[2], q[3]), pack_codes(q[4], q[5], q[6], q[7])};
}

// How a wavefront's lanes lie over rows of head_dim elements: lane l has unit l % units of row l / units.
struct Lanes {
    int units, rows, unit, row;
    bool active;
    __device__ __forceinline__ Lanes(int head_dim, int lane) : units(head_dim / 16), rows(64 / units), unit(lane % units), row(lane / units), active(row < rows) {}
};

constexpr int kAhead = 4;  // rows a lane has on their way

// Heads [first, last) of token t, no more than a round of kAhead rows a lane.
template <bool kBf16>
__device__ __forceinline__ void rows_vector(const RopeAppendParams& p, int t, int first, int last, int lane) {
    const Lanes l(p.head_dim, lane);
    const int Hq = p.q ? p.num_heads_q : 0, Hkv = p.num_heads_kv;
    const Unit turned = unit_of(p, l.unit, p.rotary), plain = unit_of(p, l.unit, 0);
    const auto source = [&](int head) -> const uint16_t* {
        if (head < Hq) return (const uint16_t*)p.q + t * p.q_token + head * p.q_head;
        if (head < Hq + Hkv) return (const uint16_t*)p.k_new + t * p.k_token + (head - Hq) * p.k_head;
        return (const uint16_t*)p.v_new + t * p.v_token + (head - Hq - Hkv) * p.v_head;
    };
    // (the rows ahead of the chain of loads that finds the token's place)
    Raw raw[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; i++) {
        const int head = first + i * l.rows + l.row;
        if (l.active && head < last) {
            const uint16_t* const src = source(head);
            const Unit u = head < Hq + Hkv ? turned : plain;
            raw[i].lo = *(const uint4_t*)(src + u.d0);
            raw[i].up = *(const uint4_t*)(src + u.d1);
        }
    }
    const Slot slot = slot_of_token(p, t, lane);
    const int64_t row = p.rotary && slot.sequence >= 0 ? table_row(p, t, slot.position) : -1;
    Turn turn;
    if (row >= 0 && turned.rotated) load_turn(p, turned, row, turn);
#pragma unroll
    for (int i = 0; i < kAhead; i++) {
        const int head = first + i * l.rows + l.row;
        // (wavefront-uniform as long as the pieces of a row reduce among themselves: every lane of a row takes the same way)
        if (!l.active || head >= last) continue;
        const bool value = head >= Hq + Hkv;
        const Unit u = value ? plain : turned;
        float x[16];
        floats_of<kBf16>(raw[i], x);
        if (!value && row >= 0 && turned.rotated) turn_unit(p, turn, x);
        if (head < Hq) {
            const Raw out = bits_of<kBf16>(x);
            uint16_t* const dst = (uint16_t*)p.q_out + t * p.out_token + head * p.out_head;
            *(uint4_t*)(dst + u.d0) = out.lo;
            *(uint4_t*)(dst + u.d1) = out.up;
            continue;
        }
        const int h = head - Hq - (value ? Hkv : 0);
        uint8_t* const cache = value ? p.value_cache : p.key_cache;
        const int64_t cache_row = ((int64_t)slot.block * Hkv + h) * p.block_size + slot.position % p.block_size;
        if (p.cache_dtype == HIPATTN_U8) {
            float mn = x[0], mx = x[0];
#pragma unroll
            for (int e = 1; e < 16; e++) mn = fminf(mn, x[e]), mx = fmaxf(mx, x[e]);
            for (int d = 1; d < l.units; d <<= 1) {
                mn = fminf(mn, __shfl_xor(mn, d, 64));
                mx = fmaxf(mx, __shfl_xor(mx, d, 64));
            }
            float scale = (mx - mn) / 255.0f;
            if (scale == 0.0f) scale = 0.0001f;
            const float zp = -mn / scale + 0.0f;  // -0 becomes +0
            const float inv = 1.0f / scale;
            int q[2][8];
#pragma unroll
            for (int e = 0; e < 16; e++) q[e >> 3][e & 7] = (int)fminf(fmaxf(rintf(fmaf(x[e], inv, zp)), 0.0f), 255.0f);
            if (slot.block < 0) continue;
            uint8_t* const dst = cache + cache_row * (p.head_dim + 8);
            if (l.unit == 0) *(float2*)dst = make_float2(scale, zp);
            *(uint2_t*)(dst + 8 + u.d0) = pack_bytes(q[0]);
            *(uint2_t*)(dst + 8 + u.d1) = pack_bytes(q[1]);
        } else if (slot.block >= 0) {
            uint16_t* const dst = (uint16_t*)cache + cache_row * p.head_dim;
            const Raw out = p.cache_dtype == HIPATTN_BF16 ? bits_of<true>(x) : bits_of<false>(x);
            *(uint4_t*)(dst + u.d0) = out.lo;
            *(uint4_t*)(dst + u.d1) = out.up;
        }
    }
}

// The new rows of one i8 block-head.  Up to kAhead rounds of rows (32 rows of 128 elements) stay in registers between the largest
// magnitude and the codes; further ones are read again.
template <bool kBf16>
__device__ __forceinline__ void block_vector(const RopeAppendParams& p, const BlockItem& b, int lane) {
    const Lanes l(p.head_dim, lane);
    const int rotary = b.value ? 0 : p.rotary;
    const Unit u = unit_of(p, l.unit, rotary);
    const uint16_t* const src = b.value ? (const uint16_t*)p.v_new + b.head * p.v_head : (const uint16_t*)p.k_new + b.head * p.k_head;
    const int64_t token = b.value ? p.v_token : p.k_token, head_index = (int64_t)b.block * p.num_heads_kv + b.head;
    int8_t* const codes = (int8_t*)(b.value ? p.value_cache : p.key_cache) + head_index * p.block_size * p.head_dim;
    float* const scales = (b.value ? p.value_scales : p.key_scales) + head_index;
    const int n = b.r1 - b.r0;
    const float stored = *scales;
    Raw raw[kAhead];
    const auto load = [&](int n0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int r = n0 + i * l.rows + l.row;
            raw[i].lo = raw[i].up = (uint4_t){0u, 0u, 0u, 0u};
            if (l.active && r < n) {
                raw[i].lo = *(const uint4_t*)(src + (b.t0 + r) * token + u.d0);
                raw[i].up = *(const uint4_t*)(src + (b.t0 + r) * token + u.d1);
            }
        }
    };
    float x[kAhead][16];
    float peak = 0.0f;
    const auto turn = [&](int n0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            if (n0 + i * l.rows >= n) break;  // (wavefront-uniform)
            const int r = n0 + i * l.rows + l.row;
            floats_of<kBf16>(raw[i], x[i]);
            if (u.rotated && l.active && r < n) {
                const int64_t row = table_row(p, b.t0 + r, b.position0 + r);
                if (row >= 0) {
                    Turn t;
                    load_turn(p, u, row, t);
                    turn_unit(p, t, x[i]);
                }
            }
        }
    };
    const int round = kAhead * l.rows;
    for (int n0 = 0; n0 < n; n0 += round) {
        load(n0);
        turn(n0);
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            if (n0 + i * l.rows >= n) break;
#pragma unroll
            for (int e = 0; e < 16; e++) peak = fmaxf(peak, fabsf(x[i][e]));
        }
    }
    const float before = b.r0 == 0 ? 0.0f : stored;
    const float scale = fmaxf(before, scale_of_peak(wave_max(peak)));
    const float inverse = scale > 0.0f ? 1.0f / scale : 0.0f;
    if (scale > before && b.r0 > 0) {
        const float ratio = before / scale;
        for (int64_t i = lane; i < (int64_t)b.r0 * p.head_dim / 16; i += 64) {
            uint4_t w = *(const uint4_t*)(codes + 16 * i);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                int q[4];
#pragma unroll
                for (int k = 0; k < 4; k++) q[k] = (int)rintf((float)(int8_t)(w[e] >> (8 * k)) * ratio);
                w[e] = pack_codes(q[0], q[1], q[2], q[3]);
            }
            *(uint4_t*)(codes + 16 * i) = w;
        }
    }
    const bool held = n <= round;
    for (int n0 = 0; n0 < n; n0 += round) {
        if (!held) {
            load(n0);
            turn(n0);
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int r = n0 + i * l.rows + l.row;
            if (!l.active || r >= n) continue;
            const float* const v = x[i];
            int8_t* const dst = codes + (int64_t)(b.r0 + r) * p.head_dim;
            *(uint2_t*)(dst + u.d0) = (uint2_t){codes4(v[0], v[1], v[2], v[3], inverse), codes4(v[4], v[5], v[6], v[7], inverse)};
            *(uint2_t*)(dst + u.d1) = (uint2_t){codes4(v[8], v[9], v[10], v[11], inverse), codes4(v[12], v[13], v[14], v[15], inverse)};
        }
    }
    if (lane == 0) *scales = scale;
}

// Wavefronts [0, block_items): blocks; behind them `shares` for each token, heads_per_wave heads each.
template <bool kBf16>
__global__ __launch_bounds__(64 * kWavesPerGroup) void rope_append_kernel(RopeAppendParams p, int64_t first_group, int64_t block_items, int row_heads,
                                                                           int heads_per_wave, int shares) {
    const int lane = threadIdx.x & 63;
    const int64_t w = (first_group + blockIdx.x) * kWavesPerGroup + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (w < block_items) {
        BlockItem item;
        if (find_block_item(p, w, lane, item)) block_vector<kBf16>(p, item, lane);
        return;
    }
    const int64_t t = (w - block_items) / shares;
    if (t >= p.num_tokens) return;
    const int first = (int)((w - block_items) % shares) * heads_per_wave;
    rows_vector<kBf16>(p, (int)t, first, min(first + heads_per_wave, row_heads), lane);
}

bool takes_vector(const RopeAppendParams& p) {
    const auto all = [](auto... x) { return ((uintptr_t)0 | ... | (uintptr_t)x); };
    if (p.kv_dtype != HIPATTN_F16 && p.kv_dtype != HIPATTN_BF16) return false;
    if ((p.q && p.q_dtype != p.kv_dtype) || p.cache_dtype == HIPATTN_F32 || p.head_dim % 16 != 0 || p.rotary % 16 != 0) return false;
    const int units = p.head_dim / 16;
    if (p.cache_dtype == HIPATTN_U8 && (units & (units - 1)) != 0) return false;  // (minimum and maximum over a row's lanes, by halves)
    if (all(p.k_new, p.v_new, p.key_cache, p.value_cache, p.q, p.q_out, p.cos, p.sin) & 15) return false;
    if (all(p.k_token, p.v_token, p.k_head, p.v_head, p.q_token, p.q_head, p.out_token, p.out_head) & 7) return false;
    return p.rotary == 0 || p.table_row_stride % (p.table_dtype == HIPATTN_F32 ? 4 : 8) == 0;
}

}  // namespace

hipError_t launch_rope_append(const RopeAppendParams& p, hipStream_t stream) {
    if (p.num_tokens == 0) return hipSuccess;
    // (without sequences nothing is stored and no index array looked at: queries alone)
    const bool stores = p.num_seqs > 0, blocks = p.cache_dtype == HIPATTN_I8;
    const int64_t block_items = stores && blocks ? (p.num_tokens / p.block_size + 2 * (int64_t)p.num_seqs) * 2 * p.num_heads_kv : 0;
    const int row_heads = (p.q ? p.num_heads_q : 0) + (stores && !blocks ? 2 * p.num_heads_kv : 0);
    // (a launch of 2^32 threads or more would run modulo 2^32 of them, without an error)
    const auto launch = [&](auto kernel, int64_t waves, auto... last) -> hipError_t {
        constexpr int kLanes = 64 * kWavesPerGroup;
        const int64_t groups = (waves + kWavesPerGroup - 1) / kWavesPerGroup, most = 0xffffffffLL / kLanes;
        for (int64_t first = 0; first < groups; first += most) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(groups - first, most)), dim3(kLanes), 0, stream, p, first, block_items, row_heads, last...);
            if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        }
        return hipSuccess;
    };
    if (takes_vector(p)) {
        // a round of rows is what a wavefront has on its way at once
        const int round = kAhead * (64 / (p.head_dim / 16));
        const int shares = std::max((row_heads + round - 1) / round, 1);
        const int64_t waves = block_items + (row_heads > 0 ? (int64_t)p.num_tokens * shares : 0);
        return launch(p.kv_dtype == HIPATTN_BF16 ? rope_append_kernel<true> : rope_append_kernel<false>, waves, round, shares);
    }
    return launch(rope_append_scalar_kernel, block_items + (int64_t)p.num_tokens * row_heads);
}

}  // namespace hipattn
