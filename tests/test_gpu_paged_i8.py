"""Paged attention over caches of 8-bit codes with a scale per block and kv head (hipattn_paged_attention_i8) against fp64.

Bounds, before any run: the shape-generic kernels work in fp32, a context of n keys sums n products of relative error 2^-24 behind
scores of up to about 8 D^0.5 2^-24 off: 2e-5 of the largest value.  The matrix-core kernels round probabilities (and the chunk
kernel queries and values) to fp16: the bounds the framework states for its other 8-bit cache, 2e-3 for fp32 and fp16 results on
single-token rows, 1e-2 for bf16 results and chunks, relative to max(1, |ref|)."""
import ctypes

import numpy as np
import pytest

import int8_reference as R
from helpers import scaled_bound_error
from int8_reference import BF16, F16, F32, I8
from openvino_contrib_amd import workloads as W

pytestmark = pytest.mark.gpu


def run(hip, b, q_dtype=F16, out_dtype=None, window=0, flags=0, scale=0.0, sinks=None, alibi=None, new_rows=None, bound_len=None, small_workspace=False):
    out_dtype = q_dtype if out_dtype is None else out_dtype
    dev = R.Device(hip, b)
    T = b.tokens
    q_st, q = W.to_storage(b.rng.standard_normal((T, b.Hq, b.D)).astype(np.float32), q_dtype)
    up = hip.DeviceBuffer.from_numpy
    esz = hip.DTYPE_BYTES[out_dtype]
    out = hip.DeviceBuffer(T * b.Hq * b.D * esz)
    out.fill(0xFF)
    skip = hip.PA_SKIP_CACHE_WRITE if new_rows is None else 0
    keep = [up(x) if x is not None else None for x in (sinks, alibi)]
    pa = hip.PaDesc(q_dtype, F16, I8, out_dtype, b.Hq, b.Hkv, b.D, b.bs, b.blocks, T, len(b.seqs), b.longest if bound_len is None else bound_len,
                    window, scale, skip | flags, 0, keep[1].ptr if keep[1] else None, keep[0].ptr if keep[0] else None)
    if small_workspace:  # (what a bound on the contexts leaves out: room for the new prompts in fp16)
        pa.max_context_len = 64
    ws = hip.DeviceBuffer(max(16, hip.paged_attention_workspace_size(pa)))
    pa.max_context_len = b.longest if bound_len is None else bound_len
    ws.fill(0xA5)
    k, v = (up(x) for x in new_rows) if new_rows is not None else (None, None)
    hip.paged_attention_i8(pa, up(q_st), k, v, *dev.caches, *dev.scales, *dev.index, out, ws)
    got = out.download(np.float32 if out_dtype == F32 else np.uint16, (T, b.Hq, b.D))
    path = hip.last_kernel_path()
    got = got if out_dtype == F32 else (W.f16_bits_to_f32 if out_dtype == F16 else W.bf16_bits_to_f32)(got)
    return got, q, dev, path


def check(hip, b, bound, label="", window=0, scale=0.0, **kw):
    got, q, dev, path = run(hip, b, window=window, scale=scale, **kw)
    ref = b.attention(q, window, scale or None)
    inside = ~np.isnan(ref)
    err = scaled_bound_error(np.where(inside, got, 0), np.where(inside, ref, 0), "%s %s" % (label, path))
    assert err <= bound, err
    return path


def bound_of(path_fast, q_dtype, out_dtype, chunks):
    if not path_fast:
        return 2e-5 + (0 if out_dtype == F32 else 2.0 ** -11 if out_dtype == F16 else 2.0 ** -8)
    return 2e-3 if out_dtype != BF16 and not chunks else 1e-2


DECODE = [(0, 1), (15, 1), (31, 1), (32, 1), (777, 1), (2999, 1), (64, 1)]
MIXED = [(0, 70), (300, 1), (33, 129), (1500, 1), (0, 2), (63, 1), (0, 0), (500, 64)]


@pytest.mark.parametrize("D,bs", [(64, 16), (128, 32), (33, 5), (8, 1), (512, 8)])
def test_generic(hip, D, bs):
    for seqs in ([(40, 1), (0, 9), (13, 30)], [(200, 1)]):
        for out in (F32, BF16):
            b = R.Batch(1, seqs, 4, 2, D, bs)
            check(hip, b, bound_of(False, F32, out, True), q_dtype=F32, out_dtype=out, flags=hip.PA_FORCE_GENERIC)
            check(hip, b, bound_of(False, F32, out, True), q_dtype=F32, out_dtype=out, window=11, flags=hip.PA_FORCE_GENERIC)


@pytest.mark.parametrize("q_dtype", [F16, BF16])
@pytest.mark.parametrize("D", [16, 48, 64, 80, 96, 112, 128])
@pytest.mark.parametrize("bs", [16, 32, 64])
def test_decode_rows(hip, bs, D, q_dtype):
    b = R.Batch(2, DECODE, 8, 2, D, bs)
    for out in (F32, q_dtype):
        check(hip, b, bound_of(True, q_dtype, out, False), q_dtype=q_dtype, out_dtype=out)
    check(hip, b, bound_of(True, q_dtype, F32, False), q_dtype=q_dtype, out_dtype=F32, window=45)


@pytest.mark.parametrize("q_dtype", [F16, BF16])
@pytest.mark.parametrize("D,bs", [(64, 16), (64, 64), (80, 32), (128, 16), (128, 32), (128, 128), (96, 16), (16, 32)])
def test_mixed_batches(hip, D, bs, q_dtype):
    b = R.Batch(3, MIXED, 8, 2, D, bs)
    check(hip, b, bound_of(True, q_dtype, F32, True), q_dtype=q_dtype, out_dtype=F32)
    check(hip, b, bound_of(True, q_dtype, q_dtype, True), q_dtype=q_dtype, window=100)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 3), (16, 1), (32, 8), (12, 4), (32, 1), (48, 3), (17, 1), (40, 8)])
def test_heads(hip, Hq, Hkv):
    for seqs in (DECODE, MIXED, [(100, 3), (0, 20)]):
        b = R.Batch(4, seqs, Hq, Hkv, 128, 32)
        check(hip, b, bound_of(True, F16, F32, True), out_dtype=F32)


@pytest.mark.parametrize("window", [1, 2, 16, 31, 32, 33, 500, 100000])
def test_windows(hip, window):
    b = R.Batch(5, MIXED + DECODE, 8, 2, 128, 32)
    check(hip, b, bound_of(True, F16, F32, True), out_dtype=F32, window=window)


def test_rows_behind_the_context_and_unused_blocks_may_hold_anything(hip):
    for D, bs in ((128, 32), (64, 16), (128, 64), (72, 16)):
        b = R.Batch(6, MIXED, 8, 2, D, bs)
        want = R.Batch(6, MIXED, 8, 2, D, bs)
        used = set()
        for s, (past, new) in enumerate(b.seqs):
            for e in range(b.table_begins[s], b.table_begins[s + 1]):
                used.add(int(b.table[e]))
                rows = past + new - (e - b.table_begins[s]) * bs
                if rows < bs:
                    b.codes[:, b.table[e], :, rows:] = -128
        for i in set(range(b.blocks)) - used:
            b.codes[:, i], b.scales[:, i] = -128, np.nan
        got, q, _, _ = run(hip, b, out_dtype=F32)
        ref = want.attention(q)
        assert scaled_bound_error(got, ref) <= 1e-2


def test_entries_without_a_block(hip):
    for bs in (16, 32, 64):
        b = R.Batch(7, MIXED + DECODE, 8, 2, 128, bs)
        b.table[::3] = -1
        b.table[1::5] = b.blocks
        b.table[b.table_begins[1]:b.table_begins[2]] = -7  # a row with nothing to attend: zeros
        check(hip, b, bound_of(True, F16, F32, True), out_dtype=F32)
        check(hip, b, bound_of(True, F16, F32, True), out_dtype=F32, window=70)


@pytest.mark.parametrize("D,bs", [(128, 32), (64, 16), (80, 16)])
def test_scales_of_very_different_size(hip, D, bs):
    """Blocks whose values lie many orders of magnitude apart, zeros among them: a block's probabilities are weighed by its own scale."""
    b = R.Batch(8, DECODE + [(3000, 1), (100, 50)], 8, 2, D, bs)
    b.scales[1] *= np.float32(10.0) ** b.rng.integers(-4, 3, b.scales[1].shape).astype(np.float32)
    b.scales[0] *= np.float32(2.0) ** b.rng.integers(-6, 2, b.scales[0].shape).astype(np.float32)
    b.scales[:, ::5], b.codes[:, ::5] = 0, 0
    got, q, _, path = run(hip, b, out_dtype=F32)
    ref = b.attention(q)
    # every result relative to the largest value among its rows' blocks
    assert np.max(np.abs(got - ref)) <= 1e-2 * max(1.0, np.abs(ref).max())
    tiny = R.Batch(8, DECODE, 8, 2, D, bs)
    tiny.scales[1] *= np.float32(1e-7)  # a cache of small values is no less exact, relative to them
    got, q, _, path = run(hip, tiny, out_dtype=F32)
    ref = tiny.attention(q)
    assert np.max(np.abs(got - ref)) <= 2e-3 * np.abs(ref).max(), path


def test_large_scores(hip):
    """Scores of some hundreds: softmax picks single keys."""
    b = R.Batch(9, DECODE + [(50, 40)], 8, 2, 128, 32)
    check(hip, b, 2e-2, out_dtype=F32, scale=2.0)


def test_write_and_attend_in_one_call(hip):
    for D, bs in ((128, 32), (64, 16), (40, 8)):
        b = R.Batch(10, MIXED, 8, 2, D, bs)
        st, val = zip(*[W.to_storage(b.rng.standard_normal((b.tokens, 2, D)).astype(np.float32), F16) for _ in range(2)])
        got, q, dev, _ = run(hip, b, out_dtype=F32, new_rows=st)
        b.append(*val)
        codes, scales = dev.cache_state()
        assert np.array_equal(codes, b.codes) and np.array_equal(scales, b.scales)
        assert scaled_bound_error(got, b.attention(q)) <= 1e-2


def test_sinks_and_distance_bias(hip):
    b = R.Batch(11, [(40, 1), (0, 20), (333, 1)], 8, 2, 128, 32)
    sinks, slopes = b.rng.standard_normal(8).astype(np.float32), (2.0 ** -np.arange(1, 9)).astype(np.float32)
    for kw in (dict(sinks=sinks), dict(alibi=slopes), dict(sinks=sinks, alibi=slopes)):
        got, q, _, _ = run(hip, b, out_dtype=F32, **kw)
        for s, (past, new) in enumerate(b.seqs):
            blocks = b.table[b.table_begins[s]:b.table_begins[s + 1]]
            kv = (b.codes[:, blocks].astype(np.float64) * b.scales[:, blocks].astype(np.float64)[..., None, None]).transpose(0, 2, 1, 3, 4).reshape(2, 2, -1, 128)
            for i in range(new):
                t, p = b.begins[s] + i, past + i
                for h in range(8):
                    sc = kv[0, h // 4, :p + 1] @ q[t, h].astype(np.float64) / np.sqrt(128)
                    if "alibi" in kw:
                        sc += slopes[h] * (np.arange(p + 1) - p)
                    top = max(sc.max(), sinks[h] if "sinks" in kw else -np.inf)
                    w = np.exp(sc - top)
                    den = w.sum() + (np.exp(sinks[h] - top) if "sinks" in kw else 0)
                    assert np.max(np.abs(got[t, h] - w @ kv[1, h // 4, :p + 1] / den)) <= 2e-3


def test_long_context_and_many_rows(hip):
    b = R.Batch(12, [(20000, 1), (3, 1), (9000, 5)], 8, 1, 128, 32)
    check(hip, b, bound_of(True, F16, F32, True), out_dtype=F32)
    check(hip, b, bound_of(True, F16, F32, True), out_dtype=F32, bound_len=0)
    b = R.Batch(13, [(i * 7 % 90, 1) for i in range(300)], 4, 1, 128, 32)
    check(hip, b, bound_of(True, F16, F32, False), out_dtype=F32)


@pytest.mark.parametrize("bs", [16, 32, 64])
def test_new_prompts_are_expanded_once(hip, bs):
    """Prompts long enough for a copy of their rows in fp16 beside short ones, others behind cached tokens and decode rows, with and without
    room for the copy; entries without a block among the prompts', scales that are not numbers in blocks that nobody uses."""
    for seqs in ([(0, 400), (0, 383), (0, 700), (100, 450), (0, 1), (900, 1), (0, 384)], [(0, 1000)], [(0, 500), (0, 0), (3, 2)], [(1000, 390), (77, 2), (2100, 600)]):
        for edit in (False, True):
            b = R.Batch(14, seqs, 4, 2, 128, bs)
            if edit:
                b.table[2::7] = -1
                b.table[4::9] = b.blocks
            used = set(int(x) for x in b.table)
            for i in set(range(b.blocks)) - used:
                b.scales[:, i] = np.nan
            for small in (False, True):
                check(hip, b, bound_of(True, F16, F32, True), out_dtype=F32, small_workspace=small)
            check(hip, b, bound_of(True, BF16, BF16, True), q_dtype=BF16, window=333)
            check(hip, b, bound_of(True, F16, F32, True), out_dtype=F32, window=1500, bound_len=0)


@pytest.mark.parametrize("D", [8, 40, 72, 136, 192, 248, 256])
@pytest.mark.parametrize("bs", [8, 32, 64])
def test_query_tiles_at_other_head_sizes(hip, D, bs):
    b = R.Batch(15, [(0, 70), (300, 1), (33, 129), (0, 2), (500, 64)], 4, 2, D, bs)
    check(hip, b, bound_of(True, F16, F32, True), out_dtype=F32)
    check(hip, b, bound_of(True, BF16, BF16, True), q_dtype=BF16, window=90)


@pytest.mark.parametrize("factor", [1e-8, 1e-4, 1e6])
@pytest.mark.parametrize("D,seqs", [(128, [(40, 1), (700, 1), (31, 1)]), (64, [(40, 1), (700, 1)]), (64, [(0, 70), (300, 30)]), (192, [(0, 50), (100, 1)])])
def test_values_beyond_the_range_of_16_bits(hip, D, seqs, factor):
    """Codes are multiplied as they are and their scale joins in fp32, in the decode and the query-tile kernels: results are as close to fp64,
    relative to their size, as at any other magnitude (probabilities rounded to fp16: the bound of the fp16 results)."""
    b = R.Batch(16, seqs, 8, 2, D, 32)
    b.scales[1] *= np.float32(factor)
    got, q, _, path = run(hip, b, out_dtype=F32)
    ref = b.attention(q)
    assert np.max(np.abs(got - ref)) <= 2e-3 * np.abs(ref).max(), path


def test_refusals(hip):
    L, p = hip.lib(), ctypes.c_void_p(16)
    pa = hip.PaDesc(BF16, BF16, I8, BF16, 8, 2, 128, 32, 100, 4, 2, 64, 0, 0.0, 0, 0)

    def call(scales=p, q=p, new=p, ws=p, nbytes=1 << 30):
        return L.hipattn_paged_attention_i8(ctypes.byref(pa), q, new, new, p, p, scales, scales, p, p, p, p, p, ws, nbytes, None)

    assert call(scales=None) == hip.INVALID_ARGUMENT and b"scales" in L.hipattn_last_error_string()
    assert call(q=None) == hip.INVALID_ARGUMENT and call(new=None) == hip.INVALID_ARGUMENT
    n = hip.paged_attention_workspace_size(pa)
    if n:
        assert call(nbytes=n - 1) == hip.WORKSPACE_TOO_SMALL and call(ws=None) == hip.WORKSPACE_TOO_SMALL
    pa.cache_dtype = F16
    assert call() == hip.INVALID_ARGUMENT
    pa.cache_dtype = I8
    pa.num_heads_kv = 3
    assert call() == hip.INVALID_ARGUMENT
    pa.num_heads_kv = 2
    score = ctypes.c_void_p(16)
    assert L.hipattn_paged_attention_scores(ctypes.byref(pa), p, p, p, p, p, p, None, score, 10, p, 1 << 20, None) == hip.UNSUPPORTED
    assert L.hipattn_rotate_key_cache(ctypes.byref(pa), p, p, 1, p, 1, p, F32, 4, None) == hip.UNSUPPORTED


class ScaledNormal:
    """Draws of N(0, 1) times a factor, for a batch's queries."""

    def __init__(self, rng, factor):
        self.rng, self.factor = rng, factor

    def standard_normal(self, shape):
        return self.rng.standard_normal(shape) * self.factor


CHUNKS = [[(0, 70), (300, 30), (90, 1)], [(0, 450), (200, 400), (90, 1)]]  # rows converted tile by tile; expanded once, ahead of the kernel


@pytest.mark.parametrize("factor", [1.0, 1e-2, 1e-3, 1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("bs", [16, 32])
@pytest.mark.parametrize("seqs", CHUNKS)
def test_chunks_of_small_values(hip, seqs, bs, factor):
    """The chunk kernel's values are the fp16 numbers nearest to code * scale.  Off fp64, relative to the largest result: 2^-11 for the value,
    2^-11 for the probability and 2^-11 for the sum that divides it, some 2e-4 from the keys' roundings: below 2e-3; and half of fp16's
    smallest step, 2^-25, whatever the size."""
    b = R.Batch(17, seqs, 8, 2, 128, bs)
    b.scales[1] *= np.float32(factor)
    got, q, _, path = run(hip, b, out_dtype=F32)
    ref = b.attention(q)
    assert np.max(np.abs(got - ref)) <= 2e-3 * np.abs(ref).max() + 2.0 ** -25, path


@pytest.mark.parametrize("factor", [1.0, 1e-1, 1e-2, 1e-3])
@pytest.mark.parametrize("bs", [16, 32])
@pytest.mark.parametrize("seqs", CHUNKS)
def test_chunks_of_small_keys(hip, seqs, bs, factor):
    """Small keys under large queries, scores as at any other size.  A score is a sum of 128 products of keys that are each rounded to fp16 (rms
    1.7e-4 of it, also at 1e-3, where the smaller ones lie among fp16's last steps): 2.4e-4 rms in units of the exponent, 8e-4 of a weight
    at four and a half times that, twice for two keys; with the three roundings of 2^-11 below 4e-3 of the largest result."""
    b = R.Batch(18, seqs, 8, 2, 128, bs)
    b.scales[0] *= np.float32(factor)
    b.rng = ScaledNormal(b.rng, 1 / factor)
    got, q, _, path = run(hip, b, out_dtype=F32)
    ref = b.attention(q)
    assert np.max(np.abs(got - ref)) <= 4e-3 * np.abs(ref).max(), path


@pytest.mark.parametrize("scale", [1000.0, 1e20, 3e38, -1e20, -600.0, np.inf, np.nan])
@pytest.mark.parametrize("bs", [16, 32])
@pytest.mark.parametrize("D,new", [(128, 30), (128, 400), (128, 1), (64, 30)])
def test_blocks_ahead_of_the_window_may_have_any_scale(hip, D, new, bs, scale):
    """Blocks that the window has left, in the first 64 keys that a kernel looks at, with whatever codes and scales their next owner put there."""
    past, window = 330, 40
    b = R.Batch(19, [(past, new), (0, 3)], 4, 2, D, bs)
    for e in range((past - window + 1) // bs):
        block = b.table[b.table_begins[0] + e]
        b.scales[:, block] = scale
        b.codes[:, block, :, ::3], b.codes[:, block, :, 1::3], b.codes[:, block, :, 2::3] = -128, 0, 127
    got, q, _, path = run(hip, b, out_dtype=F32, window=window)
    ref = b.attention(q, window)
    assert np.isfinite(got).all(), path
    assert scaled_bound_error(got, ref, path) <= 1e-2


@pytest.mark.parametrize("seqs", CHUNKS)
def test_values_up_to_the_largest_of_16_bits(hip, seqs):
    """Chunks of values up to 65,504 are attended as any others; larger ones are cut to that in a block, and stay finite."""
    b = R.Batch(20, seqs, 8, 2, 128, 32)
    b.scales[1] = np.float32(65504 / 127)
    got, q, _, path = run(hip, b, out_dtype=F32)
    ref = b.attention(q)
    assert np.max(np.abs(got - ref)) <= 2e-3 * np.abs(ref).max(), path
    b.scales[1] *= 4
    got, q, _, path = run(hip, b, out_dtype=F32)
    assert np.isfinite(got).all(), path


@pytest.mark.parametrize("Hq,Hkv", [(32, 1), (48, 3), (24, 1)])
def test_expanded_prompts_of_shared_kv_heads(hip, Hq, Hkv):
    """More query heads to a kv head than the kernels take at once: the groups share one copy of the prompts' rows."""
    for seqs in ([(0, 400), (700, 1), (100, 450), (5, 3)], [(0, 700)]):
        b = R.Batch(21, seqs, Hq, Hkv, 128, 32)
        check(hip, b, bound_of(True, F16, F32, True), out_dtype=F32)
        check(hip, b, bound_of(True, F16, F32, True), out_dtype=F32, window=130, small_workspace=True)
