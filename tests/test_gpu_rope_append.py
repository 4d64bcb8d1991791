"""Appending rotated keys and values to a paged cache (hipattn_rope_append) against plain fp32 arithmetic in which every operation
is rounded by itself: cache bytes, codes, scales and rotated queries agree to the bit, and the values the codes stand for lie within
half a step of the fp64 rotation."""
import ctypes

import numpy as np
import pytest

import int8_reference as R
from int8_reference import BF16, F16, F32, I8, U8
from openvino_contrib_amd import workloads as W

pytestmark = pytest.mark.gpu

RAGGED = [(0, 1), (31, 1), (32, 1), (5, 70), (0, 0), (64, 32), (100, 3), (0, 33)]


def run(hip, seed, seqs, Hq, Hkv, D, bs, q_dtype, kv_dtype, cache_dtype, rotary=None, interleaved=False, table_dtype=F32, packed=True,
        head_major=False, positions=None, with_q=True, in_place=False, lead=0, table_edit=None, std=1.0, calls=1, rows=None):
    rotary = D if rotary is None else rotary
    b = R.Batch(seed, seqs, Hq, Hkv, D, bs, lead=lead, std=std)
    if table_edit:
        table_edit(b)
    rng, T = b.rng, b.tokens
    widths = (Hq, Hkv, Hkv)
    stored, value = zip(*[W.to_storage((rng.standard_normal((T, w, D)) * std).astype(np.float32), t)
                          for w, t in zip(widths, (q_dtype, kv_dtype, kv_dtype))])
    rows = rows or b.longest
    tables, (cos, sin) = R.table_rows(rng, rows, rotary, interleaved, table_dtype)
    place = np.full(T, -1)
    for s, (past, new) in enumerate(seqs):
        place[b.begins[s]:b.begins[s] + new] = past + np.arange(new)
    inside = place >= 0
    at = place if positions is None else np.where(inside, positions[:T], -1)
    turn = (at >= 0) & (at < rows)
    c, s_ = (np.where(turn[:, None], t[np.clip(at, 0, rows - 1)], np.float32(np.nan)) for t in (cos, sin))
    q = R.rotated(value[0], c, s_, rotary, interleaved)
    k, v = R.rotated(value[1], c, s_, rotary, interleaved), value[2]

    up = hip.DeviceBuffer.from_numpy
    esz = np.dtype(W.np_storage_dtype(q_dtype)).itemsize
    d = hip.RopeAppendDesc(table_dtype=table_dtype, rotary_ndims=rotary, interleaved=int(interleaved), table_rows=rows,
                           table_row_stride=cos.shape[1])
    if packed and q_dtype == kv_dtype:
        joint = up(np.concatenate([x.reshape(T, -1) for x in stored], 1))
        stride = (Hq + 2 * Hkv) * D
        views = []
        for first in (0, Hq * D, (Hq + Hkv) * D):
            view = hip.DeviceBuffer.__new__(hip.DeviceBuffer)
            view.ptr, view.nbytes = ctypes.c_void_p(joint.ptr.value + first * esz), 0
            view.free = lambda: None
            views.append(view)
        d.q_token_stride = d.k_token_stride = d.v_token_stride = stride
        dq, dk, dv = views
    elif head_major:
        dq, dk, dv = (up(x.transpose(1, 0, 2)) for x in stored)
        d.q_token_stride = d.k_token_stride = d.v_token_stride = D
        d.q_head_stride = d.k_head_stride = d.v_head_stride = T * D
    else:
        dq, dk, dv = (up(x) for x in stored)
    q_out = hip.DeviceBuffer(max(1, T * Hq * D * esz))
    q_out.fill(0xFF)
    if in_place:
        q_out, d.q_out_token_stride, d.q_out_head_stride = dq, d.q_token_stride, d.q_head_stride
    dev = R.Device(hip, b)
    row_bytes = hip.cache_row_bytes(cache_dtype, D) if cache_dtype != I8 else D
    if cache_dtype != I8:
        start = rng.integers(0, 256, (2, b.blocks, Hkv, bs, row_bytes), dtype=np.uint8)
        dev.caches = [up(x) for x in start]
    pa = hip.PaDesc(q_dtype, kv_dtype, cache_dtype, q_dtype, Hq, Hkv, D, bs, b.blocks, T, len(seqs), b.longest, 0, 0.0, 0, 0)
    dpos = up(positions[:T].astype(np.int32)) if positions is not None else None
    for _ in range(calls):
        hip.rope_append(pa, d, dq if with_q else None, dk, dv, up(tables[0]), up(tables[1]), dpos, q_out if with_q else None, *dev.caches,
                        *(dev.scales if cache_dtype == I8 else (None, None)), *dev.index)

    if with_q and not (in_place and packed):
        got = q_out.download(W.np_storage_dtype(q_dtype), (Hq, T, D) if in_place and head_major else (T, Hq, D))
        want = W.to_storage(q, q_dtype)[0]
        assert np.array_equal(got.transpose(1, 0, 2) if in_place and head_major else got, want)
    if cache_dtype == I8:
        for _ in range(calls):
            b.append(k, v)
        codes, scales = dev.cache_state()
        assert np.array_equal(scales, b.scales)
        assert np.array_equal(codes, b.codes), "%d codes differ" % (codes != b.codes).sum()
        for s, (past, new) in enumerate(seqs):  # and the values against the rotation in 64 bits: half a step, and fp32's rounding
            for i in range(new):
                where = b.slot(s, past + i)
                for which, x in enumerate((k, v)):
                    if where is not None:
                        step = scales[which, where[0]].astype(np.float64)[:, None]
                        exact = x[b.begins[s] + i].astype(np.float64)
                        # (a block of magnitudes below 127e-30 is defined to be zeros)
                        assert np.all(np.abs(codes[which, where[0], :, where[1]] * step - exact) <= np.where(step > 0, step * (0.5 + 1e-4), 127.01e-30))
    else:
        want = start
        for s, (past, new) in enumerate(seqs):
            for i in range(new):
                where = b.slot(s, past + i)
                for which, x in enumerate((k, v)):
                    if where is not None:
                        want[which, where[0], :, where[1]] = W.cache_rows_from_f32(x[b.begins[s] + i], cache_dtype)
        got = np.stack([x.download(np.uint8, start.shape[1:]) for x in dev.caches])
        assert np.array_equal(got, want), "%d bytes differ" % (got != want).sum()
    return b, dev


@pytest.mark.parametrize("cache", [F16, BF16, F32, U8, I8])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_types(hip, dtype, cache):
    run(hip, 1, RAGGED, 8, 2, 128, 32, dtype, dtype, cache)


@pytest.mark.parametrize("cache", [BF16, U8, I8])
@pytest.mark.parametrize("D,rotary,interleaved", [(64, 64, False), (64, 64, True), (80, 80, False), (80, 32, False), (128, 64, True), (96, 96, True),
                                                  (256, 256, False), (256, 128, True), (512, 512, False), (72, 72, False), (8, 8, False),
                                                  (120, 20, True), (112, 112, False), (16, 16, True), (128, 16, False)])
def test_head_sizes_and_rotations(hip, D, rotary, interleaved, cache):
    run(hip, 2, RAGGED, 6, 3, D, 16, BF16, BF16, cache, rotary=rotary, interleaved=interleaved)


@pytest.mark.parametrize("D,rotary", [(33, 32), (5, 4), (2, 2), (130, 126)])
def test_odd_head_sizes(hip, D, rotary):
    for cache in (F16, F32, I8):
        run(hip, 3, RAGGED, 4, 2, D, 8, F16, F16, cache, rotary=rotary)


@pytest.mark.parametrize("bs", [1, 2, 7, 16, 32, 64, 100, 256])
def test_block_sizes(hip, bs):
    for cache in (I8, F16):
        run(hip, 4, RAGGED + [(300, 257), (255, 2)], 4, 2, 128, bs, F16, F16, cache)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (32, 8), (64, 8), (40, 1), (7, 7), (25, 5)])
def test_heads(hip, Hq, Hkv):
    for cache in (I8, BF16):
        run(hip, 5, [(77, 1), (0, 40), (31, 2)], Hq, Hkv, 128, 32, BF16, BF16, cache)


@pytest.mark.parametrize("layout", ["packed", "apart", "head_major", "in_place", "in_place_heads", "no_q"])
def test_layouts(hip, layout):
    how = {"packed": dict(), "apart": dict(packed=False), "head_major": dict(packed=False, head_major=True), "in_place": dict(packed=False, in_place=True),
           "in_place_heads": dict(packed=False, head_major=True, in_place=True), "no_q": dict(packed=False, with_q=False)}[layout]
    for cache in (I8, F16, U8):
        for D in (128, 72):
            run(hip, 6, RAGGED, 8, 2, D, 32, F16, F16, cache, **how)


@pytest.mark.parametrize("table", [F16, BF16])
def test_tables_of_16_bits_and_mixed_types(hip, table):
    run(hip, 7, RAGGED, 8, 2, 128, 32, BF16, BF16, I8, table_dtype=table)
    run(hip, 7, RAGGED, 8, 2, 64, 32, F16, F16, F16, table_dtype=table, interleaved=True)
    run(hip, 7, RAGGED, 8, 2, 128, 32, BF16, F16, I8, table_dtype=table)  # queries of another type than keys
    run(hip, 7, RAGGED, 8, 2, 128, 32, BF16, F32, U8, table_dtype=table)


def test_positions_and_rows_outside_the_table(hip):
    given = np.random.default_rng(8).integers(-3, 60, 200)
    for cache in (I8, BF16):
        run(hip, 8, RAGGED, 8, 2, 128, 32, BF16, BF16, cache, positions=given, rows=50)
        run(hip, 8, RAGGED, 8, 2, 128, 32, BF16, BF16, cache, rows=40)  # tokens beyond the table are not turned


def test_entries_without_a_block_and_tokens_without_a_sequence(hip):
    def edit(b):
        b.table[::3] = [-1, b.blocks, 1 << 30, -5][0:1] * len(b.table[::3])
        b.table[1::7] = b.blocks
        b.table_begins[-1] -= 1  # the last sequence's table ends before its tokens do

    for cache in (I8, F16, U8):
        run(hip, 9, RAGGED, 8, 2, 128, 32, F16, F16, cache, table_edit=edit)
        run(hip, 9, RAGGED, 8, 2, 128, 32, F16, F16, cache, lead=5)


@pytest.mark.parametrize("tokens,bs", [(1, 32), (2, 32), (513, 16), (3000, 32), (2500, 64)])
def test_lengths(hip, tokens, bs):
    for cache in (I8, F16):
        run(hip, 10, [(0, tokens)], 4, 1, 64, bs, F16, F16, cache)
        run(hip, 10, [(17, tokens), (4000, 1)], 4, 1, 128, bs, BF16, BF16, cache)


def test_many_sequences(hip):
    seqs = [(i * 37 % 200, i % 4) for i in range(700)]
    for cache in (I8, F16):
        run(hip, 11, seqs, 4, 2, 64, 16, F16, F16, cache)


def test_a_repeated_call_changes_nothing(hip):
    run(hip, 12, RAGGED, 8, 2, 128, 32, BF16, BF16, I8, calls=3)


@pytest.mark.parametrize("std", [1e-36, 1e-20, 1e-4, 3e4])
def test_magnitudes(hip, std):
    run(hip, 13, RAGGED, 4, 2, 128, 32, BF16, BF16, I8, std=std)


@pytest.mark.parametrize("D,bs", [(128, 32), (72, 16), (64, 64)])
def test_scales_grow_token_by_token(hip, D, bs):
    """One token at a time with rows of very different size, zeros first: the codes that are there are scaled with their block."""
    Hq, Hkv, T = 4, 2, 2 * bs + 3
    b = R.Batch(14, [(0, T)], Hq, Hkv, D, bs)
    rng = b.rng
    size = np.float32(2.0) ** rng.integers(-6, 7, T)
    size[:3] = 0
    k, v = (W.to_storage((rng.standard_normal((T, Hkv, D)) * size[:, None, None]).astype(np.float32), F16) for _ in range(2))
    dev = R.Device(hip, b)
    desc = hip.RopeAppendDesc()
    for t in range(T):
        b.seqs, b.past, b.begins = [(t, 1)], np.array([t], np.int32), np.array([0, 1], np.int32)
        dev.index[0].upload(b.past)
        dev.index[1].upload(b.begins)
        pa = hip.PaDesc(F16, F16, I8, F16, Hq, Hkv, D, bs, b.blocks, 1, 1, T, 0, 0.0, 0, 0)
        up = hip.DeviceBuffer.from_numpy
        hip.rope_append(pa, desc, None, up(k[0][t]), up(v[0][t]), None, None, None, None, *dev.caches, *dev.scales, *dev.index)
        b.append(k[1][t:t + 1], v[1][t:t + 1])
    codes, scales = dev.cache_state()
    assert np.array_equal(scales, b.scales) and np.array_equal(codes, b.codes)
    # every growth of the scale rounds the codes once more, each by at most half a step of a scale no larger than the last
    for i, x in enumerate((k[1], v[1])):
        blocks = b.table[np.arange(T) // bs]
        held = codes[i, blocks, :, np.arange(T) % bs] * scales[i, blocks][:, :, None].astype(np.float64)
        assert np.all(np.abs(held - x) <= scales[i, blocks][:, :, None] * 0.5 * 13)


def test_infinite_new_rows_stay_in_their_block(hip):
    b = R.Batch(15, [(0, 40), (0, 40)], 4, 2, 128, 32)
    k = b.rng.standard_normal((80, 2, 128)).astype(np.float32)
    k[3] = np.inf
    k[5, 0, 7] = np.nan
    dev = R.Device(hip, b)
    pa = hip.PaDesc(F32, F32, I8, F32, 4, 2, 128, 32, b.blocks, 80, 2, 40, 0, 0.0, 0, 0)
    up = hip.DeviceBuffer.from_numpy
    hip.rope_append(pa, hip.RopeAppendDesc(), None, up(k), up(k), None, None, None, None, *dev.caches, *dev.scales, *dev.index)
    codes, scales = dev.cache_state()
    b.append(np.where(np.isfinite(k), k, 0), np.where(np.isfinite(k), k, 0))
    spoiled = b.table[0]
    others = [i for i in range(b.blocks) if i != spoiled]
    assert np.array_equal(codes[:, others], b.codes[:, others]) and np.array_equal(scales[:, others], b.scales[:, others])


def test_refusals(hip):
    L = hip.lib()
    p = ctypes.c_void_p(16)

    def call(pa, r, q=p, k=p, cos=p, sin=p, q_out=p, cache=p, scales=p, index=p):
        return L.hipattn_rope_append(ctypes.byref(pa), ctypes.byref(r) if r else None, q, k, k, cos, sin, None, q_out, cache, cache, scales,
                                     scales, index, index, index, index, None)

    def pa(**kw):
        d = hip.PaDesc(BF16, BF16, I8, BF16, 8, 2, 128, 32, 100, 4, 2, 64, 0, 0.0, 0, 0)
        for name, x in kw.items():
            setattr(d, name, x)
        return d

    def r(**kw):
        d = hip.RopeAppendDesc(table_dtype=F32, rotary_ndims=128, table_rows=64, table_row_stride=128)
        for name, x in kw.items():
            setattr(d, name, x)
        return d

    bad = [call(pa(), None), call(pa(), r(), k=None), call(pa(), r(), scales=None), call(pa(), r(), cos=None), call(pa(), r(), q=None),
           call(pa(), r(), q_out=None), call(pa(), r(), index=None), call(pa(), r(), cache=None), call(pa(), r(rotary_ndims=127)),
           call(pa(), r(rotary_ndims=130)), call(pa(), r(rotary_ndims=-2)), call(pa(), r(table_dtype=U8)), call(pa(), r(table_row_stride=64)),
           call(pa(), r(table_rows=-1)), call(pa(), r(k_token_stride=-1)), call(pa(), r(q_out_token_stride=64)), call(pa(kv_dtype=I8), r()),
           call(pa(q_dtype=U8), r()), call(pa(cache_dtype=9), r()), call(pa(num_heads_kv=3), r()), call(pa(head_dim=0), r()),
           call(pa(num_blocks=0), r())]
    assert bad == [hip.INVALID_ARGUMENT] * len(bad)
    assert call(pa(head_dim=513), r()) == hip.UNSUPPORTED
    assert call(pa(num_tokens=0), r()) == hip.OK and call(pa(num_seqs=0), r()) == hip.OK
    # the writer and the 16-bit entry point have no place for the scales
    one = p
    assert L.hipattn_kv_cache_write(ctypes.byref(pa()), one, one, one, one, one, one, one, one, None) == hip.UNSUPPORTED
    assert L.hipattn_paged_attention(ctypes.byref(pa()), one, one, one, one, one, one, one, one, one, one, one, 1 << 30, None) == hip.INVALID_ARGUMENT


@pytest.mark.parametrize("D,dtype", [(128, BF16), (72, F16), (33, F32)])
def test_a_batch_without_sequences_copies_its_queries(hip, D, dtype):
    """Every token is outside every sequence: queries are not turned, nothing is stored, and the index arrays are not looked at."""
    T, Hq = 5, 6
    q = W.to_storage(np.random.default_rng(16).standard_normal((T, Hq, D)).astype(np.float32), dtype)[0]
    up = hip.DeviceBuffer.from_numpy
    dq, out = up(q), hip.DeviceBuffer(q.nbytes)
    out.fill(0xFF)
    table = up(np.ones((8, D), np.float32))
    rope = hip.RopeAppendDesc(table_dtype=F32, rotary_ndims=D // 2 * 2, table_rows=8, table_row_stride=D)
    for cache in (I8, F16):
        pa = hip.PaDesc(dtype, dtype, cache, dtype, Hq, 2, D, 32, 4, T, 0, 8, 0, 0.0, 0, 0)
        hip.rope_append(pa, rope, dq, None, None, table, table, None, out, *[None] * 8)
        assert np.array_equal(out.download(q.dtype, q.shape), q)
        out.fill(0xFF)
    hip.rope_append(pa, rope, dq, None, None, table, table, None, dq, *[None] * 8)  # in place: as it is
    assert np.array_equal(dq.download(q.dtype, q.shape), q)
    hip.rope_append(pa, rope, None, None, None, table, table, None, None, *[None] * 8)


def test_more_rows_than_a_launch_takes(hip):
    """A launch has at most 2^32 threads, 67 million rows of a wavefront each: tokens of 62 query heads, a key and a value."""
    T, Hq, bs = (1 << 20) + 300, 62, 1024
    q, new, out = hip.DeviceBuffer(2 * T * Hq), hip.DeviceBuffer(2 * T), hip.DeviceBuffer(2 * T * Hq)
    blocks = -(-T // bs)
    caches = [hip.DeviceBuffer(2 * blocks * bs) for _ in range(2)]
    q.fill(0x3C)
    new.fill(0x2A)
    for b in (out, *caches):
        b.fill(0xFF)
    up = hip.DeviceBuffer.from_numpy
    index = [up(np.array(a, np.int32)) for a in ([0], [0, T], np.arange(blocks), [0, blocks])]
    pa = hip.PaDesc(F16, F16, F16, F16, Hq, 1, 1, bs, blocks, T, 1, T, 0, 0.0, 0, 0)
    hip.rope_append(pa, hip.RopeAppendDesc(), q, new, new, None, None, None, out, *caches, None, None, *index)
    assert np.all(out.download(np.uint16, (T * Hq,)) == 0x3C3C)
    for c in caches:
        assert np.all(c.download(np.uint16, (blocks * bs,))[:T] == 0x2A2A)
