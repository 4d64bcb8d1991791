"""Appending and attending over i8 caches as a server does: recorded once and replayed on changing inputs, and in a pool whose offsets
pass 32 bits.  The plain forms and bounds are those of test_gpu_paged_i8.py; the stored codes and scales have to be equal."""
import ctypes

import numpy as np
import pytest

import int8_reference as R
from helpers import scaled_bound_error
from int8_reference import F16, F32, I8
from openvino_contrib_amd import workloads as W

pytestmark = pytest.mark.gpu


def inputs(b):
    stored, value = zip(*[W.to_storage(b.rng.standard_normal((b.tokens, h, b.D)).astype(np.float32), F16) for h in (b.Hq, b.Hkv, b.Hkv)])
    return stored, value


class Step:
    def __init__(self, hip, b, blocks, caches, scales, index, rows, cos, sin):
        self.hip, self.b, self.caches, self.scales, self.index = hip, b, caches, scales, index
        new = hip.DeviceBuffer
        self.x = [new(2 * b.tokens * h * b.D) for h in (b.Hq, b.Hkv, b.Hkv)]
        self.q, self.out = new(2 * b.tokens * b.Hq * b.D), new(4 * b.tokens * b.Hq * b.D)
        self.tables = [hip.DeviceBuffer.from_numpy(t) if t is not None else None for t in (cos, sin)]
        self.pa = hip.PaDesc(F16, F16, I8, F32, b.Hq, b.Hkv, b.D, b.bs, blocks, b.tokens, len(b.seqs), b.longest, 0, 0.0, hip.PA_SKIP_CACHE_WRITE, 0)
        self.rope = hip.RopeAppendDesc(table_dtype=F32, rotary_ndims=b.D, table_rows=rows, table_row_stride=b.D)
        self.ws = new(max(16, hip.paged_attention_workspace_size(self.pa)))
        self.ws.fill(0xA5)

    def run(self, stream=None):
        self.hip.rope_append(self.pa, self.rope, *self.x, *self.tables, None, self.q, *self.caches, *self.scales, *self.index, stream=stream)
        self.hip.paged_attention_i8(self.pa, self.q, None, None, *self.caches, *self.scales, *self.index, self.out, self.ws, stream)

    def result(self, stream=None):
        return self.out.download(np.float32, (self.b.tokens, self.b.Hq, self.b.D), stream)


def expect(b, value, cos, sin):
    place = np.concatenate([past + np.arange(new) for past, new in b.seqs])
    q, k = (R.rotated(x, cos[place], sin[place], b.D, False) for x in value[:2])
    b.append(k, value[2])
    return b.attention(W.f16_bits_to_f32(W.to_storage(q, F16)[0]))


@pytest.mark.parametrize("seqs", [[(1, 1), (1000, 1), (31, 1), (0, 1)], [(0, 400), (700, 40), (63, 1), (0, 3)]])
def test_recorded_once_replayed_on_other_inputs(hip, seqs):
    b = R.Batch(21, seqs, 8, 2, 128, 32)
    (cos, sin), (cos_v, sin_v) = R.table_rows(b.rng, b.longest, b.D, False, F32)
    dev = R.Device(hip, b)
    step = Step(hip, b, b.blocks, dev.caches, dev.scales, dev.index, b.longest, cos, sin)
    stream = hip.Stream()
    for buf in step.x:
        buf.fill(0, stream)
    step.run(stream)  # (the eager step ahead of the recording; its cache is set back below)
    stream.synchronize()
    L, graph = hip.lib(), ctypes.c_void_p()
    hip.check(L.hipattn_stream_begin_capture(stream.handle))
    step.run(stream)
    hip.check(L.hipattn_stream_end_capture(stream.handle, ctypes.byref(graph)))
    codes, scales = b.codes.copy(), b.scales.copy()
    for replay in range(5):
        b.codes, b.scales = codes.copy(), scales.copy()
        for i in range(2):
            dev.caches[i].upload(codes[i], stream)
            dev.scales[i].upload(scales[i], stream)
        stored, value = inputs(b)
        for buf, x in zip(step.x, stored):
            buf.upload(x, stream)
        step.out.fill(0xFF, stream)
        hip.check(L.hipattn_graph_launch(graph, stream.handle))
        got = step.result(stream)
        assert scaled_bound_error(got, expect(b, value, cos_v, sin_v), "replay %d" % replay) <= 1e-2
        held, held_scales = dev.cache_state()
        assert np.array_equal(held, b.codes) and np.array_equal(held_scales, b.scales)
        step.run(stream)  # (what the cache holds stays; the eager result is the recorded one)
        assert np.array_equal(step.result(stream), got)
    hip.check(L.hipattn_graph_destroy(graph))
    stream.close()


class Part:
    """A span of a device buffer."""

    def __init__(self, buf, offset, nbytes):
        self.ptr, self.nbytes = ctypes.c_void_p(buf.ptr.value + offset), nbytes


@pytest.mark.parametrize("D,bs,Hkv", [(128, 32, 8), (64, 16, 8), (80, 8, 8), (33, 5, 16)])  # stream-K and chunk, the same, query-tile, generic
def test_pools_beyond_32_bits(hip, D, bs, Hkv):
    b = R.Batch(22, [(0, 300), (90, 1), (400, 30), (5, 1)], 2 * Hkv, Hkv, D, bs)
    block_bytes = Hkv * bs * D
    first = ((1 << 32) // block_bytes) + 7  # the blocks in use lie behind the 2^32nd byte and element of each cache
    blocks = first + b.blocks
    assert first * block_bytes > 1 << 32
    (cos, sin), (cos_v, sin_v) = R.table_rows(b.rng, b.longest, D, False, F32) if D % 2 == 0 else ((None, None), (None, None))
    caches = [hip.DeviceBuffer(blocks * block_bytes) for _ in range(2)]
    scales = [hip.DeviceBuffer(blocks * Hkv * 4) for _ in range(2)]
    up = hip.DeviceBuffer.from_numpy
    index = [up(a) for a in (b.past, b.begins, b.table + np.int32(first), b.table_begins)]
    parts = [Part(c, first * block_bytes, b.blocks * block_bytes) for c in caches], [Part(s, first * Hkv * 4, b.blocks * Hkv * 4) for s in scales]
    for i in range(2):
        caches[i].fill(0x11)
        scales[i].fill(0)
        for part, x in ((parts[0][i], b.codes[i]), (parts[1][i], b.scales[i])):
            hip.check(hip.lib().hipattn_memcpy_h2d_async(part.ptr, np.ascontiguousarray(x).ctypes.data_as(ctypes.c_void_p), x.nbytes, None))
            hip.check(hip.lib().hipattn_stream_synchronize(None))
    stored, value = inputs(b)
    if D % 2:
        step = Step(hip, b, blocks, caches, scales, index, 1, None, None)
        b.append(value[1], value[2])
        want = b.attention(value[0])
    else:
        step = Step(hip, b, blocks, caches, scales, index, b.longest, cos, sin)
        want = expect(b, value, cos_v, sin_v)
    for buf, x in zip(step.x, stored):
        buf.upload(x)
    step.run()
    got = step.result()
    assert scaled_bound_error(got, want, "%s" % hip.last_kernel_path()) <= 1e-2
    for held, wanted in zip(parts[0] + parts[1], list(b.codes) + list(b.scales)):
        there = np.empty_like(wanted)
        hip.check(hip.lib().hipattn_memcpy_d2h_async(there.ctypes.data_as(ctypes.c_void_p), held.ptr, there.nbytes, None))
        hip.check(hip.lib().hipattn_stream_synchronize(None))
        assert np.array_equal(there, wanted)
