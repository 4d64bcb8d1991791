"""The 8-bit entry points without a GPU: what include/hipops_int8.h declares is bound and exported, descriptors have the header's layout,
and the plain implementation the GPU tests compare with does what its formulas say."""
import ctypes
import os
import re

import numpy as np

import int8_reference as R
from openvino_contrib_amd import capi, ops_capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_header_binding_and_library_agree():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "hipops_int8.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(hipops_[a-z0-9_]+)\s*\(", text)))
    assert names == sorted(ops_capi.SYMBOLS_INT8)
    L = ctypes.CDLL(ops_capi.LIB_PATH)
    for name in names:
        assert hasattr(L, name), name


def test_descriptor_layouts():
    assert ctypes.sizeof(capi.RopeAppendDesc) == 16 + 9 * 8 and capi.RopeAppendDesc.q_token_stride.offset == 24
    assert ctypes.sizeof(ops_capi.QuantizeDesc) == 24 + 3 * 8 and ops_capi.QuantizeDesc.rows.offset == 24
    assert ctypes.sizeof(ops_capi.MatmulI8Desc) == 8 + 6 * 8


def test_i8_rows_are_head_dim_bytes():
    assert capi.cache_row_bytes(capi.I8, 128) == 128


def test_reference_append_keeps_every_value_within_its_steps():
    b = R.Batch(1, [(0, 20)], 2, 1, 8, 16)
    x = (b.rng.standard_normal((20, 1, 8)) * np.geomspace(1e-3, 10, 20)[:, None, None]).astype(np.float32)
    for t in range(20):
        b.seqs, b.past, b.begins = [(t, 1)], np.array([t], np.int32), np.array([0, 1], np.int32)
        b.append(x[t:t + 1], -x[t:t + 1])
    for t in range(20):
        block, row = b.table[t // 16], t % 16
        for which, sign in ((0, 1), (1, -1)):
            held = b.codes[which, block, 0, row] * b.scales[which, block, 0].astype(np.float64)
            # half a step at every growth; scales that grow by a factor of 1.6 a token add up to 2.7 half steps
            assert np.all(np.abs(held - sign * x[t, 0]) <= b.scales[which, block, 0] * 0.5 * 6)


def test_reference_rotation_preserves_norms_and_pairs():
    rng = np.random.default_rng(2)
    angle = rng.uniform(-3, 3, (5, 8)).astype(np.float32)
    x = rng.standard_normal((5, 3, 24)).astype(np.float32)
    both = np.concatenate([angle, angle], 1)
    y = R.rotated(x, np.cos(both), np.sin(both), 16, False)
    z = R.rotated(x, np.cos(angle), np.sin(angle), 16, True)
    for r in (y, z):
        assert np.array_equal(r[..., 16:], x[..., 16:])
        assert np.allclose((r[..., :16] ** 2).sum(-1), (x[..., :16] ** 2).sum(-1), rtol=1e-5)
    order = np.argsort(np.concatenate([np.arange(0, 16, 2), np.arange(1, 16, 2)]))  # the interleaved layout is the other one permuted
    halves = np.concatenate([x[..., 0:16:2], x[..., 1:16:2], x[..., 16:]], -1)
    assert np.allclose(R.rotated(halves, np.cos(both), np.sin(both), 16, False)[..., order], z[..., :16], atol=1e-6)


def test_reference_attention_of_one_key_is_its_value():
    b = R.Batch(3, [(0, 1)], 4, 2, 16, 16)
    q = b.rng.standard_normal((1, 4, 16)).astype(np.float32)
    out = b.attention(q)
    value = b.codes[1, b.table[0], :, 0] * b.scales[1, b.table[0]][:, None].astype(np.float64)
    assert np.allclose(out[0], np.repeat(value, 2, 0))


def test_rotation_in_place_keeps_its_strides():
    L, p = capi.lib(), ctypes.c_void_p(16)
    pa = capi.PaDesc(capi.BF16, capi.BF16, capi.I8, capi.BF16, 4, 2, 64, 32, 10, 3, 1, 40, 0, 0.0, 0, 0)

    def call(q_out=p, **strides):
        d = capi.RopeAppendDesc(table_dtype=capi.F32, rotary_ndims=64, table_rows=8, table_row_stride=64)
        for name, value in strides.items():
            setattr(d, name, value)
        # (no key pointer: a call whose strides are accepted is refused for that)
        status = L.hipattn_rope_append(ctypes.byref(pa), ctypes.byref(d), p, None, None, p, p, None, q_out, p, p, p, p, p, p, p, p, None)
        assert status == capi.INVALID_ARGUMENT
        return L.hipattn_last_error_string()

    assert b"in place" in call(q_token_stride=512) and b"in place" in call(q_out_head_stride=128, q_out_token_stride=512)
    assert b"null pointer" in call() and b"null pointer" in call(q_token_stride=512, q_out_token_stride=512)
    assert b"null pointer" in call(q_token_stride=256) and b"null pointer" in call(q_out=ctypes.c_void_p(32), q_token_stride=512)
