"""Rows as 8-bit codes (hipops_quantize_rows) and products of codes (hipops_matmul_i8).

A product's integer sum is exact, so a result may differ from the fp64 value only by fp32 arithmetic (four operations, 2^-24 each, of
the terms' magnitudes) and one rounding to its type.  Plain quantisation is defined to the bit in fp32; behind a norm or a GLU the
value in front of the rounding is a few 2^-24 off (the sum of `width` squares by sqrt(width) 2^-24 at most), which moves a code by
one where it lies that close to a half, and the scale by as much."""
import ctypes

import numpy as np
import pytest

import int8_reference as R
from openvino_contrib_amd import workloads as W
from test_gpu_layer_ops import BF16, F16, F32, download, ops, upload  # noqa: F401

pytestmark = pytest.mark.gpu

HALF_ULP = {F32: 0.0, F16: 2.0 ** -11, BF16: 2.0 ** -8}


# ------------------------------------------------------------------------------ rows as codes
def quantised(hip, ops, x, x_dtype, source=0, gamma=None, g_dtype=F32, eps=1e-5, act=0, gate_first=1, stride=0, offset=0):
    rows, taken = x.shape
    width = taken // 2 if source == 2 else taken
    stored, exact = W.to_storage(x, x_dtype)
    padded = np.zeros((rows, stride or taken), stored.dtype)
    padded[:, :taken] = stored
    flat = np.concatenate([np.zeros(offset, stored.dtype), padded.reshape(-1)])
    buf = hip.DeviceBuffer.from_numpy(flat)
    view = hip.DeviceBuffer.__new__(hip.DeviceBuffer)
    view.ptr, view.nbytes, view.free = ctypes.c_void_p(buf.ptr.value + offset * stored.itemsize), 0, lambda: None
    dg, g = (None, np.float32(1)) if gamma is None else upload(hip, gamma, g_dtype)
    codes, scales = hip.DeviceBuffer(rows * width), hip.DeviceBuffer(rows * 4)
    codes.fill(0x80)
    ops.quantize_rows(ops.QuantizeDesc(source, x_dtype, g_dtype, act, gate_first, eps, rows, width, stride), view, dg, codes, scales)
    return codes.download(np.int8, (rows, width)), scales.download(np.float32, (rows,)), exact, g


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 8), (3, 37), (64, 4096), (5, 4104), (2, 8192), (2, 14336), (3, 32768), (2, 33000), (2, 32776), (700, 72),
                                        (1, 4095), (9, 512), (4, 520)])
def test_quantize_plain(hip, ops, rows, width, dtype):  # noqa: F811
    rng = np.random.default_rng(rows + width)
    x = rng.standard_normal((rows, width)).astype(np.float32) * np.float32(2.0) ** rng.integers(-8, 9, (rows, 1)).astype(np.float32)
    x[rows // 2] = 0 if rows > 1 else x[0]
    codes, scales, exact, _ = quantised(hip, ops, x, dtype)
    want = R.scale_of_peak(np.abs(exact).max(1))
    assert np.array_equal(scales, want) and np.array_equal(codes, R.codes_of(exact, want[:, None]))


def test_quantize_strides_and_alignment(hip, ops):  # noqa: F811
    rng = np.random.default_rng(2)
    for width, stride, offset in ((64, 72, 0), (64, 67, 0), (64, 64, 1), (64, 64, 8), (33, 40, 3)):
        for source in (0, 1, 2):
            x = rng.standard_normal((5, width * (2 if source == 2 else 1))).astype(np.float32)
            s = 0 if stride == width else stride * (2 if source == 2 else 1)
            codes, scales, exact, _ = quantised(hip, ops, x, F16, source, stride=s, offset=offset)
            plain, plain_scales, _, _ = quantised(hip, ops, x, F16, source)
            if source == 0:
                assert np.array_equal(codes, plain) and np.array_equal(scales, plain_scales)
            assert np.max(np.abs(codes.astype(int) - plain)) <= 1 and np.allclose(scales, plain_scales, rtol=1e-5)


def near(codes, scales, y):
    """codes and scales against the fp64 values y: the scale within the arithmetic's error, codes those of a value that close."""
    width = y.shape[1]
    rel = 2.0 ** -24 * (8 + np.sqrt(width))
    want = np.abs(y).max(1) / 127
    assert np.all(np.abs(scales - want) <= want * rel)
    exact = y / np.where(want > 0, want, 1)[:, None]
    assert np.all(np.abs(codes - exact) <= 0.5 + 127 * 4 * rel)


@pytest.mark.parametrize("dtype,g_dtype", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32), (F16, BF16)])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 4096), (64, 4096), (3, 37), (2, 8200), (2, 16384), (2, 40000), (300, 128)])
def test_quantize_norm(hip, ops, rows, width, dtype, g_dtype):  # noqa: F811
    rng = np.random.default_rng(rows * 7 + width)
    x = rng.standard_normal((rows, width)).astype(np.float32) * 3
    gamma = 1 + 0.3 * rng.standard_normal(width)
    for g in (gamma, None):
        codes, scales, exact, gv = quantised(hip, ops, x, dtype, 1, g, g_dtype)
        e = exact.astype(np.float64)
        near(codes, scales, e / np.sqrt((e ** 2).mean(1, keepdims=True) + np.float64(np.float32(1e-5))) * np.asarray(gv, np.float64))


def test_quantize_norm_of_zeros(hip, ops):  # noqa: F811
    codes, scales, _, _ = quantised(hip, ops, np.zeros((2, 64), np.float32), F16, 1, eps=0.0)
    x = np.zeros((3, 64), np.float32)
    codes, scales, _, _ = quantised(hip, ops, x, BF16, 1, np.ones(64), BF16)
    assert not codes.any() and not scales.any()


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("gate_first", [0, 1])
@pytest.mark.parametrize("rows,width", [(1, 1), (4, 14336), (33, 256), (2, 100), (3, 77)])
def test_quantize_glu(hip, ops, rows, width, gate_first, act):  # noqa: F811
    from scipy.special import erf

    rng = np.random.default_rng(rows + width + act)
    x = rng.standard_normal((rows, 2 * width)).astype(np.float32) * 2
    for dtype in (F16, BF16, F32):
        codes, scales, exact, _ = quantised(hip, ops, x, dtype, 2, act=act, gate_first=gate_first)
        e = exact.astype(np.float64)
        gate, up = (e[:, :width], e[:, width:]) if gate_first else (e[:, width:], e[:, :width])
        a = gate / (1 + np.exp(-gate)) if act == 0 else gate * 0.5 * (1 + erf(gate / np.sqrt(2))) if act == 1 else \
            gate * 0.5 * (1 + np.tanh(np.sqrt(2 / np.pi) * (gate + 0.044715 * gate ** 3)))
        y = a * up
        want = np.abs(y).max(1) / 127
        # the activations are good to about 2^-20 of the largest |gate| where their two halves cancel
        slack = 2.0 ** -20 * np.abs(gate).max() * np.abs(up).max()
        assert np.all(np.abs(scales - want) <= want * 1e-5 + slack / 127)
        step = np.where(want > 0, want, 1)[:, None]
        assert np.all(np.abs(codes - y / step) <= 0.5 + 127e-5 * 2 + slack / step)


def test_a_row_of_infinities_leaves_the_others(hip, ops):  # noqa: F811
    x = np.random.default_rng(3).standard_normal((4, 256)).astype(np.float32)
    want = quantised(hip, ops, x, F16)
    x[1, 5], x[2, 7] = np.inf, np.nan
    got = quantised(hip, ops, x, F16)
    for r in (0, 3):
        assert np.array_equal(got[0][r], want[0][r]) and got[1][r] == want[1][r]


def test_quantize_refusals(hip, ops):  # noqa: F811
    L, p = ops.lib(), ctypes.c_void_p(16)

    def call(x=p, codes=p, scales=p, **kw):
        d = ops.QuantizeDesc(0, F16, F16, 0, 1, 1e-5, 4, 64, 0)
        for name, value in kw.items():
            setattr(d, name, value)
        return L.hipops_quantize_rows(ctypes.byref(d), x, None, codes, scales, None)

    bad = [call(x=None), call(codes=None), call(scales=None), call(source=3), call(source=-1), call(width=0), call(rows=-1), call(x_row_stride=63),
           call(source=2, x_row_stride=127), call(source=2, glu_activation=3), call(source=1, eps=-1.0), call(source=1, eps=float("nan")),
           L.hipops_quantize_rows(None, p, None, p, p, None)]
    assert bad == [hip.INVALID_ARGUMENT] * len(bad)
    assert call(x_dtype=3) == hip.UNSUPPORTED and call(rows=1 << 31) == hip.UNSUPPORTED and call(rows=0) == hip.OK


# ------------------------------------------------------------------------------ products of codes
def product(hip, ops, m, n, k, c_dtype=BF16, bias=False, residual=False, scales=True, pad=(0, 0, 0), offset=0, seed=0, extreme=False, in_place=False):
    rng = np.random.default_rng(seed + 7 * m + 13 * n + k)
    lda, ldb, ldc = k + pad[0], k + pad[1], n + pad[2]
    a, b = (rng.integers(-128, 128, shape, dtype=np.int8) for shape in ((m, lda), (n, ldb)))
    if extreme:
        a[:, :k], b[:, :k] = -128, -128
    up = hip.DeviceBuffer.from_numpy

    def moved(x):
        buf = up(np.concatenate([np.zeros(offset, np.int8), x.reshape(-1), np.zeros(16, np.int8)]))
        view = hip.DeviceBuffer.__new__(hip.DeviceBuffer)
        view.ptr, view.nbytes, view.free, view.owner = ctypes.c_void_p(buf.ptr.value + offset), 0, lambda: None, buf
        return view

    da, db = moved(a), moved(b)
    sa, sb = ((rng.uniform(0.5, 1.5, x) / 1000).astype(np.float32) for x in (m, n))
    sum_ = a[:, :k].astype(np.float64) @ b[:, :k].astype(np.float64).T
    term = sum_ * sa[:, None].astype(np.float64) * sb if scales else sum_
    size, ref = np.abs(term), term
    dbias = dres = None
    if bias:
        dbias, v = upload(hip, rng.standard_normal(n), c_dtype)
        ref, size = ref + v, size + np.abs(v)
    if residual:
        dres, v = upload(hip, rng.standard_normal((m, ldc)), c_dtype)
        ref, size = ref + v[:, :n], size + np.abs(v[:, :n])
    d = ops.MatmulI8Desc(c_dtype, m, n, k, lda if pad[0] else 0, ldb if pad[1] else 0, ldc if pad[2] else 0)
    esz = hip.DTYPE_BYTES[c_dtype]
    need = ops.matmul_i8_workspace_size(d)
    results = []
    for ws in ([hip.DeviceBuffer(need)] if need else []) + [None]:
        if ws is not None:
            ws.fill(0xA5)
        c = hip.DeviceBuffer(m * ldc * esz)
        c.fill(0x7E)
        if in_place and residual:
            c.upload(W.to_storage(np.asarray(v, np.float32), c_dtype)[0])
        ops.matmul_i8(d, da, up(sa) if scales else None, db, up(sb) if scales else None, dbias, c if in_place and residual else dres, c, ws)
        raw = c.download(W.np_storage_dtype(c_dtype), (m, ldc))
        results.append(raw)
        got = W.f16_bits_to_f32(raw) if c_dtype == F16 else W.bf16_bits_to_f32(raw) if c_dtype == BF16 else raw
        if ldc > n and not (in_place and residual):
            assert np.all(raw.view(np.uint8).reshape(m, ldc, esz)[:, n:] == 0x7E), "elements between rows were written"
        err = np.abs(got[:, :n].astype(np.float64) - ref)
        bound = 4 * 2.0 ** -24 * size + HALF_ULP[c_dtype] * np.abs(ref) * 1.001 + (6e-8 if c_dtype == F16 else 0)  # (fp16's smallest step)
        assert np.all(err <= bound), "off by %.3g at %s" % (err.max(), np.unravel_index(np.argmax(err - bound), err.shape))
    assert all(np.array_equal(r, results[0]) for r in results)


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 16), (1, 4096, 4096), (2, 100, 4160), (4, 28672, 4096), (7, 1024, 14336), (15, 68, 704), (16, 512, 640),
                                   (16, 4096, 4096), (17, 6144, 320), (31, 64, 128), (32, 6144, 4096), (33, 68, 704), (48, 512, 2048), (64, 28676, 320), (64, 4096, 14336),
                                   (65, 128, 1024), (100, 5500, 192), (127, 129, 272), (128, 128, 128), (129, 4096, 4096), (255, 257, 4096), (256, 256, 64),
                                   (300, 1000, 16), (512, 6144, 4096), (1111, 4096, 1024), (2049, 300, 528), (1000, 24, 8192), (4096, 16, 256)])
def test_products(hip, ops, m, n, k):  # noqa: F811
    for c_dtype in (BF16, F16, F32):
        product(hip, ops, m, n, k, c_dtype)
    product(hip, ops, m, n, k, BF16, bias=True, residual=True)


@pytest.mark.parametrize("m,n,k", [(1, 77, 33), (5, 33, 4095), (16, 100, 31), (64, 513, 777), (130, 257, 1001), (300, 66, 17), (3, 5, 7), (520, 300, 100)])
def test_odd_sizes(hip, ops, m, n, k):  # noqa: F811
    for c_dtype in (BF16, F32):
        product(hip, ops, m, n, k, c_dtype, bias=True)


@pytest.mark.parametrize("m", [1, 16, 40, 130, 600])
def test_strides_alignment_and_missing_inputs(hip, ops, m):  # noqa: F811
    product(hip, ops, m, 320, 256, BF16, pad=(16, 32, 0))
    product(hip, ops, m, 320, 256, F16, pad=(0, 0, 8), residual=True, bias=True)
    product(hip, ops, m, 320, 256, F32, pad=(3, 5, 7), residual=True)
    product(hip, ops, m, 321, 256, F32, pad=(16, 0, 3), residual=True, bias=True)
    product(hip, ops, m, 320, 256, BF16, offset=1)
    product(hip, ops, m, 320, 256, BF16, offset=16)
    product(hip, ops, m, 320, 256, F32, scales=False)
    product(hip, ops, m, 320, 256, BF16, residual=True, in_place=True)


def test_sums_up_to_the_last_bit(hip, ops):  # noqa: F811
    """The longest k with codes of -128 throughout comes to 2^31 - 16,384; k = 0 leaves bias and residual."""
    for m in (1, 20, 300):
        product(hip, ops, m, 40, 131071, F32, extreme=True)
        product(hip, ops, m, 40, 131056, F32, extreme=True)
        c, one = hip.DeviceBuffer(m * 40 * 4), np.arange(40, dtype=np.float32)
        c.fill(0xFF)
        ops.matmul_i8(ops.MatmulI8Desc(F32, m, 40, 0, 0, 0, 0), None, None, None, None, hip.DeviceBuffer.from_numpy(one), None, c)
        assert np.array_equal(c.download(np.float32, (m, 40)), np.broadcast_to(one, (m, 40)))


def test_rows_of_scale_infinity_stay_apart(hip, ops):  # noqa: F811
    rng = np.random.default_rng(5)
    for m in (5, 40, 300):
        a, b = rng.integers(-127, 128, (m, 256), dtype=np.int8), rng.integers(-127, 128, (64, 256), dtype=np.int8)
        sa = np.ones(m, np.float32)
        sa[1], sa[3] = np.inf, np.nan
        up = hip.DeviceBuffer.from_numpy
        c = hip.DeviceBuffer(m * 64 * 4)
        ops.matmul_i8(ops.MatmulI8Desc(F32, m, 64, 256, 0, 0, 0), up(a), up(sa), up(b), None, None, None, c)
        got = c.download(np.float32, (m, 64))
        keep = [i for i in range(m) if i not in (1, 3)]
        assert np.array_equal(got[keep], (a.astype(np.int64) @ b.astype(np.int64).T)[keep].astype(np.float32))


def test_on_a_stream_of_its_own_and_captured(hip, ops):  # noqa: F811
    """A captured quantisation and product (k in parts), replayed between eager calls and other inputs."""
    rng = np.random.default_rng(6)
    m, n, k = 64, 256, 8192
    stream = hip.Stream()
    up = hip.DeviceBuffer.from_numpy
    x = [W.to_storage(rng.standard_normal((m, k)).astype(np.float32), BF16)[0] for _ in range(3)]
    dx, b = up(x[0]), up(rng.integers(-127, 128, (n, k), dtype=np.int8))
    codes, scales, c = hip.DeviceBuffer(m * k), hip.DeviceBuffer(4 * m), hip.DeviceBuffer(m * n * 4)
    d = ops.MatmulI8Desc(F32, m, n, k, 0, 0, 0)
    ws = hip.DeviceBuffer(max(16, ops.matmul_i8_workspace_size(d)))
    ws.fill(0xFF, stream)

    def step(s):
        ops.quantize_rows(ops.QuantizeDesc(0, BF16, BF16, 0, 1, 1e-5, m, k, 0), dx, None, codes, scales, s)
        ops.matmul_i8(d, codes, scales, b, None, None, None, c, ws, s)

    want = []
    for i in range(3):
        dx.upload(x[i])
        step(stream)
        want.append(c.download(np.float32, (m, n), stream))
    L = hip.lib()
    hip.check(L.hipattn_stream_begin_capture(stream.handle))
    step(stream)
    graph = ctypes.c_void_p()
    hip.check(L.hipattn_stream_end_capture(stream.handle, ctypes.byref(graph)))
    for i in (1, 2, 0, 0, 2):
        dx.upload(x[i], stream)
        c.fill(0xFF, stream)
        hip.check(L.hipattn_graph_launch(graph, stream.handle))
        assert np.array_equal(c.download(np.float32, (m, n), stream), want[i])
        step(stream)
        assert np.array_equal(c.download(np.float32, (m, n), stream), want[i])
    hip.check(L.hipattn_graph_destroy(graph))
    stream.close()


@pytest.mark.parametrize("m", [1, 15, 16, 17, 24, 31, 32, 33])
def test_products_of_few_rows(hip, ops, m):  # noqa: F811
    """Up to 32 rows: one and two tiles of activations, 16 and 32 weight rows to a workgroup (n that fills the device with either), steps that
    end inside a lane's quarter; the results of calls with and without a workspace are the same to the bit."""
    for n, k in ((5, 16), (16, 48), (17, 80), (4096, 2048), (6144, 2048), (6145, 64), (8190, 528), (12300, 1040), (128, 8192)):
        product(hip, ops, m, n, k, BF16, bias=True, residual=True, seed=n)
        product(hip, ops, m, n, k, F32, bias=True, seed=n)


@pytest.mark.parametrize("m", [1, 7, 16, 17, 32])
@pytest.mark.parametrize("offset", [0, 3])
def test_products_of_few_rows_at_any_address(hip, ops, m, offset):  # noqa: F811
    """Rows that begin anywhere and end inside a piece: k of less than a piece, of whole ones, of a few bytes more in each quarter of a step."""
    for n, k in ((3, 1), (17, 15), (16, 16), (40, 17), (33, 63), (50, 65), (320, 1001), (100, 2047), (18, 16 * 37 + 9), (4100, 130)):
        product(hip, ops, m, n, k, BF16, bias=True, residual=True, offset=offset, seed=n)
        product(hip, ops, m, n, k, F32, pad=(5, 3, 1), offset=offset, extreme=True, seed=n)


def test_product_refusals(hip, ops):  # noqa: F811
    L, p = ops.lib(), ctypes.c_void_p(16)

    def call(a=p, b=p, c=p, ws=None, nbytes=0, **kw):
        d = ops.MatmulI8Desc(BF16, 4, 64, 64, 0, 0, 0)
        for name, value in kw.items():
            setattr(d, name, value)
        return L.hipops_matmul_i8(ctypes.byref(d), a, None, b, None, None, None, c, ws, nbytes, None)

    bad = [call(a=None), call(b=None), call(c=None), call(m=-1), call(n=-1), call(k=-1), call(lda=63), call(ldb=63), call(ldc=63),
           L.hipops_matmul_i8(None, p, None, p, None, None, None, p, None, 0, None)]
    assert bad == [hip.INVALID_ARGUMENT] * len(bad)
    assert call(c_dtype=3) == hip.UNSUPPORTED and call(k=131072) == hip.UNSUPPORTED and call(m=1 << 31) == hip.UNSUPPORTED
    assert call(m=0) == hip.OK and call(n=0) == hip.OK
    n = ctypes.c_size_t(0)
    assert L.hipops_matmul_i8_workspace_size(ctypes.byref(ops.MatmulI8Desc(BF16, 4, 64, 131072, 0, 0, 0)), ctypes.byref(n)) == hip.UNSUPPORTED
    assert L.hipops_matmul_i8_workspace_size(ctypes.byref(ops.MatmulI8Desc(BF16, 4, 64, 64, 0, 0, 0)), None) == hip.INVALID_ARGUMENT


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("gamma", [False, True])
@pytest.mark.parametrize("rows,width", [(3, 64), (5, 4096), (4, 14336), (1500, 512), (4, 37), (2, 33000)])
def test_rows_of_zeros_without_an_epsilon(hip, ops, rows, width, gamma, dtype):  # noqa: F811
    """A row whose mean square and eps are both 0 has scale 0 and codes 0, in every form of the kernel; its neighbours are what they are alone."""
    x = np.random.default_rng(width).standard_normal((rows, width)).astype(np.float32)
    x[1::2] = 0
    g = np.random.default_rng(1).standard_normal(width) if gamma else None
    codes, scales, exact, gv = quantised(hip, ops, x, dtype, 1, g, dtype, eps=0.0)
    assert not codes[1::2].any() and np.array_equal(scales[1::2], np.zeros(len(scales[1::2]), np.float32))
    e = exact[::2].astype(np.float64)
    near(codes[::2], scales[::2], e / np.sqrt((e ** 2).mean(1, keepdims=True)) * np.asarray(gv, np.float64))


def test_more_rows_than_a_launch_takes(hip, ops):  # noqa: F811
    """A launch has at most 2^32 threads: 16.8 million rows of 256 of them, 67 million of 64."""
    for rows, width in (((1 << 24) + 5, 3), ((1 << 26) + 9, 8)):
        x, codes, scales = hip.DeviceBuffer(rows * width * 2), hip.DeviceBuffer(rows * width), hip.DeviceBuffer(rows * 4)
        x.fill(0x3C)
        codes.fill(0x11)
        scales.fill(0xFF)
        ops.quantize_rows(ops.QuantizeDesc(0, F16, F16, 0, 1, 1e-5, rows, width, 0), x, None, codes, scales)
        assert np.all(codes.download(np.int8, (rows * width,)) == 127)
        assert np.all(scales.download(np.float32, (rows,)) == R.scale_of_peak(np.float32(W.f16_bits_to_f32(np.array([0x3C3C], np.uint16))[0])))
        for b in (x, codes, scales):
            b.free()


def test_more_columns_than_a_launch_takes(hip, ops):  # noqa: F811
    """A launch has at most 2^32 threads, which 2^27 or 2^28 columns of few rows reach."""
    n, k, m = (1 << 28) + 40, 16, 2
    a, b, c, bias = hip.DeviceBuffer(m * k), hip.DeviceBuffer(n * k), hip.DeviceBuffer(2 * m * n), hip.DeviceBuffer(2 * n)
    scales = hip.DeviceBuffer(4 * n)
    a.fill(1)
    b.fill(2)
    bias.fill(0x3C)
    scales.fill(0x3C)
    c.fill(0xFF)
    ops.matmul_i8(ops.MatmulI8Desc(F16, m, n, k, 0, 0, 0), a, None, b, scales, bias, None, c)
    s, plus = np.full(4, 0x3C, np.uint8).view(np.float32)[0], np.float32(W.f16_bits_to_f32(np.array([0x3C3C], np.uint16))[0])
    want = W.to_storage(np.array([np.float32(32) * s + plus], np.float32), F16)[0][0]
    assert np.all(c.download(np.uint16, (m * n,)) == want)
    # and rows: 2^30 of a column each
    for x in (a, b, c, bias, scales):
        x.free()
    m = (1 << 30) + 70
    a, b, c, bias = hip.DeviceBuffer(m), hip.DeviceBuffer(1), hip.DeviceBuffer(2 * m), hip.DeviceBuffer(2)
    a.fill(1)
    b.fill(2)
    bias.fill(0x3C)
    c.fill(0xFF)
    ops.matmul_i8(ops.MatmulI8Desc(F16, m, 1, 1, 0, 0, 0), a, None, b, None, bias, None, c)
    want = W.to_storage(np.array([2 + plus], np.float32), F16)[0][0]
    assert np.all(c.download(np.uint16, (m,)) == want)
