"""Rows as e4m3 codes (hipops_quantize_fp8) and products of codes with a scale for each block of 128 (hipops_matmul_fp8).

Plain quantisation is defined to the bit in fp32.  Behind a norm or a GLU the value in front of the rounding is a few 2^-24 off (a norm: the
sum of `width` squares by sqrt(width) 2^-24), so a code is the nearest of a value that close: half a step (2^-4 of the value, 2^-10 of the
scale at the bottom of the range) and that little more.

A product adds k terms in fp32, in an order of its own: an element is off by at most (k / 128 + 130) 2^-24 of the sum of its terms' magnitudes
(128 additions in a block, one for each block, and the scales' two products), and in the 2-norm, where roundings go either way, by less than
sqrt(k + 16) 2^-24 of the terms' 2-norm; one rounding to its type comes on top.  Results of 16 bits (and codes) come from the matrix instruction
for 8-bit operands, which aligns eight neighbouring products to the largest of them and keeps 14 bits below it: each is off by at most 2^-14
of that one, hence by at most 8 x 2^-14 of the sum of the eight magnitudes, an element by 2^-11 of its terms' and, roundings going either way, less than
2^-13.5 of the terms' 2-norm (a product's error has a variance of (2^-14 L)^2 / 12 with L the largest, the squares of eight add up to L^2 or more:
sqrt(8 / 12) 2^-14)."""
import ctypes

import numpy as np
import pytest

import experts_reference as R
from openvino_contrib_amd import workloads as W
from test_gpu_layer_ops import BF16, F16, F32, ops, upload  # noqa: F401

pytestmark = pytest.mark.gpu

HALF_ULP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def values(raw, dtype):
    return W.f16_bits_to_f32(raw) if dtype == F16 else W.bf16_bits_to_f32(raw) if dtype == BF16 else raw


def moved(hip, x, offset):
    """x on the device, `offset` bytes behind an allocation's beginning, sixteen spare bytes at its end"""
    buf = hip.DeviceBuffer.from_numpy(np.concatenate([np.zeros(offset, np.uint8), np.ascontiguousarray(x).view(np.uint8).reshape(-1), np.zeros(16, np.uint8)]))
    view = hip.DeviceBuffer.__new__(hip.DeviceBuffer)
    view.ptr, view.nbytes, view.free, view.owner = ctypes.c_void_p(buf.ptr.value + offset), 0, lambda: None, buf
    return view


# ------------------------------------------------------------------------------ rows as codes
def quantised(hip, ops, x, x_dtype, source=0, gamma=None, g_dtype=F32, eps=1e-5, act=0, gate_first=1, stride=0, offset=0, by_row=False):
    rows, taken = x.shape
    width = taken // 2 if source == 2 else taken
    stored, exact = W.to_storage(x, x_dtype)
    padded = np.zeros((rows, stride or taken), stored.dtype)
    padded[:, :taken] = stored
    dx = moved(hip, padded, offset * stored.itemsize)
    dg, g = (None, np.float32(1)) if gamma is None else upload(hip, gamma, g_dtype)
    n = R.blocks(width)
    codes, scales = hip.DeviceBuffer(rows * width), hip.DeviceBuffer(rows * n * 4)
    codes.fill(0x7F)
    scales.fill(0xFF)
    ops.quantize_fp8(ops.QuantizeFp8Desc(source, x_dtype, g_dtype, act, gate_first, eps, rows, width, stride, n if by_row else 0, 1 if by_row else 0), dx, dg, codes, scales)
    s = scales.download(np.float32, (rows, n) if by_row else (n, rows))
    return codes.download(np.uint8, (rows, width)), s if by_row else s.T, exact, g


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 8), (3, 37), (64, 4096), (5, 4104), (2, 14336), (3, 33000), (700, 72), (1, 4095), (9, 512), (4, 520), (17, 128),
                                        (1030, 264), (2, 127), (2, 129)])
def test_quantise_plain(hip, ops, rows, width, dtype):  # noqa: F811
    rng = np.random.default_rng(rows + width)
    x = rng.standard_normal((rows, width)).astype(np.float32) * np.float32(2.0) ** rng.integers(-8, 9, (rows, 1)).astype(np.float32)
    x[rows // 2] = 0 if rows > 1 else x[0]
    for by_row in (False, True):
        codes, scales, exact, _ = quantised(hip, ops, x, dtype, by_row=by_row)
        want, want_scales = R.quantised(exact)
        assert np.array_equal(scales, want_scales) and np.array_equal(R.VALUES[codes], R.VALUES[want])


def test_quantise_spans_of_magnitudes(hip, ops):  # noqa: F811
    """A block from 1e-12 of its largest value up: codes down to the format's smallest numbers and zero; scales about the smallest; exact halves."""
    rng = np.random.default_rng(0)
    x = (rng.choice([-1, 1], (64, 512)) * np.geomspace(1e-12, 1, 512)).astype(np.float32) * np.geomspace(1e-37, 1e30, 64).astype(np.float32)[:, None]
    x[0, :] = 0
    steps = (R.VALUES[:126] + R.VALUES[1:127]) / 2
    x[1, :128], x[1, 128:256], x[2, :128] = 448, -448, 448
    x[1, 1:127], x[1, 129:255] = steps, -steps
    codes, scales, exact, _ = quantised(hip, ops, x, F32)
    want, want_scales = R.quantised(exact)
    assert np.array_equal(scales, want_scales) and np.array_equal(R.VALUES[codes], R.VALUES[want])


def near(codes, scales, y, slack):
    """codes of a value within slack of y, scales of the largest such"""
    width = y.shape[1]
    s = R.spread(scales.astype(np.float64), width)
    peak = np.stack([np.abs(part).max(1) for part in np.split(y, range(128, width, 128), 1)], 1)
    most = np.stack([np.broadcast_to(slack, y.shape)[:, i:i + 128].max(1) for i in range(0, width, 128)], 1)
    assert np.all(np.abs(scales - peak / 448) <= peak / 448 * 2.0 ** -22 + most / 448)
    assert np.all(np.abs(R.VALUES[codes] * s - y) <= np.maximum(np.abs(y) * 2.0 ** -4, s * 2.0 ** -10) + np.abs(y) * 2.0 ** -21 + 2 * slack)


@pytest.mark.parametrize("dtype,g_dtype", [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32), (F16, BF16)])
@pytest.mark.parametrize("rows,width", [(1, 1), (1, 4096), (64, 4096), (3, 37), (2, 8200), (2, 16384), (2, 40000), (300, 128), (1500, 1024), (1025, 136), (1, 32768), (1100, 5120)])
def test_quantise_norm(hip, ops, rows, width, dtype, g_dtype):  # noqa: F811
    rng = np.random.default_rng(rows * 7 + width)
    x = rng.standard_normal((rows, width)).astype(np.float32) * 3
    gamma = 1 + 0.3 * rng.standard_normal(width)
    for g in (gamma, None):
        codes, scales, exact, gv = quantised(hip, ops, x, dtype, 1, g, g_dtype)
        e = exact.astype(np.float64)
        y = e / np.sqrt((e ** 2).mean(1, keepdims=True) + np.float64(np.float32(1e-5))) * np.asarray(gv, np.float64)
        near(codes, scales, y, np.abs(y) * 2.0 ** -24 * (8 + np.sqrt(width)))


def test_quantise_norm_of_zeros(hip, ops):  # noqa: F811
    for rows, width in ((2, 64), (1100, 64), (2, 63)):
        x = np.zeros((rows, width), np.float32)
        for eps in (0.0, 1e-5):
            codes, scales, _, _ = quantised(hip, ops, x, BF16, 1, np.ones(width), BF16, eps=eps)
            assert not codes.any() and not scales.any()


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("gate_first", [0, 1])
@pytest.mark.parametrize("rows,width", [(1, 1), (4, 14336), (33, 256), (2, 100), (3, 77), (1030, 136)])
def test_quantise_glu(hip, ops, rows, width, gate_first, act):  # noqa: F811
    rng = np.random.default_rng(rows + width + act)
    x = rng.standard_normal((rows, 2 * width)).astype(np.float32) * 2
    for dtype in (F16, BF16, F32):
        codes, scales, exact, _ = quantised(hip, ops, x, dtype, 2, act=act, gate_first=gate_first)
        e = exact.astype(np.float64)
        # the activations are good to about 2^-20 of the largest |gate| where their two halves cancel
        near(codes, scales, R.gated(e, act, gate_first), 2.0 ** -20 * np.abs(e).max() ** 2)


def test_quantise_strides_and_alignment(hip, ops):  # noqa: F811
    rng = np.random.default_rng(2)
    for width, stride, offset in ((256, 264, 0), (256, 259, 0), (256, 256, 1), (256, 256, 8), (133, 140, 3)):
        x = rng.standard_normal((5, width)).astype(np.float32)
        codes, scales, exact, _ = quantised(hip, ops, x, F16, stride=stride if stride != width else 0, offset=offset)
        want, want_scales = R.quantised(exact)
        assert np.array_equal(scales, want_scales) and np.array_equal(R.VALUES[codes], R.VALUES[want])
        for source in (1, 2):
            x = rng.standard_normal((5, width * source)).astype(np.float32)
            s = 0 if stride == width else stride * source
            codes, scales, _, _ = quantised(hip, ops, x, F16, source, stride=s, offset=offset)
            plain, plain_scales, _, _ = quantised(hip, ops, x, F16, source)
            assert np.allclose(scales, plain_scales, rtol=1e-5)
            assert np.all(np.abs(R.VALUES[codes] - R.VALUES[plain]) <= np.maximum(np.abs(R.VALUES[plain]) / 8, 2.0 ** -9) * 1.01)


@pytest.mark.parametrize("width", [1 << 24, (1 << 24) + 129])
@pytest.mark.parametrize("source", [0, 2])
def test_quantise_the_widest_rows(hip, ops, width, source):  # noqa: F811
    """A row's workgroups fill the grid's second dimension half, and wider rows take a workgroup each: 64 blocks over and over have the same codes every time."""
    rng = np.random.default_rng(width)
    halves = [rng.standard_normal((3, 8192)).astype(np.float32) for _ in range(2 if source == 2 else 1)]
    want, want_scales, _, _ = quantised(hip, ops, np.concatenate(halves, 1), F16, source)
    wide = lambda x, n: np.tile(x, (1, -(-n // x.shape[1])))[:, :n]
    codes, scales, _, _ = quantised(hip, ops, np.concatenate([wide(h, width) for h in halves], 1), F16, source)
    whole = width // 128
    assert np.array_equal(codes[:, :whole * 128], wide(want, whole * 128)) and np.array_equal(scales[:, :whole], wide(want_scales, whole))
    if width % 128:  # (a single column in the last block)
        assert width % 128 == 1 and np.array_equal(R.VALUES[codes[:, -1]], np.sign(R.VALUES[codes[:, -1]]) * 448.0)
        assert np.array_equal(np.sign(R.VALUES[codes[:, -1]]), np.sign(R.VALUES[want[:, whole * 128 % 8192]]))


def test_a_block_of_infinities_leaves_the_others(hip, ops):  # noqa: F811
    x = np.random.default_rng(3).standard_normal((4, 512)).astype(np.float32)
    want = quantised(hip, ops, x, F16)
    x[1, 130], x[2, 511] = np.inf, np.nan
    got = quantised(hip, ops, x, F16)
    keep = np.ones((4, 4), bool)
    keep[1, 1] = keep[2, 3] = False
    assert np.array_equal(got[1][keep], want[1][keep]) and np.array_equal(got[0][R.spread(keep, 512)], want[0][R.spread(keep, 512)])


def test_more_rows_than_a_launch_has_threads(hip, ops):  # noqa: F811
    """17 million rows of three elements: the scalar form's 256 lanes a row pass 2^32 threads."""
    rows = (1 << 32) // 256 + 5000
    x = np.tile(np.array([1, -2, 4], np.float16).view(np.uint16), rows)
    dx = hip.DeviceBuffer.from_numpy(x)
    codes, scales = hip.DeviceBuffer(rows * 3), hip.DeviceBuffer(rows * 4)
    codes.fill(0)
    scales.fill(0)
    ops.quantize_fp8(ops.QuantizeFp8Desc(0, F16, F16, 0, 0, 0.0, rows, 3), dx, None, codes, scales)
    want, s = R.quantised(np.array([[1, -2, 4]], np.float32))
    assert np.all(codes.download(np.uint8, (rows, 3)) == want) and np.all(scales.download(np.float32, (rows,)) == s[0, 0])


@pytest.mark.parametrize("source", [0, 1, 2])
@pytest.mark.parametrize("by_row", [False, True])
def test_more_rows_than_a_quantising_launch_takes(hip, ops, source, by_row):  # noqa: F811
    """64 lanes a row: 2^26 rows and some go in two launches.  Eleven rows over and over, which the launches' ends do not divide by, are those rows every time."""
    rows, width = (1 << 26) + 5000, 3
    some = np.random.default_rng(source).standard_normal((11, width * (2 if source == 2 else 1))).astype(np.float32)
    want, want_scales, exact, _ = quantised(hip, ops, some, F16, source)
    if source == 0:
        ref, ref_scales = R.quantised(exact)
        assert np.array_equal(R.VALUES[want], R.VALUES[ref]) and np.array_equal(want_scales, ref_scales)
    x = hip.DeviceBuffer.from_numpy(np.tile(W.to_storage(some, F16)[0], (-(-rows // 11), 1))[:rows])
    codes, scales = hip.DeviceBuffer(rows * width), hip.DeviceBuffer(rows * 4)
    codes.fill(0x7F)
    scales.fill(0xFF)
    ops.quantize_fp8(ops.QuantizeFp8Desc(source, F16, F16, 0, 1, 1e-5, rows, width, 0, int(by_row), int(by_row)), x, None, codes, scales)
    for got, pattern in ((codes.download(np.uint8, (rows, width)), want), (scales.download(np.uint32, (rows, 1)), np.ascontiguousarray(want_scales).view(np.uint32))):
        whole = rows // 11 * 11
        assert np.all(got[:whole].reshape(-1, 11, pattern.shape[1]) == pattern) and np.all(got[whole:] == pattern[:rows - whole])


# ------------------------------------------------------------------------------ products
def bounds(k, dtype, ref, size, coarse=None):
    """The largest error of each element; coarse: summed by the instruction for 8-bit operands."""
    instruction = 2.0 ** -11 if (dtype != F32 if coarse is None else coarse) else 0.0
    return (instruction + 2.0 ** -24 * (k / 128 + 130)) * size + HALF_ULP[dtype] * np.abs(ref) * 1.001 + (3e-8 if dtype == F16 else 0)  # (half fp16's smallest step)


def off(got, ref, size, terms, k, dtype, label=""):
    error = np.abs(got.astype(np.float64) - ref)
    bound = bounds(k, dtype, ref, size)
    assert np.all(error <= bound), "%s off by %.3g at %s" % (label, error.max(), np.unravel_index(np.argmax(error - bound), error.shape))
    # terms: the sum of the squares of an element's terms.  Roundings of partial sums go either way.
    limit = (np.sqrt(k + 16) * 2.0 ** -24 + (2.0 ** -13.5 if dtype != F32 else 0)) * np.sqrt(terms.sum()) + HALF_ULP[dtype] * np.linalg.norm(ref)
    found = np.linalg.norm(got - ref)
    assert found <= limit, "%s: 2-norm of the error %.3g, at most %.3g" % (label, found, limit)


def product(hip, ops, m, n, k, c_dtype, bias=False, residual=False, pad=(0, 0, 0), offset=0, by_row=False, in_place=False, seed=0):
    rng = np.random.default_rng(m * 7 + n * 3 + k + seed)
    lda, ldb, ldc = k + pad[0], k + pad[1], n + pad[2]
    a, b = R.codes_of_normals(rng, (m, lda)), R.codes_of_normals(rng, (n, ldb))
    a[:, k:], b[:, k:] = 0x7F, 0xFF  # (what lies between rows is no number)
    up = hip.DeviceBuffer.from_numpy
    da, db = moved(hip, a, offset), moved(hip, b, offset)
    sa = (rng.uniform(0.5, 1.5, (m, R.blocks(k))) / 100).astype(np.float32)
    sb = (rng.uniform(0.5, 1.5, (R.blocks(n), R.blocks(k))) / 100 / np.sqrt(max(k, 1))).astype(np.float32)
    ref, size, terms = R.product(a[:, :k], sa, b[:, :k], sb)
    dbias = dres = None
    if bias:
        dbias, v = upload(hip, rng.standard_normal(n), c_dtype)
        ref, size = ref + v, size + np.abs(v)
    if residual:
        dres, v = upload(hip, rng.standard_normal((m, ldc)), c_dtype)
        ref, size = ref + v[:, :n], size + np.abs(v[:, :n])
    terms = terms + (ref ** 2 if bias or residual else 0)
    strides = (sa.shape[1], 1) if by_row else (0, 0)
    d = ops.MatmulFp8Desc(c_dtype, m, n, k, lda if pad[0] else 0, ldb if pad[1] else 0, ldc if pad[2] else 0, *strides)
    esz = hip.DTYPE_BYTES[c_dtype]
    need = ops.matmul_fp8_workspace_size(d)
    dsa, dsb = up(sa if by_row else np.ascontiguousarray(sa.T)), up(sb)
    for ws in ([hip.DeviceBuffer(need)] if need else []) + [None]:
        raws = []
        for again in range(2):
            if ws is not None:
                ws.fill(0xA5 if again else 0xFF)
            c = hip.DeviceBuffer(m * ldc * esz)
            c.fill(0x7E)
            if in_place and residual:
                c.upload(W.to_storage(np.asarray(v, np.float32), c_dtype)[0])
            ops.matmul_fp8(d, da, dsa, db, dsb, dbias, c if in_place and residual else dres, c, ws)
            raws.append(c.download(W.np_storage_dtype(c_dtype), (m, ldc)))
        raw = raws[0]
        assert np.array_equal(raw, raws[1]), "another result the second time"
        if ldc > n and not (in_place and residual):
            assert np.all(raw.view(np.uint8).reshape(m, ldc, esz)[:, n:] == 0x7E), "elements between rows were written"
        off(values(raw, c_dtype)[:, :n], ref, size, terms, k, c_dtype, "%d x %d x %d%s" % (m, n, k, "" if ws is None else " with a workspace"))


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 16), (1, 4096, 4096), (2, 100, 4160), (4, 14336, 2048), (7, 1024, 14336), (15, 68, 704), (16, 512, 640),
                                   (16, 4096, 4096), (17, 6144, 320), (31, 64, 128), (33, 68, 704), (48, 512, 2048), (64, 14340, 320), (64, 4096, 7168),
                                   (65, 128, 1024), (100, 5500, 192), (127, 129, 272), (128, 128, 128), (129, 4096, 2048), (255, 257, 4096), (256, 256, 64),
                                   (300, 1000, 16), (512, 3000, 2048), (1111, 2048, 1024), (2049, 300, 528), (1000, 24, 8192), (2500, 16, 256), (32, 2048, 16384)])
def test_products(hip, ops, m, n, k):  # noqa: F811
    print("[fp8]", m, n, k, flush=True)
    for c_dtype in (BF16, F16, F32):
        product(hip, ops, m, n, k, c_dtype)
    product(hip, ops, m, n, k, BF16, bias=True, residual=True)


@pytest.mark.parametrize("m,n,k", [(4100, 4096, 512), (3000, 6160, 656), (8192, 2048, 1040), (2300, 8192, 4096), (7001, 4112, 528), (5000, 4096, 640)])
def test_many_rows(hip, ops, m, n, k):  # noqa: F811
    """Tiles of 256 x 256 by workgroups that stay: several tiles each, short last stages, edges in both directions."""
    product(hip, ops, m, n, k, BF16, bias=True)
    product(hip, ops, m, n, k, F16, residual=True, by_row=True)


@pytest.mark.parametrize("m,n,k", [(7001, 1728, 1024), (1501, 8256, 1024), (2751, 4416, 1152), (9000, 8256, 512)])
def test_tiles_of_256_rows(hip, ops, m, n, k):  # noqa: F811
    """Sizes that go to workgroups that stay: one tile each and several, an even and an odd number of stages, edges in both directions."""
    product(hip, ops, m, n, k, BF16, bias=True)
    product(hip, ops, m, n, k, F16, residual=True, by_row=True, pad=(16, 64, 8))
    product(hip, ops, m, n, k, F16, residual=True, by_row=True, pad=(16, 48, 8))
    if m * n < 1 << 24:
        product(hip, ops, m, n, k, BF16, bias=True, residual=True, in_place=True)


@pytest.mark.parametrize("m,n,k", [(1751, 6949, 2048), (2001, 6181, 2048)])
def test_columns_beside_whole_runs(hip, ops, m, n, k):  # noqa: F811
    """Tiles of 256 rows for whole runs of 64 columns, a launch of its own for the rest, which begins at a block of scales or inside one."""
    product(hip, ops, m, n, k, BF16, bias=True, residual=True)
    product(hip, ops, m, n, k, F16, residual=True, by_row=True, pad=(16, 64, 8), in_place=True)


def test_columns_beside_an_odd_number_of_runs(hip, ops):  # noqa: F811
    """The second launch begins 64 columns into a block of the weights' scales: column 6,208."""
    product(hip, ops, 2001, 6245, 2048, BF16, bias=True, residual=True)
    product(hip, ops, 2001, 6245, 2048, F16, residual=True, by_row=True, pad=(16, 64, 8), in_place=True)


def far_apart(hip, scales, row, block):
    """scales [rows, blocks] some way apart in a large buffer, where a row's or a block's lie side by side"""
    assert min(row, block) == 1
    held = hip.DeviceBuffer(4 * ((scales.shape[0] - 1) * row + (scales.shape[1] - 1) * block + 1))
    for i, run in enumerate(scales if block == 1 else np.ascontiguousarray(scales.T)):
        hip.check(hip.lib().hipattn_memcpy_h2d_async(ctypes.c_void_p(held.ptr.value + 4 * i * max(row, block)), run.ctypes.data_as(ctypes.c_void_p), run.nbytes, None))
    hip.check(hip.lib().hipattn_stream_synchronize(None))
    return held


@pytest.mark.parametrize("row,block", [(1, (1 << 30) + 8), (160000, 1)])
def test_scales_far_apart(hip, ops, row, block):  # noqa: F811
    """Scales that 32 bits do not reach from the first (34 and 4.5 GB of them): the same results as side by side."""
    m, n, k = 7001, 1728, 1024
    rng = np.random.default_rng(row)
    a, b = hip.DeviceBuffer.from_numpy(R.codes_of_normals(rng, (m, k))), hip.DeviceBuffer.from_numpy(R.codes_of_normals(rng, (n, k)))
    sa, sb = (rng.uniform(0.5, 1.5, (r, 8)).astype(np.float32) for r in (m, -(-n // 128)))
    results = []
    for strides, scales in (((row, block), far_apart(hip, sa, row, block)), ((8, 1), hip.DeviceBuffer.from_numpy(sa))):
        d = ops.MatmulFp8Desc(F32, m, n, k, 0, 0, 0, *strides)
        for dtype in (F32, BF16):
            d.c_dtype = dtype
            c = hip.DeviceBuffer(m * n * 4)
            c.fill(0)
            ops.matmul_fp8(d, a, scales, b, hip.DeviceBuffer.from_numpy(sb), None, None, c, None)
            results.append(values(c.download(W.np_storage_dtype(dtype), (m, n)), dtype))
    assert np.array_equal(results[0], results[2])
    assert np.linalg.norm(results[1] - results[3]) <= 2.0 ** -7 * np.linalg.norm(results[3])


@pytest.mark.parametrize("m,n,k", [(1, 77, 33), (5, 33, 4095), (16, 100, 31), (64, 513, 777), (130, 257, 1001), (300, 66, 17), (3, 5, 7), (520, 300, 100), (40, 200, 129)])
def test_odd_sizes(hip, ops, m, n, k):  # noqa: F811
    for c_dtype in (BF16, F32):
        product(hip, ops, m, n, k, c_dtype, bias=True)


@pytest.mark.parametrize("m", [1, 16, 40, 130, 600])
def test_strides_and_alignment(hip, ops, m):  # noqa: F811
    product(hip, ops, m, 320, 256, BF16, pad=(16, 32, 0))
    product(hip, ops, m, 320, 256, F16, pad=(0, 0, 8), residual=True, bias=True)
    product(hip, ops, m, 320, 256, F32, pad=(3, 5, 7), residual=True)
    product(hip, ops, m, 321, 384, F32, pad=(16, 0, 3), residual=True, bias=True)
    product(hip, ops, m, 320, 256, BF16, offset=1)
    product(hip, ops, m, 320, 256, BF16, offset=16)
    product(hip, ops, m, 320, 640, F32, by_row=True)
    product(hip, ops, m, 320, 256, BF16, residual=True, in_place=True)


@pytest.mark.parametrize("m", [1, 20, 70, 300])
def test_no_columns_no_k(hip, ops, m):  # noqa: F811
    one = np.arange(40, dtype=np.float32)
    c = hip.DeviceBuffer(m * 40 * 4)
    c.fill(0xFF)
    ops.matmul_fp8(ops.MatmulFp8Desc(F32, m, 40, 0), None, None, None, None, hip.DeviceBuffer.from_numpy(one), None, c)
    assert np.array_equal(c.download(np.float32, (m, 40)), np.broadcast_to(one, (m, 40)))
    ops.matmul_fp8(ops.MatmulFp8Desc(F32, m, 0, 128), None, None, None, None, None, None, None)
    ops.matmul_fp8(ops.MatmulFp8Desc(F32, 0, 40, 128), None, None, None, None, None, None, None)


@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (20, 256, 512), (70, 256, 512), (300, 256, 512), (40, 256, 500), (600, 512, 4096)])
def test_what_is_no_number_stays_where_it_is(hip, ops, m, n, k):  # noqa: F811
    """NaN codes, infinite and NaN scales reach their rows (blocks of columns) and no others."""
    rng = np.random.default_rng(5)
    a, b = R.codes_of_normals(rng, (m, k)), R.codes_of_normals(rng, (n, k))
    sa, sb = np.full((m, R.blocks(k)), 0.01, np.float32), np.full((R.blocks(n), R.blocks(k)), 0.01, np.float32)
    up = hip.DeviceBuffer.from_numpy
    d = ops.MatmulFp8Desc(F32, m, n, k)
    need = ops.matmul_fp8_workspace_size(d)
    ws = hip.DeviceBuffer(need) if need else None

    def call():
        c = hip.DeviceBuffer(m * n * 4)
        ops.matmul_fp8(d, up(a), up(np.ascontiguousarray(sa.T)), up(b), up(sb), None, None, c, ws)
        return c.download(np.float32, (m, n))

    want = call()
    assert np.all(np.isfinite(want))
    row, column = m // 2, 133
    a[row, k - 1], b[column, 0] = 0x7F, 0xFF
    if m > 3:
        sa[1, 1], sa[3, 0] = np.inf, np.nan
    sb[0, 2] = np.inf
    got = call()
    bad = np.zeros((m, n), bool)
    bad[row], bad[:, column], bad[:, :128] = True, True, True
    if m > 3:
        bad[[1, 3]] = True
    assert np.array_equal(got[~bad], want[~bad]) and not np.any(np.isfinite(got[bad]))


def test_offsets_beyond_32_bits(hip, ops):  # noqa: F811
    """Rows of a and b that lie more than 2^32 bytes behind the first: a stride of 2^26 bytes, read and not stored in between."""
    m, n, k, ld = 70, 40, 256, 1 << 26
    rng = np.random.default_rng(8)
    a, b = R.codes_of_normals(rng, (m, k)), R.codes_of_normals(rng, (n, k))
    lib, check = hip.lib(), hip.check
    big = {}
    for name, x in (("a", a), ("b", b)):
        big[name] = hip.DeviceBuffer(ld * x.shape[0])
        for r in range(x.shape[0]):
            row = np.ascontiguousarray(x[r])
            check(lib.hipattn_memcpy_h2d_async(ctypes.c_void_p(big[name].ptr.value + r * ld), row.ctypes.data_as(ctypes.c_void_p), k, None))
            check(lib.hipattn_stream_synchronize(None))
    sa, sb = np.full((m, 2), 0.01, np.float32), np.full((1, 2), 0.01, np.float32)
    up = hip.DeviceBuffer.from_numpy
    results = []
    for lda, ldb, x, w in ((0, 0, up(a), up(b)), (ld, ld, big["a"], big["b"])):
        for rows in (1, 16, m):
            c = hip.DeviceBuffer(rows * n * 4)
            ops.matmul_fp8(ops.MatmulFp8Desc(F32, rows, n, k, lda, ldb, 0, 2, 1), x, up(sa), w, up(sb), None, None, c)
            results.append(c.download(np.float32, (rows, n)))
    ref, size, _ = R.product(a, sa, b, sb)
    for got in results:
        assert np.all(np.abs(got - ref[:len(got)]) <= bounds(k, F32, ref, size)[:len(got)])


@pytest.mark.parametrize("n,k", [(2, 1), (1, 16)])
def test_more_rows_than_a_launch_takes(hip, ops, n, k):  # noqa: F811
    """2^30 rows and some, at any address and at multiples of 16 bytes, go in several launches: rows of ones, and some others about the launches' ends."""
    m = (1 << 30) + 5000
    a, s, c = hip.DeviceBuffer(m * k), hip.DeviceBuffer(m * 4), hip.DeviceBuffer(m * n * 2)
    a.fill(0x38)
    s.fill(0x3F)
    c.fill(0x7E)
    scale, one = np.full(4, 0x3F, np.uint8).view(np.float32)[0], np.full((1, k), 0x38, np.uint8)
    rng = np.random.default_rng(n)
    rows = [0, 1, 127, (1 << 28) - 1, 1 << 28, (1 << 29) + 77, (1 << 30) - 1, 1 << 30, m - 1]
    some = R.codes_of_normals(rng, (len(rows), k))
    b = R.codes_of_normals(rng, (n, k))
    for r, x in zip(rows, some):
        hip.check(hip.lib().hipattn_memcpy_h2d_async(ctypes.c_void_p(a.ptr.value + r * k), x.ctypes.data_as(ctypes.c_void_p), k, None))
    hip.check(hip.lib().hipattn_stream_synchronize(None))
    ops.matmul_fp8(ops.MatmulFp8Desc(F16, m, n, k), a, s, hip.DeviceBuffer.from_numpy(b), hip.DeviceBuffer.from_numpy(np.full((1, 1), 0.01, np.float32)), None, None, c)
    got = c.download(np.uint16, (m, n))
    # a block's sum of 16 products or one: bounds() with the instruction's share, which is not there for one
    ref, size, _ = R.product(np.concatenate([some, one]), np.full((len(rows) + 1, 1), scale), b, np.full((1, 1), 0.01, np.float32))
    assert np.all(np.abs(values(got[rows], F16) - ref[:-1]) <= bounds(k, F16, ref, size)[:-1])
    assert np.all(np.abs(values(got[2], F16) - ref[-1]) <= bounds(k, F16, ref, size)[-1])
    got[rows] = got[2]
    assert np.all(got == got[2])
