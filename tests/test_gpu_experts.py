"""Routing to experts, the experts' products and the sum over a token's experts (include/hipops_experts.h) against numpy.

Routing compares in 64 bits, so indices and lists equal the reference's; weights are fp64 results rounded to fp32 (a few 2^-53 in front of
that).  Products: the bounds of test_gpu_fp8_ops.py.  Sums of top_k terms: top_k 2^-24 of the terms' magnitudes and the result's rounding."""
import numpy as np
import pytest

import experts_reference as R
from openvino_contrib_amd import workloads as W
from test_gpu_fp8_ops import HALF_ULP, bounds, near, off, values
from test_gpu_layer_ops import BF16, F16, F32, ops, upload  # noqa: F401

pytestmark = pytest.mark.gpu
E4M3 = 105


# ------------------------------------------------------------------------------ routing
def routed(hip, ops, logits, bias, top_k, dtype=F32, score="softmax", groups=1, kept=1, group_top=1, renormalise=True, scale=1.0, stride=0, lists=True, stream=None):
    tokens, experts = logits.shape
    padded = np.full((tokens, stride or experts), 1e9, np.float32)
    padded[:, :experts] = logits
    dl, exact = upload(hip, padded, dtype)
    d = ops.RouteDesc(dtype, ops.ROUTE_SIGMOID if score == "sigmoid" else ops.ROUTE_SOFTMAX, int(renormalise), experts, top_k, groups, kept, group_top, scale, tokens, stride)
    pairs = tokens * top_k
    new = [hip.DeviceBuffer(max(4, n)) for n in (4 * pairs, 4 * pairs, 4 * (experts + 1), 4 * pairs, 4 * pairs)]
    for b in new:
        b.fill(0xEE)
    need = ops.route_experts_workspace_size(d)
    ws = hip.DeviceBuffer(need) if need else None
    if ws:
        ws.fill(0xA5)
    db = hip.DeviceBuffer.from_numpy(np.asarray(bias, np.float32)) if bias is not None else None
    ops.route_experts(d, dl, db, *new[:2], *(new[2:] if lists else (None,) * 3), workspace=ws, stream=stream)
    kinds = (np.int32, np.float32, np.int32, np.int32, np.int32)
    shapes = ((tokens, top_k), (tokens, top_k), (experts + 1,), (pairs,), (tokens, top_k))
    return [b.download(t, s) for b, t, s in zip(new, kinds, shapes)], exact[:, :experts]


def check_routing(hip, ops, logits, bias, top_k, **how):
    (indices, weights, begins, order, slots), exact = routed(hip, ops, logits, bias, top_k, **how)
    ref = {k: v for k, v in how.items() if k not in ("dtype", "stride")}
    want, want_weights = R.route(exact.astype(np.float64), bias, top_k, **ref)
    assert np.array_equal(indices, want), np.argwhere(indices != want)[:4]
    assert np.all(np.abs(weights - want_weights) <= np.abs(want_weights) * 2.0 ** -23)
    for got, ref in zip((begins, order, slots), R.lists(want, logits.shape[1])):
        assert np.array_equal(got, ref)


@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (1, 8, 2), (3, 60, 4), (64, 64, 8), (5, 65, 65 - 1), (33, 128, 6), (200, 160, 6), (16, 256, 8), (17, 256, 8), (130, 384, 10),
                                                  (7, 1024, 64), (1000, 8, 8), (3000, 16, 2), (1, 256, 8), (4, 512, 3), (9000, 64, 8), (2, 63, 63)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_routing(hip, ops, tokens, experts, top_k, score):  # noqa: F811
    rng = np.random.default_rng(tokens + experts)
    logits = rng.standard_normal((tokens, experts)) * 1.5
    bias = rng.standard_normal(experts).astype(np.float32) * np.float32(0.05)
    for dtype in (F32, BF16):  # (logits of 16 bits: equal ones are common)
        check_routing(hip, ops, logits, None, top_k, dtype=dtype, score=score)
    check_routing(hip, ops, logits, bias, top_k, dtype=F16, score=score, renormalise=False, scale=2.5)
    check_routing(hip, ops, logits, bias, top_k, score=score, stride=experts + 3)


@pytest.mark.parametrize("experts,groups,kept,top_k", [(8, 4, 2, 3), (64, 8, 3, 6), (256, 8, 4, 8), (160, 8, 3, 6), (256, 64, 5, 20), (64, 64, 9, 9), (1024, 2, 1, 64), (100, 10, 10, 7), (6, 2, 1, 3)])
@pytest.mark.parametrize("group_top", [1, 2])
def test_routing_in_groups(hip, ops, experts, groups, kept, top_k, group_top):  # noqa: F811
    rng = np.random.default_rng(experts + groups)
    logits = rng.standard_normal((67, experts)) * 1.5
    bias = rng.standard_normal(experts).astype(np.float32) * np.float32(0.05)
    for score in ("softmax", "sigmoid"):
        for b in (None, bias):
            check_routing(hip, ops, logits, b, top_k, score=score, groups=groups, kept=kept, group_top=group_top, scale=2.5)


def test_equal_and_nearly_equal_choices(hip, ops):  # noqa: F811
    """Ties go to the lowest index, within a row, between lanes and between groups; scores that fp32 would call equal do not."""
    ones = np.zeros((3, 256))
    check_routing(hip, ops, ones, None, 8)
    check_routing(hip, ops, ones, None, 8, groups=8, kept=4, group_top=2)
    check_routing(hip, ops, ones, np.zeros(256, np.float32), 8, score="sigmoid", groups=8, kept=4, group_top=2)
    few = np.random.default_rng(1).integers(0, 3, (50, 256)).astype(np.float64)
    for groups in (1, 8):
        check_routing(hip, ops, few, None, 8, groups=groups, kept=3, group_top=1)
        check_routing(hip, ops, few, None, 8, score="sigmoid", groups=groups, kept=3, group_top=2)
    # neighbouring fp32 numbers near 12: their sigmoids differ by some 2^-42
    x = np.float32(12) + np.arange(64, dtype=np.float32) * np.float32(2.0 ** -20)
    rows = np.stack([np.random.default_rng(s).permutation(x) for s in range(20)]).astype(np.float64)
    check_routing(hip, ops, rows, None, 8, score="sigmoid")
    check_routing(hip, ops, rows, np.full(64, 0.25, np.float32), 8, score="sigmoid")
    # sums of a score and a bias that agree to fp32
    logits = np.random.default_rng(2).standard_normal((40, 64))
    near_ties = (-1 / (1 + np.exp(-logits[0].astype(np.float32).astype(np.float64)))).astype(np.float32)
    check_routing(hip, ops, np.broadcast_to(logits[0], (4, 64)).copy(), near_ties, 8, score="sigmoid")


def test_logits_that_are_no_numbers(hip, ops):  # noqa: F811
    rng = np.random.default_rng(3)
    for score in ("softmax", "sigmoid"):
        logits = rng.standard_normal((12, 64))
        logits[0] = -np.inf
        logits[1] = np.nan
        logits[2, 5] = np.inf
        logits[3, [7, 9]] = np.inf
        logits[4, 3] = np.nan
        logits[5, 1:] = -np.inf
        logits[6] = np.finfo(np.float32).min
        logits[7] = -1000.0
        logits[8, 8:] = np.nan
        logits[9, :60] = -np.inf
        for groups in (1, 8):
            check_routing(hip, ops, logits, None, 8, score=score, groups=groups, kept=2, group_top=2)
        bias = np.zeros(64, np.float32)
        bias[10:20], bias[30] = -np.inf, np.nan
        check_routing(hip, ops, logits, bias, 60, score=score)
        check_routing(hip, ops, logits, bias, 8, score=score)


def test_routing_without_tokens_or_lists(hip, ops):  # noqa: F811
    d = ops.RouteDesc(F32, 0, 1, 16, 2, 1, 1, 1, 1.0, 0, 0)
    begins = hip.DeviceBuffer(17 * 4)
    begins.fill(0xEE)
    ops.route_experts(d, None, None, None, None, begins, None, None)
    assert not begins.download(np.int32, (17,)).any()
    ops.route_experts(d, None, None, None, None)
    logits = np.random.default_rng(4).standard_normal((40, 16))
    with_lists, _ = routed(hip, ops, logits, None, 2)
    without, _ = routed(hip, ops, logits, None, 2, lists=False)
    assert np.array_equal(with_lists[0], without[0]) and np.array_equal(with_lists[1], without[1])
    assert np.all(without[2].view(np.uint8) == 0xEE)


def test_lists_of_one_sought_expert(hip, ops):  # noqa: F811
    """All tokens at the same experts, and experts without any: counts far apart."""
    logits = np.tile(np.linspace(3, -3, 300), (5000, 1))
    check_routing(hip, ops, logits, None, 3)
    check_routing(hip, ops, -logits, None, 1, score="sigmoid")


@pytest.mark.parametrize("tokens", [8, 9, 1024, 1025, 4096, 4097, 32768, 32769, 1 << 18, (1 << 18) + 1, 700001])
@pytest.mark.parametrize("experts,top_k", [(5, 2), (130, 3)])
def test_lists_about_the_lengths_of_runs(hip, ops, tokens, experts, top_k):  # noqa: F811
    """Every token chooses expert 3 (a run's count of it is the run's length, 224 at most), and others as they come."""
    logits = np.random.default_rng(tokens).standard_normal((tokens, experts)).astype(np.float32)
    logits[:, 3] = 9
    (indices, weights, *found), _ = routed(hip, ops, logits, None, top_k)
    want = np.argsort(-logits, 1, kind="stable")[:, :top_k]
    assert np.array_equal(indices, want)
    for got, ref in zip(found, R.lists(indices, experts)):
        assert np.array_equal(got, ref)
    y = np.exp(np.take_along_axis(logits, want, 1).astype(np.float64))
    y /= y.sum(1, keepdims=True)
    assert np.all(np.abs(weights - y) <= y * 2.0 ** -23)


def test_routing_of_more_tokens_than_a_launch_takes(hip, ops):  # noqa: F811
    """224 tokens to a workgroup of 1,024 threads: 2^32 of those are passed, and the call (without lists) goes in two launches.  Rows of equal logits, some others
    about the launches' ends."""
    import ctypes

    most = 224 * ((1 << 32) // 1024 - 1)
    tokens = most + 5000
    logits, indices, weights = hip.DeviceBuffer(4 * tokens), hip.DeviceBuffer(4 * tokens), hip.DeviceBuffer(4 * tokens)
    logits.fill(0)
    indices.fill(0xEE)
    weights.fill(0xEE)
    rows, row = [3, 1 << 28, most - 1, most, most + 300, tokens - 1], np.array([-1, 1], np.float16)
    for r in rows:
        hip.check(hip.lib().hipattn_memcpy_h2d_async(ctypes.c_void_p(logits.ptr.value + 4 * r), row.ctypes.data_as(ctypes.c_void_p), 4, None))
    hip.check(hip.lib().hipattn_stream_synchronize(None))
    ops.route_experts(ops.RouteDesc(logits_dtype=F16, experts=2, top_k=1, scale=3.0, tokens=tokens), logits, None, indices, weights)
    got = indices.download(np.int32, (tokens,))
    assert np.all(got[rows] == 1)
    got[rows] = 0
    assert not got.any()
    got = weights.download(np.float32, (tokens,))
    assert np.all(np.abs(got[rows] - 3 / (1 + np.exp(-2.0))) <= 3 * 2.0 ** -23)
    got[rows] = 1.5
    assert np.all(got == 1.5)


# ------------------------------------------------------------------------------ products
def experts_case(seed, counts, n, k, tokens=None, top_k=1):
    """Codes and lists of experts with `counts` rows; tokens: of that many rows of a, each place a random one."""
    rng = np.random.default_rng(seed)
    E, rows = len(counts), int(sum(counts))
    begins = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    a_rows = tokens if tokens else max(rows, 1)
    a, b = R.codes_of_normals(rng, (a_rows, k)), R.codes_of_normals(rng, (E, n, k))
    sa = (rng.uniform(0.5, 1.5, (a_rows, R.blocks(k))) / 100).astype(np.float32)
    sb = (rng.uniform(0.5, 1.5, (E, R.blocks(n), R.blocks(k))) / 100 / np.sqrt(k)).astype(np.float32)
    order = rng.integers(0, a_rows * top_k, rows).astype(np.int32) if tokens else None
    return dict(E=E, rows=rows, begins=begins, a=a, b=b, sa=sa, sb=sb, order=order, n=n, k=k, top_k=top_k)


def experts_reference(c):
    ref, size, terms = (np.zeros((c["rows"], c["n"])) for _ in range(3))
    for e in range(c["E"]):
        p = slice(c["begins"][e], c["begins"][e + 1])
        at = np.arange(c["rows"])[p] if c["order"] is None else c["order"][p] // c["top_k"]
        if len(at):
            ref[p], size[p], terms[p] = R.product(c["a"][at], c["sa"][at], c["b"][e], c["sb"][e])
    return ref, size, terms


def run_experts(hip, ops, c, c_dtype, spare=0, gated=False, act=0, gate_first=1, pad=0, by_row=False, workspace=None):
    up = hip.DeviceBuffer.from_numpy
    a_rows, k, n = c["a"].shape[0], c["k"], c["n"]
    stored = np.full((a_rows, k + pad), 0x7F, np.uint8)
    stored[:, :k] = c["a"]
    rows = c["rows"] + spare
    strides = (c["sa"].shape[1], 1) if by_row else (0, 0)
    gated = gated or c_dtype == E4M3
    d = ops.MatmulFp8ExpertsDesc(c_dtype, int(gated), act, gate_first, c["top_k"], c["E"], rows, n, k, a_rows, k + pad if pad else 0, *strides)
    width, esz = n // 2 if gated else n, 1 if c_dtype == E4M3 else hip.DTYPE_BYTES[c_dtype]
    need = ops.matmul_fp8_experts_workspace_size(d)
    order = up(np.concatenate([c["order"], np.full(spare, -5, np.int32)])) if c["order"] is not None else None
    dev = [up(stored), up(c["sa"] if by_row else np.ascontiguousarray(c["sa"].T)), up(c["b"]), up(c["sb"]), up(c["begins"]), order]
    found = []
    for again in range(2):
        out, scales = hip.DeviceBuffer(max(1, rows * width * esz)), hip.DeviceBuffer(max(4, rows * R.blocks(width) * 4))
        out.fill(0x7E)
        scales.fill(0x7E)
        ws = hip.DeviceBuffer(workspace or need) if workspace or need else None
        if ws:
            ws.fill(0xFF if again else 0xA5)
        ops.matmul_fp8_experts(d, *dev, out, scales if c_dtype == E4M3 else None, ws)
        raw = out.download(np.uint8 if c_dtype == E4M3 else W.np_storage_dtype(c_dtype), (rows, width))
        s = scales.download(np.float32, (R.blocks(width), rows)).T
        assert np.all(raw[c["rows"]:].view(np.uint8) == 0x7E), "rows behind the last expert's were written"
        assert np.all(np.ascontiguousarray(s[c["rows"]:]).view(np.uint8) == 0x7E)
        found.append((raw[:c["rows"]], s[:c["rows"]]))
    assert np.array_equal(found[0][0], found[1][0]) and np.array_equal(found[0][1], found[1][1]), "another result the second time"
    return found[0]


COUNTS = {
    "none": [0, 0, 0],
    "one": [0, 1, 0, 0],
    "few": [3, 0, 1, 7, 2, 0, 5, 1],
    "sixteens": [16, 32, 0, 48, 16, 17, 15],
    "decode": [2] * 40 + [0] * 20 + [9, 30, 1, 1],
    "uneven": [130, 0, 257, 1, 64, 500, 3],
    "many": [700, 1100, 256, 0],
    "lone": [40],
    "large": [900, 0, 257, 1800, 128, 1],
}


def check_experts(hip, ops, counts, n, k, c_dtype, tokens=None, top_k=1, **how):
    c = experts_case(len(counts) + n + k, counts, n, k, tokens, top_k)
    print("[experts]", counts[:8], n, k, c_dtype, tokens, how, flush=True)
    raw, scales = run_experts(hip, ops, c, c_dtype, **how)
    if not c["rows"]:
        return
    ref, size, terms = experts_reference(c)
    if c_dtype != E4M3 and not how.get("gated"):
        off(values(raw, c_dtype), ref, size, terms, k, c_dtype)
        return
    act, gate_first = how.get("act", 0), how.get("gate_first", 1)
    y, each, half = R.gated(ref, act, gate_first), bounds(k, F32, ref, size, c_dtype != F32), n // 2
    gate, up = (slice(0, half), slice(half, n)) if gate_first else (slice(half, n), slice(0, half))
    # the activations' slope is below 1.13; their own error as in test_quantise_glu
    slack = 1.13 * each[:, gate] * (np.abs(ref[:, up]) + each[:, up]) + np.abs(ref[:, gate]) * each[:, up] + 2.0 ** -20 * np.abs(ref).max(1, keepdims=True) ** 2
    if c_dtype != E4M3:
        got = values(raw, c_dtype)
        assert np.all(np.abs(got - y) <= slack + HALF_ULP[c_dtype] * np.abs(y) * 1.001 + (3e-8 if c_dtype == F16 else 0))
        # the halves' errors in the 2-norm (see off) meet factors of the other half; three times that for their spread
        limit = 3 * (np.sqrt(k + 16) * 2.0 ** -24 + (2.0 ** -13.5 if c_dtype != F32 else 0)) * np.linalg.norm(np.sqrt(terms).max(1, keepdims=True) * np.abs(ref))
        assert np.linalg.norm(got - y) <= limit + 2.0 ** -20 * np.linalg.norm(y) + HALF_ULP[c_dtype] * np.linalg.norm(y)
        return
    near(raw, scales, y, slack)
    # in the 2-norm: half a step of a code is 2^-4 of it at most, half of that on average
    held = R.VALUES[raw] * R.spread(scales.astype(np.float64), half)
    assert np.linalg.norm(held - y) <= 2.0 ** -5 * np.linalg.norm(y)


@pytest.mark.parametrize("which", sorted(COUNTS))
@pytest.mark.parametrize("n,k", [(256, 256), (512, 1024), (200, 96), (640, 2048), (130, 4096), (528, 784)])
def test_experts_products(hip, ops, which, n, k):  # noqa: F811
    counts = COUNTS[which]
    if which == "decode" and n * k > 600000:
        counts = counts[30:]
    for c_dtype in (BF16, F32):
        check_experts(hip, ops, counts, n, k, c_dtype)
        check_experts(hip, ops, counts, n, k, c_dtype, tokens=37, top_k=3, spare=9)
    check_experts(hip, ops, counts, n, k, F16, tokens=5, by_row=True)


@pytest.mark.parametrize("which", sorted(COUNTS))
@pytest.mark.parametrize("n,k", [(256, 256), (512, 1024), (200, 96), (2560, 512), (384, 2048), (130, 130), (16, 128), (768, 656)])
def test_experts_gated(hip, ops, which, n, k):  # noqa: F811
    check_experts(hip, ops, COUNTS[which], n, k, BF16, gated=True, tokens=37, top_k=3, spare=5)
    check_experts(hip, ops, COUNTS[which], n, k, F32, gated=True, gate_first=0)
    check_experts(hip, ops, COUNTS[which], n, k, F16, gated=True, act=1)
    check_experts(hip, ops, COUNTS[which], n, k, E4M3)
    check_experts(hip, ops, COUNTS[which], n, k, E4M3, tokens=37, top_k=3, spare=5, gate_first=0)


@pytest.mark.parametrize("which", ["few", "decode", "uneven", "large"])
@pytest.mark.parametrize("n,k", [(588, 384), (1100, 384), (1270, 656), (1026, 131), (2302, 256)])
def test_experts_gated_widths_beside_the_blocks(hip, ops, which, n, k):  # noqa: F811
    """The second half's blocks of scales begin anywhere among a tile's columns: widths of 38, 38, 123, 1 and 127 beyond whole blocks."""
    check_experts(hip, ops, COUNTS[which], n, k, BF16, gated=True, tokens=37, top_k=3, spare=5)
    check_experts(hip, ops, COUNTS[which], n, k, F32, gated=True, gate_first=0)


@pytest.mark.parametrize("act", [0, 1, 2])
def test_experts_activations(hip, ops, act):  # noqa: F811
    for counts in (COUNTS["few"], COUNTS["uneven"]):
        for gate_first in (0, 1):
            check_experts(hip, ops, counts, 512, 256, E4M3, act=act, gate_first=gate_first)
            check_experts(hip, ops, counts, 512, 256, BF16, gated=True, act=act, gate_first=gate_first)


@pytest.mark.parametrize("n,k", [(77, 33), (513, 777), (258, 129)])
def test_experts_odd_sizes(hip, ops, n, k):  # noqa: F811
    for which in ("few", "uneven"):
        check_experts(hip, ops, COUNTS[which], n, k, F32, tokens=50, top_k=2)
        check_experts(hip, ops, COUNTS[which], n, k, BF16, pad=3)
        if n % 2 == 0:
            check_experts(hip, ops, COUNTS[which], n, k, E4M3, tokens=50)
    check_experts(hip, ops, COUNTS["uneven"], 256, 256, BF16, pad=16)
    check_experts(hip, ops, COUNTS["few"], 256, 256, BF16, pad=16)


def test_experts_codes_in_a_small_workspace(hip, ops):  # noqa: F811
    """A workspace that holds a few rows: the same codes, some rows at a time."""
    for which, n in (("few", 256), ("uneven", 256), ("few", 200), ("uneven", 200)):
        c = experts_case(1, COUNTS[which], n, 256, tokens=40)
        raw, scales = run_experts(hip, ops, c, E4M3)
        rows = 3 if which == "few" else 100
        again, again_scales = run_experts(hip, ops, c, E4M3, workspace=rows * n * 4 + 8)
        assert np.array_equal(raw, again) and np.array_equal(scales, again_scales)


@pytest.mark.parametrize("which", ["many", "large"])
@pytest.mark.parametrize("n,k", [(512, 1024), (256, 640)])
def test_experts_codes_some_rows_at_a_time(hip, ops, which, n, k):  # noqa: F811
    """The same where some rows at a time are enough for tiles of 256: launches that begin at other places than the first, inside an expert's."""
    c = experts_case(2, COUNTS[which], n, k, tokens=40)
    raw, scales = run_experts(hip, ops, c, E4M3)
    again, again_scales = run_experts(hip, ops, c, E4M3, workspace=700 * n // 2 * 4, spare=5)
    assert np.array_equal(raw, again) and np.array_equal(scales, again_scales)


@pytest.mark.parametrize("n,k,c_dtype,gated", [(256, 512, BF16, 0), (512, 640, F16, 1), (256, 512, F32, 0), (130, 100, BF16, 0)])
def test_more_places_than_a_launch_takes(hip, ops, n, k, c_dtype, gated):  # noqa: F811
    """More than 2^19 places go in two launches, which meet inside an expert's: places of the same expert and row have the same bits, and those are right."""
    begins = np.array([0, 100001, 100001, 520000, (1 << 19) + 3001], np.int32)
    c = experts_case(n + k, list(np.diff(begins)), n, k, tokens=37, top_k=2)
    out, width = c["rows"], n // 2 if gated else n
    up = hip.DeviceBuffer.from_numpy
    result = hip.DeviceBuffer((out + 3) * width * hip.DTYPE_BYTES[c_dtype])
    result.fill(0x7E)
    ops.matmul_fp8_experts(ops.MatmulFp8ExpertsDesc(c_dtype, gated, 0, 1, 2, c["E"], out, n, k, 37), up(c["a"]), up(np.ascontiguousarray(c["sa"].T)), up(c["b"]), up(c["sb"]),
                           up(begins), up(c["order"]), result)
    raw = result.download(W.np_storage_dtype(c_dtype), (out + 3, width))
    assert np.all(raw[out:].view(np.uint8) == 0x7E)
    expert, row = np.repeat(np.arange(c["E"]), np.diff(begins)), c["order"] // 2
    _, first, which = np.unique(expert * 37 + row, return_index=True, return_inverse=True)
    assert np.array_equal(raw[:out], raw[first][which])
    got = values(raw[first], c_dtype)
    ref, size, terms = (np.concatenate(x) for x in zip(*[R.product(c["a"][r][None], c["sa"][r][None], c["b"][e], c["sb"][e]) for e, r in zip(expert[first], row[first])]))
    if not gated:
        off(got, ref, size, terms, k, c_dtype)
        return
    each, gate, pair = bounds(k, F32, ref, size, True), slice(0, width), slice(width, n)
    # (as in check_experts)
    slack = 1.13 * each[:, gate] * (np.abs(ref[:, pair]) + each[:, pair]) + np.abs(ref[:, gate]) * each[:, pair] + 2.0 ** -20 * np.abs(ref).max(1, keepdims=True) ** 2
    y = R.gated(ref, 0, 1)
    assert np.all(np.abs(got - y) <= slack + HALF_ULP[c_dtype] * np.abs(y) * 1.001 + 3e-8)


@pytest.mark.parametrize("which", ["none", "few", "uneven", "large"])
@pytest.mark.parametrize("n", [2, 130, 512])
def test_experts_without_k(hip, ops, which, n):  # noqa: F811
    """Sums of nothing are zeros, their units and codes too."""
    counts = COUNTS[which]
    rows, spare, E = sum(counts), 3, len(counts)
    begins = hip.DeviceBuffer.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
    for c_dtype, gated in ((F32, 0), (BF16, 0), (F16, 1), (E4M3, 1)):
        width = n // 2 if gated else n
        size = 1 if c_dtype == E4M3 else hip.DTYPE_BYTES[c_dtype]
        d = ops.MatmulFp8ExpertsDesc(c_dtype, gated, 0, 1, 1, E, rows + spare, n, 0, rows + spare)
        out, scales = hip.DeviceBuffer((rows + spare) * width * size), hip.DeviceBuffer(4 * (rows + spare) * R.blocks(width))
        out.fill(0x7E)
        scales.fill(0x7E)
        ws = hip.DeviceBuffer(max(16, ops.matmul_fp8_experts_workspace_size(d)))
        ws.fill(0xA5)
        ops.matmul_fp8_experts(d, None, None, None, None, begins, None, out, scales if c_dtype == E4M3 else None, ws)
        got = out.download(np.uint8, (rows + spare, width * size))
        assert not np.any(got[:rows] & 0x7F) and np.all(got[rows:] == 0x7E)
        if c_dtype == E4M3:
            s = scales.download(np.uint32, (R.blocks(width), rows + spare))
            assert not s[:, :rows].any() and np.all(s[:, rows:] == 0x7E7E7E7E)


@pytest.mark.parametrize("which", ["few", "uneven", "many", "large"])
def test_experts_narrow_units_and_padded_rows(hip, ops, which):  # noqa: F811
    """One result column; rows with something between them and scales by row, in the tiles of 256 rows too."""
    for c_dtype in (BF16, F32):
        check_experts(hip, ops, COUNTS[which], 2, 256, c_dtype, gated=True, tokens=37, top_k=3, spare=5)
    check_experts(hip, ops, COUNTS[which], 2, 130, E4M3)
    for pad in (16, 48, 64):
        check_experts(hip, ops, COUNTS[which], 512, 1024, BF16, pad=pad, by_row=True)
        check_experts(hip, ops, COUNTS[which], 512, 1024, E4M3, pad=pad, by_row=True, tokens=37, top_k=3, spare=5)
        check_experts(hip, ops, COUNTS[which], 512, 1024, F16, gated=True, pad=pad, tokens=500)


def test_many_experts(hip, ops):  # noqa: F811
    rng = np.random.default_rng(0)
    for E in (65, 300, 1024):
        counts = rng.integers(0, 4, E)
        check_experts(hip, ops, list(counts), 128, 128, BF16, tokens=20, top_k=4)
        counts = np.where(rng.random(E) < 0.02, 90, 0)
        check_experts(hip, ops, list(counts), 128, 128, F32, tokens=20, top_k=4)


def test_lists_that_name_no_rows(hip, ops):  # noqa: F811
    """Entries beyond the arrays and begins out of order leave the call within them; what is right stays right."""
    for counts, n, k in (([5, 3, 40, 2], 256, 256), ([100, 300, 2, 70], 256, 256), ([5, 3, 40, 2], 130, 100)):
        c = experts_case(3, counts, n, k, tokens=20)
        ref, _ = run_experts(hip, ops, c, F32)
        c["order"][0], c["order"][6] = -1000000, 1 << 30
        got, _ = run_experts(hip, ops, c, F32)
        keep = np.ones(c["rows"], bool)
        keep[[0, 6]] = False
        assert np.array_equal(got[keep], ref[keep])
        c = experts_case(3, counts, n, k, tokens=20)
        c["begins"][1], c["begins"][2] = 1 << 30, -7
        d = ops.MatmulFp8ExpertsDesc(F32, 0, 0, 1, 1, c["E"], c["rows"], n, k, 20)
        up = hip.DeviceBuffer.from_numpy
        out = hip.DeviceBuffer(c["rows"] * n * 4)
        ops.matmul_fp8_experts(d, up(c["a"]), up(np.ascontiguousarray(c["sa"].T)), up(c["b"]), up(c["sb"]), up(c["begins"]), up(c["order"]), out)
        last = slice(c["begins"][3], c["begins"][4])
        out.download(np.float32, (c["rows"], n))[last]  # (the call comes back; its results here are nobody's)


@pytest.mark.parametrize("rows,n,k,gated", [(24, 256, 256, 1), (400, 256, 512, 0), (3000, 512, 512, 1), (3000, 512, 512, 0)])
def test_begins_that_overlap(hip, ops, rows, n, k, gated):  # noqa: F811
    """Begins that give every other expert all places: results are nobody's, but the call comes back and leaves what lies behind them."""
    rng = np.random.default_rng(rows)
    E, width = 8, n // 2 if gated else n
    up = hip.DeviceBuffer.from_numpy
    begins = np.array([0, rows, 0, rows, 0, 1 << 30, -5, rows, 0], np.int32)
    out = hip.DeviceBuffer((rows + 64) * width * 2)
    out.fill(0x7E)
    sa, sb = np.full((R.blocks(k), rows), 0.01, np.float32), np.full((E, R.blocks(n), R.blocks(k)), 0.01, np.float32)
    ops.matmul_fp8_experts(ops.MatmulFp8ExpertsDesc(BF16, gated, 0, 1, 1, E, rows, n, k, rows), up(R.codes_of_normals(rng, (rows, k))), up(sa), up(R.codes_of_normals(rng, (E, n, k))),
                           up(sb), up(begins), None, out)
    got = out.download(np.uint16, (rows + 64, width))
    assert np.all(got[rows:] == 0x7E7E) and not np.all(got[:rows] == 0x7E7E)


@pytest.mark.parametrize("which", ["few", "decode", "uneven", "large"])
def test_some_of_the_experts(hip, ops, which):  # noqa: F811
    """A device that holds some of the experts: their weights, and begins from theirs on; places of the others stay as they are."""
    import ctypes

    n, k = 512, 512
    c = experts_case(11, COUNTS[which], n, k, tokens=50, top_k=2)
    ref, size, terms = experts_reference(c)
    up = hip.DeviceBuffer.from_numpy
    first, last = c["E"] // 3, c["E"] - 1
    begins = up(c["begins"])
    part = type("Part", (), dict(ptr=ctypes.c_void_p(begins.ptr.value + 4 * first), nbytes=begins.nbytes - 4 * first))
    out = hip.DeviceBuffer(c["rows"] * n * 2)
    out.fill(0x7E)
    ops.matmul_fp8_experts(ops.MatmulFp8ExpertsDesc(BF16, 0, 0, 1, 2, last - first, c["rows"], n, k, 50), up(c["a"]), up(np.ascontiguousarray(c["sa"].T)), up(c["b"][first:last]),
                           up(c["sb"][first:last]), part, up(c["order"]), out)
    raw = out.download(np.uint16, (c["rows"], n))
    p = slice(c["begins"][first], c["begins"][last])
    assert np.all(raw[:p.start] == 0x7E7E) and np.all(raw[p.stop:] == 0x7E7E)
    off(values(raw[p], BF16), ref[p], size[p], terms[p], k, BF16)


@pytest.mark.parametrize("which", ["few", "decode", "uneven", "large"])
@pytest.mark.parametrize("rows_at_once", [0, 7])
def test_codes_of_some_of_the_experts(hip, ops, which, rows_at_once):  # noqa: F811
    """The same for codes, in a workspace for all places and for some at a time: two calls, for the first and the last experts, make one result in either order, and
    places of neither stay as they are."""
    import ctypes

    n, k = 512, 512
    c = experts_case(12, COUNTS[which], n, k, tokens=50, top_k=2)
    ref, size, _ = experts_reference(c)
    half, E, spare = n // 2, c["E"], 9
    rows = c["rows"] + spare
    if rows_at_once and c["rows"] > 200:
        rows_at_once = 130
    up = hip.DeviceBuffer.from_numpy
    a, sa, begins, order = up(c["a"]), up(np.ascontiguousarray(c["sa"].T)), up(c["begins"]), up(np.concatenate([c["order"], np.full(spare, -5, np.int32)]))
    cuts = [(E // 4, E // 2), (E // 2, E - 1)]
    held = {}
    for turn in (0, 1):
        out, scales = hip.DeviceBuffer(rows * half), hip.DeviceBuffer(4 * rows * R.blocks(half))
        out.fill(0x7E)
        scales.fill(0x7E)
        for first, last in cuts[::-1] if turn else cuts:
            d = ops.MatmulFp8ExpertsDesc(E4M3, 1, 0, 1, 2, last - first, rows, n, k, 50)
            part = type("Part", (), dict(ptr=ctypes.c_void_p(begins.ptr.value + 4 * first), nbytes=begins.nbytes - 4 * first))
            ws = hip.DeviceBuffer(4 * half * rows_at_once or ops.matmul_fp8_experts_workspace_size(d))
            ws.fill(0xA5)
            ops.matmul_fp8_experts(d, a, sa, up(c["b"][first:last]), up(c["sb"][first:last]), part, order, out, scales, ws)
        held[turn] = out.download(np.uint8, (rows, half)), np.ascontiguousarray(scales.download(np.float32, (R.blocks(half), rows)).T)
    assert np.array_equal(held[0][0], held[1][0]) and np.array_equal(held[0][1].view(np.uint32), held[1][1].view(np.uint32)), "another result in the other order"
    raw, s = held[0]
    p = slice(c["begins"][cuts[0][0]], c["begins"][cuts[1][1]])
    for outside in (slice(0, p.start), slice(p.stop, rows)):
        assert np.all(raw[outside] == 0x7E) and np.all(np.ascontiguousarray(s[outside]).view(np.uint8) == 0x7E), "places of other experts were written"
    each = bounds(k, F32, ref, size, True)
    gate, pair = slice(0, half), slice(half, n)
    # (as in check_experts)
    slack = 1.13 * each[:, gate] * (np.abs(ref[:, pair]) + each[:, pair]) + np.abs(ref[:, gate]) * each[:, pair] + 2.0 ** -20 * np.abs(ref).max(1, keepdims=True) ** 2
    near(raw[p], s[p], R.gated(ref, 0, 1)[p], slack[p])


def test_experts_weights_beyond_32_bits(hip, ops):  # noqa: F811
    """The last of 40 experts lies more than 2^32 bytes behind the first."""
    E, n, k = 40, 8192, 14336
    rng = np.random.default_rng(7)
    b, sb = R.codes_of_normals(rng, (n, k)), (rng.uniform(0.5, 1.5, (R.blocks(n), R.blocks(k))) / 1000).astype(np.float32)
    import ctypes
    weights = hip.DeviceBuffer(E * n * k)
    scales = np.zeros((E,) + sb.shape, np.float32)
    scales[-1] = sb
    hip.check(hip.lib().hipattn_memcpy_h2d_async(ctypes.c_void_p(weights.ptr.value + (E - 1) * n * k), b.ctypes.data_as(ctypes.c_void_p), n * k, None))
    hip.check(hip.lib().hipattn_stream_synchronize(None))
    up = hip.DeviceBuffer.from_numpy
    for rows in (3, 70):
        a, sa = R.codes_of_normals(rng, (rows, k)), np.full((rows, R.blocks(k)), 0.01, np.float32)
        begins = np.zeros(E + 1, np.int32)
        begins[-1] = rows
        out = hip.DeviceBuffer(rows * n * 4)
        ops.matmul_fp8_experts(ops.MatmulFp8ExpertsDesc(F32, 0, 0, 1, 1, E, rows, n, k, rows), up(a), up(np.ascontiguousarray(sa.T)), weights, up(scales), up(begins), None, out)
        got = out.download(np.float32, (rows, n))
        some = rng.permutation(n)[:64]
        x, w = R.VALUES[a] * 0.01, R.VALUES[b[some]] * R.spread(np.repeat(sb.astype(np.float64), 128, 0)[some], k)
        assert np.all(np.abs(got[:, some] - x @ w.T) <= 2.0 ** -24 * (k / 128 + 130) * (np.abs(x) @ np.abs(w).T) * 1.01)


# ------------------------------------------------------------------------------ the sum over a token's experts
@pytest.mark.parametrize("tokens,top_k,n", [(1, 1, 1), (1, 8, 4096), (64, 8, 4096), (3, 2, 37), (1000, 6, 520), (5, 1, 8), (2, 64, 2056), (700, 3, 100), (40, 2, 20000)])
@pytest.mark.parametrize("y_dtype,o_dtype", [(F32, F32), (F16, F16), (BF16, BF16), (F32, BF16), (BF16, F32)])
def test_combine(hip, ops, tokens, top_k, n, y_dtype, o_dtype):  # noqa: F811
    rng = np.random.default_rng(tokens + n)
    rows = tokens * top_k
    dy, y = upload(hip, rng.standard_normal((rows, n)), y_dtype)
    w, slots = rng.random((tokens, top_k)).astype(np.float32), rng.permutation(rows).astype(np.int32).reshape(tokens, top_k)
    slots[0, 0], slots[-1, -1] = -1, rows
    dw, ds = hip.DeviceBuffer.from_numpy(w), hip.DeviceBuffer.from_numpy(slots)
    dres, res = upload(hip, rng.standard_normal((tokens, n)), o_dtype)
    size = R.combine(np.abs(y), w, slots)
    for residual in (None, dres):
        want = R.combine(y, w, slots, res if residual else None)
        for in_place in (False, True):
            if in_place and not residual:
                continue
            out = hip.DeviceBuffer(tokens * n * hip.DTYPE_BYTES[o_dtype])
            if in_place:
                out.upload(W.to_storage(res, o_dtype)[0])
            ops.combine_experts(ops.CombineDesc(y_dtype, o_dtype, top_k, tokens, rows, n), dy, dw, ds, out if in_place else residual, out)
            got = values(out.download(W.np_storage_dtype(o_dtype), (tokens, n)), o_dtype)
            bound = (top_k + 1) * 2.0 ** -24 * (size + np.abs(res if residual else 0)) + HALF_ULP[o_dtype] * np.abs(want) * 1.001 + (3e-8 if o_dtype == F16 else 0)
            assert np.all(np.abs(got - want) <= bound)


def test_combine_alignment(hip, ops):  # noqa: F811
    """Rows off sixteen bytes, and sums beyond 2^32 bytes of rows are the next test's."""
    from test_gpu_fp8_ops import moved

    rng = np.random.default_rng(9)
    stored, y = W.to_storage(rng.standard_normal((20, 64)), BF16)
    w, slots = rng.random((10, 2)).astype(np.float32), rng.permutation(20).astype(np.int32).reshape(10, 2)
    want = R.combine(y, w, slots)
    for offset in (0, 2, 8):
        out = hip.DeviceBuffer(10 * 64 * 4)
        ops.combine_experts(ops.CombineDesc(BF16, F32, 2, 10, 20, 64), moved(hip, stored, offset), hip.DeviceBuffer.from_numpy(w), hip.DeviceBuffer.from_numpy(slots), None, out)
        assert np.allclose(out.download(np.float32, (10, 64)), want, rtol=1e-6, atol=1e-6)


def test_combine_rows_beyond_32_bits(hip, ops):  # noqa: F811
    n, rows = 8192, 300000  # 4.9 GB of bf16
    y = hip.DeviceBuffer(rows * n * 2)
    y.fill(0)
    import ctypes
    one = np.full(n, 0x3F80, np.uint16)
    for at in (rows - 1, 5):
        hip.check(hip.lib().hipattn_memcpy_h2d_async(ctypes.c_void_p(y.ptr.value + at * n * 2), one.ctypes.data_as(ctypes.c_void_p), 2 * n, None))
    hip.check(hip.lib().hipattn_stream_synchronize(None))
    up = hip.DeviceBuffer.from_numpy
    out = hip.DeviceBuffer(n * 4)
    ops.combine_experts(ops.CombineDesc(BF16, F32, 2, 1, rows, n), y, up(np.array([[2.0, 3.0]], np.float32)), up(np.array([[rows - 1, 5]], np.int32)), None, out)
    assert np.all(out.download(np.float32, (n,)) == 5.0)


def test_combine_of_more_tokens_than_a_launch_takes(hip, ops):  # noqa: F811
    """A lane for each of seven columns: 2^32 threads are passed, and the call goes in two launches.  Thirteen rows over and over, added to what is there."""
    n, rows = 7, 13
    tokens = 0xFFFFFF00 // n + 3000
    rng = np.random.default_rng(10)
    stored, y = W.to_storage(rng.standard_normal((rows, n)), F16)
    up = hip.DeviceBuffer.from_numpy
    slots, weights, out = up(np.tile(np.arange(rows, dtype=np.int32), -(-tokens // rows))[:tokens]), hip.DeviceBuffer(4 * tokens), hip.DeviceBuffer(2 * n * tokens)
    weights.fill(0x3F)
    out.fill(0x3C)
    ops.combine_experts(ops.CombineDesc(F16, F16, 1, tokens, rows, n), up(stored), weights, slots, out, out)
    got = out.download(np.uint16, (tokens, n))
    weight, residual = (np.full(4, b, np.uint8).view(t)[0].astype(np.float64) for b, t in ((0x3F, np.float32), (0x3C, np.float16)))
    want = residual + weight * y
    # one product and one sum in fp32, one rounding
    assert np.all(np.abs(values(got[:rows], F16) - want) <= 2.0 ** -23 * (residual + np.abs(weight * y)) + HALF_ULP[F16] * np.abs(want) * 1.001 + 3e-8)
    whole = tokens // rows * rows
    assert np.all(got[:whole].reshape(-1, rows, n) == got[:rows]) and np.all(got[whole:] == got[:tokens - whole])
