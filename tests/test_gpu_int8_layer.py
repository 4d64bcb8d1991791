"""A decoder layer's step in 8 bits (int8_layer.py) against the same chain in fp64, which rounds where the layer does: activations to codes
ahead of each product, keys and values to codes, operators' results to bf16.

Bound: six roundings to bf16 (2^-9 of a value each, rms) and codes that fall the other way because the value in front of them was
rounded differently (a step, 1/127 of a row's largest, for the share of values that lie within 2^-9 of a half): below 1e-2 of the
result in the 2-norm."""
import numpy as np
import pytest

import int8_reference as R
from int8_reference import BF16
from openvino_contrib_amd import workloads as W

pytestmark = pytest.mark.gpu


def bf16(x):
    return W.bf16_bits_to_f32(W.f32_to_bf16_bits(np.asarray(x, np.float32)))


class Reference:
    def __init__(self, weights, gammas, heads, kv_heads, D):
        self.w, self.g, self.H, self.K, self.D = weights, gammas, heads, kv_heads, D

    def product(self, name, y):
        codes, scales = self.w[name]
        y = np.asarray(y, np.float64)
        s = np.abs(y).max(1) / 127
        c = np.rint(y / np.where(s > 0, s, 1)[:, None])
        return (c @ codes.astype(np.float64).T) * s[:, None] * scales

    def norm(self, x, g):
        x = x.astype(np.float64)
        return x / np.sqrt((x ** 2).mean(1, keepdims=True) + 1e-5) * g

    def step(self, b, x, cos, sin):
        H, K, D, T = self.H, self.K, self.D, b.tokens
        place = np.concatenate([past + np.arange(new) for past, new in b.seqs])
        qkv = bf16(self.product("qkv", self.norm(x, self.g[0])))
        q, k, v = np.split(qkv.reshape(T, H + 2 * K, D), [H, H + K], 1)
        q = bf16(R.rotated(q, cos[place], sin[place], D, False))
        b.append(R.rotated(k, cos[place], sin[place], D, False), v)
        attended = bf16(b.attention(q).reshape(T, H * D))
        inner = bf16(self.product("o", attended) + x)
        gated = bf16(self.product("gate_up", self.norm(inner, self.g[1]))).astype(np.float64)
        ffn = gated.shape[1] // 2
        return bf16(self.product("down", gated[:, :ffn] / (1 + np.exp(-gated[:, :ffn])) * gated[:, ffn:]) + inner)


@pytest.mark.parametrize("seqs", [[(40, 1)], [(100, 1), (31, 1), (0, 1), (500, 1)], [(0, 90), (33, 1), (64, 40), (0, 3)]])
@pytest.mark.parametrize("H,K,D,hidden,ffn", [(8, 2, 64, 512, 1024), (4, 1, 128, 256, 704)])
def test_layer_steps(hip, H, K, D, hidden, ffn, seqs):
    from openvino_contrib_amd import int8_layer as L

    rng = np.random.default_rng(hidden + len(seqs))
    shapes = {"qkv": ((H + 2 * K) * D, hidden), "o": (hidden, H * D), "gate_up": (2 * ffn, hidden), "down": (hidden, ffn)}
    weights = {}
    for name, (n, k) in shapes.items():
        w = rng.standard_normal((n, k)).astype(np.float32) / np.sqrt(k).astype(np.float32)
        scale = R.scale_of_peak(np.abs(w).max(1))
        weights[name] = (R.codes_of(w, scale[:, None]), scale)
    gammas = [bf16(1 + 0.1 * rng.standard_normal(hidden)) for _ in range(2)]
    b = R.Batch(7, seqs, H, K, D, 32)
    up = hip.DeviceBuffer.from_numpy
    (cos, sin), (cos_v, sin_v) = R.table_rows(rng, b.longest + 2, D, False, R.F32)
    layer = L.DecoderLayerI8(*[L.Weights(*weights[n]) for n in shapes], *[up(W.to_storage(g, BF16)[0]) for g in gammas], up(cos), up(sin), b.longest + 2, H, K, D)
    layer.prepare(b.tokens, len(seqs), b.blocks, 32, b.longest)
    ref = Reference(weights, gammas, H, K, D)
    dev = R.Device(hip, b)
    st, x = W.to_storage(rng.standard_normal((b.tokens, hidden)).astype(np.float32), BF16)
    dx, out = up(st), hip.DeviceBuffer(b.tokens * hidden * 2)
    stream = hip.Stream()
    layer.step(dx, out, *dev.caches, *dev.scales, dev.index, stream)
    stream.synchronize()
    got = W.bf16_bits_to_f32(out.download(np.uint16, (b.tokens, hidden)))
    want = ref.step(b, x, cos_v, sin_v)
    error = np.linalg.norm(got - want) / np.linalg.norm(want)
    print("[int8 layer] relative 2-norm", error)
    assert error <= 1e-2
    codes, scales = dev.cache_state()
    held, wanted = (c * s[..., None, None].astype(np.float64) for c, s in ((codes, scales), (b.codes, b.scales)))
    assert np.linalg.norm(held - wanted) / np.linalg.norm(wanted) <= 1e-2
    stream.close()
