"""Plain implementations of the 8-bit operators for their tests: the position rotation and the append in fp32 with every
operation rounded by itself (which defines the stored codes to the bit), attention in fp64, and batches to run them on.  numpy only."""
import numpy as np

from openvino_contrib_amd import workloads as W

F32, F16, BF16, U8, I8 = 0, 1, 2, 3, 4
one = np.float32(1)


def rotated(x, cos, sin, rotary, interleaved):
    """x [..., heads, size] fp32 with one table row per leading index; NaN rows of cos stand for "not rotated"."""
    x = np.array(x, np.float32)
    c, s = cos[..., None, :].astype(np.float32), sin[..., None, :].astype(np.float32)
    h = rotary // 2
    a, b = (x[..., 0:rotary:2].copy(), x[..., 1:rotary:2].copy()) if interleaved else (x[..., :h].copy(), x[..., h:rotary].copy())
    ca, cb = (c[..., :h], c[..., :h]) if interleaved else (c[..., :h], c[..., h:rotary])
    sa, sb = (s[..., :h], s[..., :h]) if interleaved else (s[..., :h], s[..., h:rotary])
    na, nb = a * ca - b * sa, b * cb + a * sb
    still = np.isnan(ca)
    na, nb = np.where(still, a, na), np.where(still, b, nb)
    if interleaved:
        x[..., 0:rotary:2], x[..., 1:rotary:2] = na, nb
    else:
        x[..., :h], x[..., h:rotary] = na, nb
    return x


def scale_of_peak(peak):
    s = (np.asarray(peak, np.float32) * (one / np.float32(127))).astype(np.float32)
    return np.where(s < np.float32(1e-30), np.float32(0), s)


def codes_of(x, scale):
    scale = np.asarray(scale, np.float32)
    inverse = np.where(scale > 0, one / np.where(scale > 0, scale, one), np.float32(0)).astype(np.float32)
    return np.clip(np.rint(x.astype(np.float32) * inverse), -127, 127).astype(np.int8)


class Batch:
    """Sequences [(cached tokens, new tokens)], their block table (a permutation of the pool) and an i8 cache of N(0, 1) rows."""

    def __init__(self, seed, seqs, Hq, Hkv, D, bs, spare=3, std=1.0, lead=0):
        self.rng = np.random.default_rng(seed)
        self.seqs, self.Hq, self.Hkv, self.D, self.bs = seqs, Hq, Hkv, D, bs
        self.past = np.array([p for p, _ in seqs], np.int32)
        new = [n for _, n in seqs]
        self.begins = (lead + np.concatenate([[0], np.cumsum(new)])).astype(np.int32)
        blocks = [-(-(p + n) // bs) for p, n in seqs]
        self.table_begins = np.concatenate([[0], np.cumsum(blocks)]).astype(np.int32)
        self.blocks = int(self.table_begins[-1]) + spare
        self.table = self.rng.permutation(self.blocks)[:self.table_begins[-1]].astype(np.int32)
        self.tokens = int(self.begins[-1])
        self.longest = max([p + n for p, n in seqs] + [1])
        x = (self.rng.standard_normal((2, self.blocks, Hkv, bs, D)) * std).astype(np.float32)
        self.scales = scale_of_peak(np.abs(x).max((3, 4)))  # [K or V, block, head]
        self.codes = codes_of(x, self.scales[..., None, None])

    def slot(self, s, position):
        """(block, row) of a position, or None where the table names no block of the pool."""
        entry = position // self.bs
        if entry >= self.table_begins[s + 1] - self.table_begins[s]:
            return None
        block = int(self.table[self.table_begins[s] + entry])
        return (block, position % self.bs) if 0 <= block < self.blocks else None

    def append(self, k, v):
        """Rows [tokens, Hkv, D] fp32 into the i8 cache, a block at a time, as the operator defines it."""
        for s, (past, new) in enumerate(self.seqs):
            for entry in range(past // self.bs, -(-(past + new) // self.bs) if new else 0):
                where = self.slot(s, entry * self.bs)
                if where is None:
                    continue
                block = where[0]
                r0, r1 = max(0, past - entry * self.bs), min(self.bs, past + new - entry * self.bs)
                t0 = self.begins[s] + entry * self.bs + r0 - past
                for which, x in enumerate((k, v)):
                    rows = x[t0:t0 + r1 - r0].transpose(1, 0, 2)  # [Hkv, rows, D]
                    before = np.where(r0 == 0, np.float32(0), self.scales[which, block])
                    scale = np.maximum(before, scale_of_peak(np.abs(rows).max((1, 2))))
                    ratio = np.where(scale > before, before / np.where(scale > 0, scale, one), one).astype(np.float32)
                    held = self.codes[which, block, :, :r0]
                    self.codes[which, block, :, :r0] = np.rint(held.astype(np.float32) * ratio[:, None, None]).astype(np.int8)
                    self.codes[which, block, :, r0:r1] = codes_of(rows, scale[:, None, None])
                    self.scales[which, block] = scale

    def attention(self, q, window=0, scale=None):
        """q [tokens, Hq, D] -> [tokens, Hq, D] in fp64; rows of tokens outside every sequence are NaN."""
        out = np.full((self.tokens, self.Hq, self.D), np.nan)
        G, scale = self.Hq // self.Hkv, scale or self.D ** -0.5
        for s, (past, new) in enumerate(self.seqs):
            if not new:
                continue
            entries = self.table[self.table_begins[s]:self.table_begins[s + 1]]
            there = (entries >= 0) & (entries < self.blocks)
            safe = np.where(there, entries, 0)
            length = min(past + new, len(entries) * self.bs)
            kv = self.codes[:, safe].astype(np.float64) * self.scales[:, safe].astype(np.float64)[..., None, None]
            kv = kv.transpose(0, 2, 1, 3, 4).reshape(2, self.Hkv, -1, self.D)[:, :, :length]
            exists = np.repeat(there, self.bs)[:length]
            for i in range(new):
                p = past + i
                j = np.arange(length)
                seen = exists & (j <= p) & (j > p - window if window > 0 else True)
                t = self.begins[s] + i
                if not seen.any():
                    out[t] = 0
                    continue
                for h in range(self.Hkv):
                    sc = kv[0, h][seen] @ q[t, h * G:(h + 1) * G].astype(np.float64).T * scale
                    w = np.exp(sc - sc.max(0))
                    out[t, h * G:(h + 1) * G] = (w / w.sum(0)).T @ kv[1, h][seen]
        return out


class Device:
    """A batch's index arrays, caches and scales on the device."""

    def __init__(self, hip, b):
        self.hip, self.b = hip, b
        up = hip.DeviceBuffer.from_numpy
        self.index = [up(a) if a.size else hip.DeviceBuffer(4) for a in (b.past, b.begins, b.table, b.table_begins)]
        self.caches = [up(b.codes[i]) for i in range(2)]
        self.scales = [up(b.scales[i]) for i in range(2)]

    def cache_state(self):
        shape = self.b.codes.shape[1:]
        return (np.stack([c.download(np.int8, shape) for c in self.caches]),
                np.stack([s.download(np.float32, shape[:2]) for s in self.scales]))


def table_rows(rng, rows, rotary, interleaved, dtype):
    """(cos, sin) tables as stored, and their fp32 values."""
    cols = rotary // 2 if interleaved else rotary
    angle = rng.uniform(-np.pi, np.pi, (rows, cols))
    pairs = [W.to_storage(f(angle).astype(np.float32), dtype) for f in (np.cos, np.sin)]
    return [p[0] for p in pairs], [p[1] for p in pairs]
