"""The operators of a decoder layer that runs in 8 bits, as cases that can be timed and compared:

* append: new keys and values rotated by their positions and appended to a paged cache, the queries rotated beside them
  (`capi.rope_append`), into 16-bit caches and into the 8-bit cache with one scale per block and kv head;
* attend: paged attention over that 8-bit cache (`capi.paged_attention_i8`);
* product: a projection with 8-bit weights, a scale per output channel, on activations of 8 bits with a scale per token
  (`ops_capi.matmul_i8`), which come as they are or are quantised on the way in (`ops_capi.quantize_rows`), behind an RMS
  norm or a GLU where the layer has one there.

`own` false: the plain forms, torch operations in fp32.  `own` true: the framework's entry points.
"""
import ctypes
import math
import random

import torch

own = False

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16), "i8": (4, torch.int8)}
TINY = 1e-30  # a scale below this stands for a block of zeros

# ----------------------------------------------------------------------------------- the cases
# A batch: `prompts` sequences of chunk_lo..chunk_hi new tokens behind past_lo..past_hi cached ones, then `decodes`
# sequences of one new token whose contexts are uniform in ctx_lo..ctx_hi; the lengths are drawn from `lengths`.
BATCH = dict(heads=32, kv_heads=8, size=128, block=32, lengths=1, prompts=0, chunk_lo=0, chunk_hi=0, past_lo=0, past_hi=0,
             decodes=0, ctx_lo=0, ctx_hi=0)
# q, k and v side by side in one buffer, as a joint projection leaves them (packed) or apart; table: fp32 angles
APPEND = dict(BATCH, path="append", type="bf16", cache="i8", rotary=128, interleaved=False, packed=True)
ATTEND = dict(BATCH, path="attend", type="bf16", window=0)
# C[m, n] of `out`; source: "codes" (8-bit activations in hand) or 16-bit ones, quantised plain, behind a norm or a GLU
PRODUCT = dict(path="product", m=1, n=4096, k=4096, out="bf16", source="plain", bias=False, residual=False)


def listed():
    return [
        # the next token of a single conversation: all latency
        dict(APPEND, name="append_one", decodes=1, ctx_lo=778, ctx_hi=778),
        # a decode step of a serving batch, a row here and there all over the cache
        dict(APPEND, name="append_decode", heads=64, decodes=128, ctx_lo=256, ctx_hi=4096, lengths=2),
        # chunks of prompts behind cached tokens, most of them ending inside a block
        dict(APPEND, name="append_chunks", heads=64, prompts=8, chunk_lo=400, chunk_hi=512, past_hi=4096, lengths=5),
        # new prompts of a model with narrow heads, pairs of neighbours rotated, into a 16-bit cache of small blocks
        dict(APPEND, name="append_prompts_f16", type="f16", cache="f16", size=64, rotary=64, interleaved=True, packed=False, block=16,
             prompts=6, chunk_lo=100, chunk_hi=3000, lengths=6),
        # attention of that single conversation
        dict(ATTEND, name="attend_one", decodes=1, ctx_lo=778, ctx_hi=778),
        # a decode step of a serving batch
        dict(ATTEND, name="attend_decode", type="f16", decodes=64, ctx_lo=512, ctx_hi=8192, lengths=1003),
        # continuous batching: chunks of prompts beside decoding sequences, with a sliding window
        dict(ATTEND, name="attend_mixed", heads=64, window=4096, prompts=8, chunk_lo=512, chunk_hi=512, past_hi=4096,
             decodes=120, ctx_lo=256, ctx_hi=8192, lengths=1005),
        # new prompts of uneven length
        dict(ATTEND, name="attend_prompts", prompts=6, chunk_lo=100, chunk_hi=3000, lengths=6),
        # a projection of a single token
        dict(PRODUCT, name="product_one", source="norm"),
        # gate and up of a serving batch, behind the norm
        dict(PRODUCT, name="product_decode", m=64, n=28672, source="norm"),
        # the way down of a few prompts, from the two halves that the GLU joins, onto the residual
        dict(PRODUCT, name="product_down", m=1111, k=14336, source="glu", residual=True),
        # q, k and v of many tokens, activations in codes already
        dict(PRODUCT, name="product_prompt", m=8192, n=6144, source="codes", bias=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    """Seconds, roughly: what keeps a drawn case below the largest listed one of its path."""
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 4e14


def draw(rng):
    path = rng.choice(("append", "attend", "product"))
    largest = max(_cost(c) for c in listed() if c["path"] == path)
    while True:
        if path == "product":
            source = rng.choice(("codes", "plain", "norm", "glu"))
            odd = rng.random() < 0.3
            case = dict(PRODUCT, m=_log_int(rng, 1, 8192), n=_log_int(rng, 64, 28672), k=_log_int(rng, 64, 16384), source=source,
                        out=rng.choice(("f16", "bf16", "bf16", "f32") if source == "codes" else ("f16", "bf16")), bias=rng.random() < 0.5,
                        residual=rng.random() < 0.5)
            if not odd:
                case.update(n=-(-case["n"] // 64) * 64, k=-(-case["k"] // 64) * 64)
        else:
            heads, kv = rng.choice(((32, 8), (32, 8), (64, 8), (16, 4), (16, 16), (32, 1)))
            size = rng.choice((64, 128, 128, 128) if path == "attend" else (64, 80, 128, 128, 256))
            case = dict(APPEND if path == "append" else ATTEND, heads=heads, kv_heads=kv, size=size, block=rng.choice((16, 32, 32, 64)),
                        type=rng.choice(("f16", "bf16")), lengths=rng.randrange(1 << 30))
            if path == "append":
                case.update(cache=rng.choice(("i8", "i8", case["type"])), rotary=rng.choice((size, size, size // 2)),
                            interleaved=rng.random() < 0.3, packed=rng.random() < 0.5)
            else:
                case["window"] = rng.choice((0, 0, 4096, _log_int(rng, 1, 4096)))
            prompts = rng.random() < 0.5
            if prompts:
                case["prompts"] = _log_int(rng, 1, 8)
                case["chunk_hi"] = _log_int(rng, 2, 3000)
                case["chunk_lo"] = max(2, int(case["chunk_hi"] * rng.uniform(0.1, 1.0)))
                case["past_hi"] = rng.choice((0, 0, _log_int(rng, 1, 4096)))
            if not prompts or rng.random() < 0.4:
                case["decodes"] = _log_int(rng, 1, 128)
                case["ctx_hi"] = _log_int(rng, 1, 8192)
                case["ctx_lo"] = max(1, int(case["ctx_hi"] * rng.uniform(0.05, 1.0)))
        if _cost(case) <= largest:
            return case


def _sequences(case):
    """[(cached tokens, new tokens)]: the prompts, then the decoding sequences."""
    r = random.Random(case["lengths"])
    seqs = [(r.randint(case["past_lo"], case["past_hi"]), r.randint(case["chunk_lo"], case["chunk_hi"])) for _ in range(case["prompts"])]
    return seqs + [(r.randint(case["ctx_lo"], case["ctx_hi"]) - 1, 1) for _ in range(case["decodes"])]


# --------------------------------------------------------------------------------------- work
def work(case):
    """What a pass cannot do without: every input once, every output once, two operations per multiply-add."""
    if case["path"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        e = TYPES[case["out"]][1].itemsize
        taken = m * k + 4 * m if case["source"] == "codes" else 2 * m * k * (2 if case["source"] == "glu" else 1)
        return {"bytes": taken + n * k + 4 * n + e * (m * n * (2 if case["residual"] else 1) + (n if case["bias"] else 0)), "flops": 2 * m * n * k}
    heads, kv, size, e = case["heads"], case["kv_heads"], case["size"], TYPES[case["type"]][1].itemsize
    seqs = _sequences(case)
    tokens = sum(n for _, n in seqs)
    if case["path"] == "append":
        row = size * TYPES[case["cache"]][1].itemsize
        read = e * tokens * (heads + 2 * kv) * size + 8 * tokens * case["rotary"] // (2 if case["interleaved"] else 1)
        scales = 8 * kv * sum(-(-(p + n) // case["block"]) - p // case["block"] for p, n in seqs) if case["cache"] == "i8" else 0
        return {"bytes": read + e * tokens * heads * size + 2 * tokens * kv * row + scales, "flops": 3 * tokens * (heads + kv) * case["rotary"]}
    window, keys, pairs = case["window"], 0, 0
    for past, new in seqs:
        first = max(0, past - window + 1) if window else 0  # of the positions that some token attends
        keys += past + new - first
        full = max(0, min(new, window - past)) if window else new  # tokens that see all before them
        pairs += full * past + full * (full + 1) // 2 + (new - full) * window
    return {"bytes": int(2 * kv * keys * (size + 4 / case["block"]) + 2 * e * tokens * heads * size), "flops": 4 * size * heads * pairs}


# ------------------------------------------------------------------------------------ prepare
class Buffer:
    """A torch tensor as the bindings take device memory."""

    def __init__(self, tensor, offset=0):
        self.tensor, self.ptr, self.nbytes = tensor, ctypes.c_void_p(tensor.data_ptr() + offset), tensor.numel() * tensor.element_size()


def _normal(gen, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * std).to(dtype)


def _scale_of(peak):
    s = peak / 127.0
    return torch.where(s < TINY, torch.zeros_like(s), s)


def _codes(x, scale):
    """rint(x / scale) as the product with the reciprocal, zeros where the scale is zero."""
    inverse = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    return torch.clamp(torch.round(x * inverse), -127, 127)


def _cache(gen, blocks, case):
    """(cache, scales or None): what earlier tokens left."""
    shape, kind = (blocks, case["kv_heads"], case["block"], case["size"]), case.get("cache", "i8")
    out = torch.empty(shape, device="cuda", dtype=TYPES[kind][1])
    scales = torch.empty(shape[:2], device="cuda", dtype=torch.float32) if kind == "i8" else None
    step = max(1, (1 << 26) // (shape[1] * shape[2] * shape[3]))
    for b in range(0, blocks, step):
        x = _normal(gen, (min(step, blocks - b),) + shape[1:], torch.float32)
        if kind == "i8":
            scales[b:b + step] = _scale_of(x.abs().amax((2, 3)))
            x = _codes(x, scales[b:b + step, :, None, None])
        out[b:b + step] = x.to(out.dtype)
    return out, scales


def _batch(case, gen):
    """The batch on the device: index arrays and caches, blocks scattered over the pool; and its lengths on the host."""
    seqs = _sequences(case)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    begins, table_begins = [0], [0]
    for past, new in seqs:
        begins.append(begins[-1] + new)
        table_begins.append(table_begins[-1] + -(-(past + new) // case["block"]))
    s = dict(seqs=seqs, tokens=begins[-1], blocks=table_begins[-1] + 3, past=i32([p for p, _ in seqs]), begins=i32(begins),
             table_begins=i32(table_begins), longest=max(p + n for p, n in seqs))
    s["table"] = torch.randperm(s["blocks"], generator=gen, device="cuda")[:table_begins[-1]].to(torch.int32)
    s["keys"], s["key_scales"] = _cache(gen, s["blocks"], case)
    s["values"], s["value_scales"] = _cache(gen, s["blocks"], case)
    return s


def _prepare_append(case, gen):
    s = _batch(case, gen)
    code, dtype = TYPES[case["type"]]
    T, H, K, D, R = s["tokens"], case["heads"], case["kv_heads"], case["size"], case["rotary"]
    widths = (H * D, K * D, K * D)
    if case["packed"]:
        s["qkv"] = _normal(gen, (T, sum(widths)), dtype)
        s["q"], s["k"], s["v"] = s["qkv"].split(widths, 1)
    else:
        s["q"], s["k"], s["v"] = (_normal(gen, (T, w), dtype) for w in widths)
    angle = torch.arange(s["longest"], device="cuda", dtype=torch.float64)[:, None] * (
        10000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R))[None, :]
    if not case["interleaved"]:
        angle = torch.cat([angle, angle], 1)
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    s["q_out"] = torch.empty((T, H * D), device="cuda", dtype=dtype)
    if own:
        from openvino_contrib_amd import capi
        s["desc"] = capi.PaDesc(code, code, TYPES[case["cache"]][0], code, H, K, D, case["block"], s["blocks"], T, len(s["seqs"]), s["longest"],
                                0, 0.0, 0, 0, None, None)
        s["rope"] = capi.RopeAppendDesc(table_dtype=0, rotary_ndims=R, interleaved=int(case["interleaved"]), table_rows=s["longest"],
                                        table_row_stride=s["cos"].shape[1], q_token_stride=s["q"].stride(0), k_token_stride=s["k"].stride(0),
                                        v_token_stride=s["v"].stride(0), q_out_token_stride=H * D)
        s["positions"] = None  # the tokens' places in the cache
        s["args"] = [Buffer(s[n]) if s[n] is not None else None for n in ("q", "k", "v", "cos", "sin", "positions", "q_out", "keys", "values",
                     "key_scales", "value_scales", "past", "begins", "table", "table_begins")]
    return s


def _prepare_attend(case, gen):
    s = _batch(case, gen)
    code, dtype = TYPES[case["type"]]
    T, H, K, D = s["tokens"], case["heads"], case["kv_heads"], case["size"]
    s["q"] = _normal(gen, (T, H * D), dtype)
    s["out"] = torch.empty_like(s["q"])
    if own:
        from openvino_contrib_amd import capi
        s["desc"] = capi.PaDesc(code, code, TYPES["i8"][0], code, H, K, D, case["block"], s["blocks"], T, len(s["seqs"]), s["longest"],
                                case["window"], 0.0, capi.PA_SKIP_CACHE_WRITE, 0, None, None)
        s["workspace"] = torch.empty(max(16, capi.paged_attention_workspace_size(s["desc"])), device="cuda", dtype=torch.uint8)
        s["args"] = [Buffer(s["q"]), None, None] + [Buffer(s[n]) for n in ("keys", "values", "key_scales", "value_scales", "past", "begins",
                                                                        "table", "table_begins", "out", "workspace")]
    return s


def _prepare_product(case, gen):
    m, n, k, out = case["m"], case["n"], case["k"], TYPES[case["out"]]
    s = {"weight": torch.randint(-127, 128, (n, k), generator=gen, device="cuda", dtype=torch.int8),
         "weight_scales": (0.5 + torch.rand(n, generator=gen, device="cuda")) / (73.0 * k ** 0.5)}
    act = out if out[0] else TYPES["f16"]  # the activations' type: that of the result
    if case["source"] == "codes":
        s["codes"] = torch.randint(-127, 128, (m, k), generator=gen, device="cuda", dtype=torch.int8)
        s["scales"] = (0.5 + torch.rand(m, generator=gen, device="cuda")) / 64.0
    else:
        s["x"] = _normal(gen, (m, 2 * k if case["source"] == "glu" else k), act[1])
    if case["source"] == "norm":
        s["gamma"] = _normal(gen, (k,), act[1], 0.1) + 1.0
    if case["bias"]:
        s["bias"] = _normal(gen, (n,), out[1])
    if case["residual"]:
        s["residual"] = _normal(gen, (m, n), out[1])
    s["out"] = torch.empty((m, n), device="cuda", dtype=out[1])
    if own:
        from openvino_contrib_amd import ops_capi
        s["desc"] = ops_capi.MatmulI8Desc(c_dtype=out[0], m=m, n=n, k=k, lda=k, ldb=k, ldc=n)
        s["workspace"] = torch.empty(max(16, ops_capi.matmul_i8_workspace_size(s["desc"])), device="cuda", dtype=torch.uint8)
        if case["source"] != "codes":
            s["codes"] = torch.empty((m, k), device="cuda", dtype=torch.int8)
            s["scales"] = torch.empty((m,), device="cuda", dtype=torch.float32)
            how = {"plain": ops_capi.QUANTIZE_PLAIN, "norm": ops_capi.QUANTIZE_RMS_NORM, "glu": ops_capi.QUANTIZE_GLU}[case["source"]]
            s["quantize"] = ops_capi.QuantizeDesc(source=how, x_dtype=act[0], gamma_dtype=act[0], glu_activation=ops_capi.GLU_SWISH,
                                                  glu_gate_first=1, eps=1e-5, rows=m, width=k, x_row_stride=s["x"].shape[1])
            s["quantize_args"] = [Buffer(s["x"]), Buffer(s["gamma"]) if "gamma" in s else None, Buffer(s["codes"]), Buffer(s["scales"])]
        s["args"] = [Buffer(s[n]) if n in s else None for n in ("codes", "scales", "weight", "weight_scales", "bias", "residual", "out", "workspace")]
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"append": _prepare_append, "attend": _prepare_attend, "product": _prepare_product}[case["path"]](case, gen)
    return dict(s, case=case)


# ------------------------------------------------------------------------------------ the plain forms
def _slots(s, case):
    """For each new token: its sequence, position and cache block."""
    begins, past, table_begins = s["begins"].long(), s["past"].long(), s["table_begins"].long()
    token = torch.arange(s["tokens"], device="cuda")
    seq = torch.searchsorted(begins, token, right=True) - 1
    position = past[seq] + token - begins[seq]
    return seq, position, s["table"].long()[table_begins[seq] + position // case["block"]]


def _rotated(x, cos, sin, case):
    """x [T, heads, size] in fp32, the first `rotary` columns turned by the angles of the rows cos, sin [T, columns]."""
    r, cos, sin = case["rotary"], cos[:, None], sin[:, None]
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        h = r // 2
        a, b = x[..., :h], x[..., h:r]
        turned = torch.cat([a * cos[..., :h] - b * sin[..., :h], b * cos[..., h:] + a * sin[..., h:]], -1)
    return torch.cat([turned, x[..., r:]], -1)


def _append_i8(s, case, x, cache, scales, seq, position, block):
    """Rows x [T, kv heads, size] into an 8-bit cache: a block's scale starts with its first row and grows with its rows."""
    size, row = case["block"], position % case["block"]
    peak = torch.zeros_like(scales).index_reduce_(0, block, x.abs().amax(-1), "amax")
    fresh = torch.zeros(len(scales), device="cuda").index_add_(0, block, (row == 0).float()) > 0
    old = torch.where(fresh[:, None], torch.zeros_like(scales), scales)
    grown = torch.maximum(old, _scale_of(peak))
    touched = torch.zeros(len(scales), dtype=torch.bool, device="cuda").index_fill_(0, block, True)
    # of the blocks that held rows before, a sequence's first is the only one
    past, first = s["past"].long(), s["table_begins"].long()[:-1]
    part = s["table"].long()[first + past // size]
    ratio = torch.where(old[part] < grown[part], old[part] / grown[part], torch.ones_like(grown[part]))
    before = torch.arange(size, device="cuda") < (past % size)[:, None]
    held = torch.where(before[:, None, :, None], torch.round(cache[part].float() * ratio[:, :, None, None]), cache[part].float())
    cache[part] = held.to(torch.int8)
    scales.copy_(torch.where(touched[:, None], grown, scales))
    cache[block, :, row] = _codes(x, grown[block][:, :, None]).to(torch.int8)


def _plain_append(s, case):
    H, K, D, T = case["heads"], case["kv_heads"], case["size"], s["tokens"]
    seq, position, block = _slots(s, case)
    cos, sin = s["cos"][position], s["sin"][position]
    q = _rotated(s["q"].reshape(T, H, D).float(), cos, sin, case)
    k = _rotated(s["k"].reshape(T, K, D).float(), cos, sin, case)
    v = s["v"].reshape(T, K, D).float()
    s["q_out"].copy_(q.reshape(T, H * D))
    if case["cache"] == "i8":
        _append_i8(s, case, k, s["keys"], s["key_scales"], seq, position, block)
        _append_i8(s, case, v, s["values"], s["value_scales"], seq, position, block)
    else:
        s["keys"][block, :, position % case["block"]] = k.to(s["keys"].dtype)
        s["values"][block, :, position % case["block"]] = v.to(s["values"].dtype)


def _held(cache, scales, blocks):
    """Blocks [S, n] of an 8-bit cache as fp32 [S * kv heads, n * block, size]."""
    x = cache[blocks].float().mul_(scales[blocks][..., None, None])
    S, n, K, B, D = x.shape
    return x.transpose(1, 2).reshape(S * K, n * B, D)


def _plain_part(s, case, first, last):
    """Sequences first..last of the batch, padded to the longest of them."""
    if first == last:
        return
    seqs = s["seqs"][first:last]
    S, H, K, D, B = len(seqs), case["heads"], case["kv_heads"], case["size"], case["block"]
    new, n_blocks = max(n for _, n in seqs), max(-(-(p + n) // B) for p, n in seqs)
    past, begins, table_begins = s["past"].long()[first:last], s["begins"].long()[first:last + 1], s["table_begins"].long()[first:last + 1]
    step = torch.arange(new, device="cuda")
    valid = step[None] < (begins[1:] - begins[:-1])[:, None]
    token = torch.where(valid, begins[:-1, None] + step[None], begins[:-1, None])
    entry = torch.arange(n_blocks, device="cuda")
    entry = torch.minimum(table_begins[:-1, None] + entry[None], table_begins[1:, None] - 1)
    blocks = s["table"].long()[entry]
    q = s["q"].reshape(-1, K, H // K, D)[token].float().mul_(D ** -0.5)  # [S, new, K, G, D]
    q = q.permute(0, 2, 3, 1, 4).reshape(S * K, H // K * new, D)
    scores = torch.bmm(q, _held(s["keys"], s["key_scales"], blocks).transpose(1, 2)).view(S, K, H // K, new, n_blocks * B)
    position, key = past[:, None] + step[None], torch.arange(n_blocks * B, device="cuda")
    hidden = key[None, None] > position[..., None]
    if case["window"]:
        hidden |= key[None, None] <= position[..., None] - case["window"]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    scores.div_(scores.sum(-1, keepdim=True))
    out = torch.bmm(scores.view(S * K, H // K * new, n_blocks * B), _held(s["values"], s["value_scales"], blocks))
    out = out.view(S, K, H // K, new, D).permute(0, 3, 1, 2, 4).reshape(S, new, H * D)
    s["out"][begins[0]:begins[-1]] = out[valid].to(s["out"].dtype)


def _plain_product(s, case):
    k = case["k"]
    if case["source"] == "codes":
        codes, scales = s["codes"].float(), s["scales"][:, None]
    else:
        y = s["x"].float()
        if case["source"] == "norm":
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + 1e-5) * s["gamma"].float()
        elif case["source"] == "glu":
            y = y[:, :k] / (1.0 + torch.exp(-y[:, :k])) * y[:, k:]
        scales = _scale_of(y.abs().amax(-1, keepdim=True))
        codes = _codes(y, scales)
    c = codes @ s["weight"].float().t()
    c = c * scales * s["weight_scales"]
    if case["bias"]:
        c = c + s["bias"].float()
    if case["residual"]:
        c = c + s["residual"].float()
    s["out"].copy_(c)


# ---------------------------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    if case["path"] == "append":
        if own:
            from openvino_contrib_amd import capi
            capi.rope_append(state["desc"], state["rope"], *state["args"])
        else:
            _plain_append(state, case)
        return {n: state[n] for n in ("q_out", "keys", "values", "key_scales", "value_scales") if state[n] is not None}
    if case["path"] == "attend":
        if own:
            from openvino_contrib_amd import capi
            capi.paged_attention_i8(state["desc"], *state["args"])
        else:
            _plain_part(state, case, 0, case["prompts"])
            _plain_part(state, case, case["prompts"], len(state["seqs"]))
        return state["out"]
    if own:
        from openvino_contrib_amd import ops_capi
        if case["source"] != "codes":
            ops_capi.quantize_rows(state["quantize"], *state["quantize_args"])
        ops_capi.matmul_i8(state["desc"], *state["args"])
    else:
        _plain_product(state, case)
    return state["out"]


# ---------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The operators' definitions in 64 bits, a sequence or a slice of rows at a time."""
    s = prepare(case, seed)
    if case["path"] == "product":
        return _exact_product(s, case)
    begins = s["begins"].tolist()
    first_entry = s["table_begins"].tolist()
    B, D, K, G = case["block"], case["size"], case["kv_heads"], case["heads"] // case["kv_heads"]
    if case["path"] == "attend":
        if work(case)["flops"] > 3e12:
            return None
        out = torch.empty(s["out"].shape, device="cuda", dtype=torch.float64)
        for i, (past, new) in enumerate(s["seqs"]):
            blocks = s["table"][first_entry[i]:first_entry[i + 1]].long()
            for h in range(K):
                k = (s["keys"][blocks, h].double() * s["key_scales"][blocks, h].double()[:, None, None]).reshape(-1, D)[:past + new]
                v = (s["values"][blocks, h].double() * s["value_scales"][blocks, h].double()[:, None, None]).reshape(-1, D)[:past + new]
                q = s["q"][begins[i]:begins[i + 1]].reshape(new, K, G, D)[:, h].double()
                at, j = past + torch.arange(new, device="cuda")[:, None], torch.arange(past + new, device="cuda")[None]
                seen = (j <= at) & (j > at - case["window"]) if case["window"] else j <= at
                for g in range(G):
                    p = torch.softmax((q[:, g] @ k.t() / math.sqrt(D)).masked_fill(~seen, -math.inf), -1)
                    out[begins[i]:begins[i + 1]].view(new, K, G, D)[:, h, g] = p @ v
        return out
    R, h = case["rotary"], case["rotary"] // 2

    def turned(x, n, past, new):
        x = x.reshape(new, n, D).double().clone()
        c, t = s["cos"][past:past + new].double()[:, None], s["sin"][past:past + new].double()[:, None]
        a, b = (x[..., 0:R:2].clone(), x[..., 1:R:2].clone()) if case["interleaved"] else (x[..., :h].clone(), x[..., h:R].clone())
        if case["interleaved"]:
            x[..., 0:R:2], x[..., 1:R:2] = a * c - b * t, b * c + a * t
        else:
            x[..., :h], x[..., h:R] = a * c[..., :h] - b * t[..., :h], b * c[..., h:] + a * t[..., h:]
        return x

    q_out = torch.empty(s["q_out"].shape, device="cuda", dtype=torch.float64)
    eight = case["cache"] == "i8"
    found = {"keys": s["key_scales"] if eight else s["keys"], "values": s["value_scales"] if eight else s["values"]}
    found = {n: x.double() for n, x in found.items()}
    for i, (past, new) in enumerate(s["seqs"]):
        rows = slice(begins[i], begins[i + 1])
        q_out[rows] = turned(s["q"][rows], K * G, past, new).reshape(new, -1)
        new_rows = {"keys": turned(s["k"][rows], K, past, new), "values": s["v"][rows].reshape(new, K, D).double()}
        blocks = s["table"][first_entry[i]:first_entry[i + 1]].long()
        for name, x in new_rows.items():
            if not eight:
                at = past + torch.arange(new, device="cuda")
                found[name][blocks[at // B], :, at % B] = x
                continue
            for b in range(past // B, (past + new - 1) // B + 1):
                peak = x[max(0, b * B - past):(b + 1) * B - past].abs().amax((0, 2)) / 127
                found[name][blocks[b]] = torch.maximum(peak, found[name][blocks[b]]) if b * B < past else peak
    if eight:
        return {"q_out": q_out, "keys": None, "values": None, "key_scales": found["keys"], "value_scales": found["values"]}
    return {"q_out": q_out, **found}


def _exact_product(s, case):
    m, k = case["m"], case["k"]
    if m * case["n"] * k > 4e11:
        return None
    out = torch.empty(s["out"].shape, device="cuda", dtype=torch.float64)
    w = s["weight"].double().t()
    for a in range(0, m, 1024):
        rows = slice(a, a + 1024)
        if case["source"] == "codes":
            c, scale = s["codes"][rows].double(), s["scales"][rows].double()
        else:
            y = s["x"][rows].double()
            if case["source"] == "norm":
                y = y / ((y ** 2).sum(1, keepdim=True) / k + 1e-5).sqrt() * s["gamma"].double()
            if case["source"] == "glu":
                y = y[:, :k] * torch.sigmoid(y[:, :k]) * y[:, k:]
            scale = y.abs().amax(1) / 127
            c = (y / scale[:, None]).round()
        out[rows] = (c @ w) * scale[:, None] * s["weight_scales"].double()
        if case["bias"]:
            out[rows] += s["bias"].double()
        if case["residual"]:
            out[rows] += s["residual"][rows].double()
    return out
