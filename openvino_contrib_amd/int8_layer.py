"""A decoder layer's step in 8 bits, out of the library's entry points: 8-bit weights and activations, a cache of 8-bit codes with a scale per
block and kv head, everything between the operators in bf16.  What `bench.py --workload int8` times, and an example of how the calls go
together:

    norm, quantised -> q | k | v product -> rotary embedding and append -> attention -> quantised -> o product + residual
    -> norm, quantised -> gate | up product -> GLU, quantised -> down product + residual

Ten calls on one stream, none of which allocates, copies to the host or waits, so the step can be recorded in a graph.
"""
import ctypes

from . import capi, ops_capi
from .capi import BF16, F32, I8


class Weights:
    """An 8-bit matrix [n, k] with a scale per row, as device buffers."""

    def __init__(self, codes, scales):
        self.n, self.k = codes.shape
        self.codes, self.scales = capi.DeviceBuffer.from_numpy(codes), capi.DeviceBuffer.from_numpy(scales)


class View:
    """Part of a device buffer, from a byte on."""

    def __init__(self, buffer, offset):
        self.ptr, self.nbytes = ctypes.c_void_p(buffer.ptr.value + offset), buffer.nbytes - offset


class DecoderLayerI8:
    """qkv, o, gate_up, down: Weights; gamma1, gamma2: bf16 device buffers; cos, sin: fp32 device tables [rows, head_dim]."""

    def __init__(self, qkv, o, gate_up, down, gamma1, gamma2, cos, sin, table_rows, heads, kv_heads, head_dim, eps=1e-5):
        self.qkv, self.o, self.gate_up, self.down, self.gamma1, self.gamma2 = qkv, o, gate_up, down, gamma1, gamma2
        self.cos, self.sin, self.table_rows, self.eps = cos, sin, table_rows, eps
        self.heads, self.kv_heads, self.head_dim, self.hidden, self.ffn = heads, kv_heads, head_dim, qkv.k, down.k

    def prepare(self, tokens, seqs, blocks, block_size, longest):
        """Buffers and descriptors for batches of this size."""
        H, K, D, T = self.heads, self.kv_heads, self.head_dim, tokens
        new = capi.DeviceBuffer
        self.tokens = T
        self.codes, self.scales = new(T * max(self.hidden, self.ffn, H * D)), new(4 * T)
        self.projected, self.q, self.attended, self.inner, self.gated = (new(2 * T * w) for w in (self.qkv.n, H * D, H * D, self.hidden, 2 * self.ffn))
        self.attention = capi.PaDesc(BF16, BF16, I8, BF16, H, K, D, block_size, blocks, T, seqs, longest, 0, 0.0, capi.PA_SKIP_CACHE_WRITE, 0)
        self.rope = capi.RopeAppendDesc(table_dtype=F32, rotary_ndims=D, table_rows=self.table_rows, table_row_stride=D, q_token_stride=self.qkv.n,
                                        k_token_stride=self.qkv.n, v_token_stride=self.qkv.n)
        need = max([capi.paged_attention_workspace_size(self.attention)] +
                   [ops_capi.matmul_i8_workspace_size(ops_capi.MatmulI8Desc(BF16, T, w.n, w.k)) for w in (self.qkv, self.o, self.gate_up, self.down)])
        self.workspace = new(max(16, need))

    def _product(self, weights, source, x, gamma, residual, out, stream):
        ops_capi.quantize_rows(ops_capi.QuantizeDesc(source, BF16, BF16, ops_capi.GLU_SWISH, 1, self.eps, self.tokens, weights.k, 0), x, gamma, self.codes,
                               self.scales, stream)
        ops_capi.matmul_i8(ops_capi.MatmulI8Desc(BF16, self.tokens, weights.n, weights.k), self.codes, self.scales, weights.codes, weights.scales, None,
                           residual, out, self.workspace, stream)

    def step(self, x, out, key_cache, value_cache, key_scales, value_scales, index, stream=None):
        """x, out: bf16 [tokens, hidden]; index: past_lens, subsequence_begins, block_indices, block_indices_begins."""
        caches = (key_cache, value_cache, key_scales, value_scales)
        plain, norm, glu = ops_capi.QUANTIZE_PLAIN, ops_capi.QUANTIZE_RMS_NORM, ops_capi.QUANTIZE_GLU
        self._product(self.qkv, norm, x, self.gamma1, None, self.projected, stream)
        k, v = (View(self.projected, 2 * w * self.head_dim) for w in (self.heads, self.heads + self.kv_heads))
        capi.rope_append(self.attention, self.rope, self.projected, k, v, self.cos, self.sin, None, self.q, *caches, *index, stream=stream)
        capi.paged_attention_i8(self.attention, self.q, None, None, *caches, *index, self.attended, self.workspace, stream)
        self._product(self.o, plain, self.attended, None, x, self.inner, stream)
        self._product(self.gate_up, norm, self.inner, self.gamma2, None, self.gated, stream)
        self._product(self.down, glu, self.gated, None, self.inner, out, stream)
