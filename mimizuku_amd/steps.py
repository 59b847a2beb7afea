"""Parts of a decoder step of one's own: products with 4-bit weights, attention over an encoder's output of any length,
the next token (mz_w4_*, mz_cross_attention, mz_sample).

    w = W4(ctx, n, k, group=64)
    w.pack(src)                                       # f16 [n][k]
    w.linear(x, out, m, epilogue=L.EPI_GELU_F16, bias=b)
    cross_attention(ctx, q, out, k, v, rows, tokens, heads, positions, slots, k_strides=..., len=lens)
    sample(ctx, logits, rows, vocab, u, tokens, temperature=0.8, top_p=0.95)

Arrays are device addresses (ints; model.Context allocates and copies them), work is enqueued on the context's stream.
The reference's weights are fp16, its cross-attention takes 1500 positions (kernels/whisper.cu:355-449) and its choice is
greedy (kernels/whisper.cu:451-493).
"""
from __future__ import annotations

import ctypes as C

from . import _lib as L
from ._lib import check
from .model import Context

HD = 64


def w4_bytes(n: int, k: int, group: int) -> int:
    """Bytes of device memory that n x k weights take."""
    b = C.c_size_t()
    check(L.lib().mz_w4_place(n, k, group, 0, None, C.byref(b)))
    return b.value


def cross_bytes(ctx: Context, a: L.CrossArgs) -> int:
    """Bytes of workspace that mz_cross_attention needs for these arguments."""
    n = C.c_size_t()
    check(L.lib().mz_cross_attention_bytes(ctx.h, C.byref(a), C.byref(n)))
    return n.value


def sample_bytes(ctx: Context, a: L.SampleArgs) -> int:
    """Bytes of workspace that mz_sample needs for these arguments: 0."""
    n = C.c_size_t()
    check(L.lib().mz_sample_bytes(ctx.h, C.byref(a), C.byref(n)))
    return n.value


class W4:
    """Weights [n][k] in 4 bits with a scale per `group` columns, in one device buffer: the context's, or w4_bytes bytes of
    the caller's at `at`. `w` is the struct that the C entry points take."""

    def __init__(self, ctx: Context, n: int, k: int, group: int = 64, at: int = 0):
        self.ctx, self.nbytes, self.w, self.base = ctx, w4_bytes(n, k, group), L.W4(), 0
        if not at:
            self.base = at = ctx.alloc(self.nbytes)
        check(L.lib().mz_w4_place(n, k, group, at, C.byref(self.w), None))

    def free(self):
        if self.base:
            self.ctx.free(self.base)
        self.base, self.w = 0, L.W4()

    def pack(self, src: int, ld: int = 0):
        """f16 weights [n][ld] at src into codes and scales (mz_w4_pack). ld 0: k."""
        check(L.lib().mz_w4_pack(self.ctx.h, C.byref(self.w), src, ld or self.w.k))

    def unpack(self, dst: int, ld: int = 0):
        """What the weights stand for, f16 [n][ld] at dst (mz_w4_unpack)."""
        check(L.lib().mz_w4_unpack(self.ctx.h, C.byref(self.w), dst, ld or self.w.k))

    def linear(self, x: int, out: int, m: int, epilogue: int = L.EPI_F16, bias: int = 0, ldx: int = 0, ldo: int = 0):
        """out = epilogue(x . weights^T + bias) for m rows f16 of x (mz_w4_linear). ldx 0: k, ldo 0: n."""
        a = L.W4LinearArgs(epilogue, m, x, ldx or self.w.k, bias, out, ldo or self.w.n)
        check(L.lib().mz_w4_linear(self.ctx.h, C.byref(self.w), C.byref(a)))


def cross_attention(ctx: Context, q: int, out: int, k: int, v: int, rows: int, tokens: int, heads: int, positions: int,
                    slots: int | None = None, kv_heads: int | None = None, k_strides=None, v_strides=None, q_strides=None,
                    out_strides=None, scale: float = 0.125, slot: int = 0, count: int = 0, first: int = 0, len: int = 0,
                    lse: int = 0, head_slot: int = 0, align: int = 0, align_heads: int = 0, align_cols: int = 0,
                    work: tuple[int, int] | None = None):
    """Attention of rows x tokens queries f16 over the keys and values f16 of `slots` (None: rows) sequences of `positions`
    (mz_cross_attention). k_strides: (slot, position, head) in elements, [slots][kv_heads][positions][64] if None;
    v_strides: as k_strides if None; q_strides, out_strides: (row, token, head), [rows][tokens][heads][64] if None. work: as
    of Kv8.attention."""
    kvh, slots = heads if kv_heads is None else kv_heads, rows if slots is None else slots
    dense, tiles = (tokens * heads * HD, heads * HD, HD), (kvh * positions * HD, HD, positions * HD)
    ks = k_strides or tiles
    a = L.CrossArgs(q, out, *(q_strides or dense), *(out_strides or dense), k, v, *ks, *(v_strides or ks), rows, tokens,
                    heads, kvh, slots, positions, scale, slot, count, first, len, lse, head_slot, align, align_heads,
                    align_cols)
    a.work, a.work_bytes = work or ctx.workspace(cross_bytes(ctx, a))
    check(L.lib().mz_cross_attention(ctx.h, C.byref(a)))


def sample(ctx: Context, logits: int, rows: int, vocab: int, u: int, tokens: int, dtype: int = L.DT_F32, ld: int = 0,
           mask: int = 0, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0,
           temperatures: int = 0, top_ks: int = 0, top_ps: int = 0, min_ps: int = 0, logp: int = 0, kept: int = 0,
           stride: int = 1, at: int = 0, at_add: int = 0, work: tuple[int, int] | None = None):
    """The next token of rows of logits from given random numbers u, 0 <= u < 1 (mz_sample). temperatures, top_ks, top_ps,
    min_ps: device arrays of a value per row, in place of the one for all. work: (address, bytes) of a workspace, which it does
    not read."""
    a = L.SampleArgs(dtype, rows, vocab, logits, ld or vocab, mask, temperature, top_p, min_p, top_k, temperatures, top_ps,
                     min_ps, top_ks, u, tokens, logp, kept, stride, at, at_add)
    a.work, a.work_bytes = work or (0, 0)
    check(L.lib().mz_sample(ctx.h, C.byref(a)))
