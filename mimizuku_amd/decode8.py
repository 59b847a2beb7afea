"""Decoding with key/value caches held in 8 bits, and the scores of what was decoded (mz_kv8_* and mz_token_scores).

    kv = Kv8(ctx, slots=32, heads=20, max_tokens=448, fmt="i8")
    kv.write(k, v, rows, tokens, pos=ctr, pos_stride=0)               # a step's keys and values at its position
    kv.attention(q, out, rows, tokens, heads, len=ctr, len_stride=0, len_add=1)
    token_scores(ctx, logits, rows, vocab, tokens=tok, logp=logp, entropy=h)

Arrays are device addresses (ints; model.Context allocates and copies them), work is enqueued on the context's stream.
The reference's caches are fp16 (src/model.rs:436-452) and its decoder keeps no probabilities.
"""
from __future__ import annotations

import ctypes as C

from . import _lib as L
from ._lib import MzError, check
from .model import Context

HD = 64
FORMATS = {"i8": L.KV8_I8, "e4m3": L.KV8_E4M3}


def attention_bytes(ctx: Context, kv: L.Kv8, a: L.Kv8Attention) -> int:
    """Bytes of workspace that mz_kv8_attention needs for these arguments."""
    n = C.c_size_t()
    check(L.lib().mz_kv8_attention_bytes(ctx.h, C.byref(kv), C.byref(a), C.byref(n)))
    return n.value


def scores_bytes(ctx: Context, a: L.ScoreArgs) -> int:
    """Bytes of workspace that mz_token_scores needs for these arguments."""
    n = C.c_size_t()
    check(L.lib().mz_token_scores_bytes(ctx.h, C.byref(a), C.byref(n)))
    return n.value


class Kv8:
    """A cache of `slots` sequences of up to max_tokens positions, `heads` heads of 64 channels, in one device buffer of
    the context. `kv` is the struct that the C entry points take."""

    def __init__(self, ctx: Context, slots: int, heads: int, max_tokens: int, fmt: str = "i8"):
        if fmt not in FORMATS:
            raise MzError(f"cache format {fmt!r}: one of {', '.join(FORMATS)}")
        self.ctx, self.fmt, self.base = ctx, fmt, 0
        n = C.c_size_t()
        check(L.lib().mz_kv8_place(FORMATS[fmt], slots, heads, max_tokens, 0, None, C.byref(n)))
        self.nbytes, self.kv = n.value, L.Kv8()
        self.base = ctx.alloc(self.nbytes)
        check(L.lib().mz_kv8_place(FORMATS[fmt], slots, heads, max_tokens, self.base, C.byref(self.kv), None))

    def free(self):
        if self.base:
            self.ctx.free(self.base)
            self.base, self.kv = 0, L.Kv8()

    def _io(self, k, v, rows, tokens, strides, slot, pos, pos_stride, pos_add, count) -> L.Kv8Io:
        h = self.kv.heads
        r, t, hs = strides or (tokens * h * HD, h * HD, HD)
        return L.Kv8Io(k, v, r, t, hs, rows, tokens, slot, pos, pos_stride, pos_add, count)

    def write(self, k: int, v: int, rows: int, tokens: int, strides=None, slot: int = 0, pos: int = 0,
              pos_stride: int = 1, pos_add: int = 0, count: int = 0):
        """Keys and values f16 of rows x tokens at their positions (mz_kv8_write). strides: (row, token, head) in
        elements, [rows][tokens][heads][64] if None."""
        a = self._io(k, v, rows, tokens, strides, slot, pos, pos_stride, pos_add, count)
        check(L.lib().mz_kv8_write(self.ctx.h, C.byref(self.kv), C.byref(a)))

    def read(self, k: int, v: int, rows: int, tokens: int, strides=None, slot: int = 0, pos: int = 0,
             pos_stride: int = 1, pos_add: int = 0, count: int = 0):
        """What the cache stands for, f16, into k and v (either may be 0) (mz_kv8_read); arguments as of write."""
        a = self._io(k, v, rows, tokens, strides, slot, pos, pos_stride, pos_add, count)
        check(L.lib().mz_kv8_read(self.ctx.h, C.byref(self.kv), C.byref(a)))

    def attention(self, q: int, out: int, rows: int, tokens: int, heads: int, q_strides=None, out_strides=None,
                  causal: bool = True, scale: float = 0.125, slot: int = 0, count: int = 0, len: int = 0,
                  len_stride: int = 1, len_add: int = 0, first: int = 0, lse: int = 0, head_slot: int = 0,
                  align: int = 0, align_heads: int = 0, align_cols: int = 0, work: tuple[int, int] | None = None):
        """Attention of rows x tokens queries f16 over the cache (mz_kv8_attention). Strides as of write, over `heads`
        query heads. work: (address, bytes) of a workspace, zero before its first use; None: the context's
        (Context.workspace)."""
        dense = (tokens * heads * HD, heads * HD, HD)
        a = L.Kv8Attention(q, out, *(q_strides or dense), *(out_strides or dense), rows, tokens, heads, int(causal), scale,
                           slot, count, len, len_stride, len_add, first, lse, head_slot, align, align_heads, align_cols)
        a.work, a.work_bytes = work or self.ctx.workspace(attention_bytes(self.ctx, self.kv, a))
        check(L.lib().mz_kv8_attention(self.ctx.h, C.byref(self.kv), C.byref(a)))


def token_scores(ctx: Context, logits: int, rows: int, vocab: int, dtype: int = L.DT_F32, ld: int = 0, mask: int = 0,
                 tokens: int = 0, token_stride: int = 1, at: int = 0, at_add: int = 0, logp: int = 0, entropy: int = 0,
                 out_stride: int = 1, alts: int = 0, alt_ids: int = 0, alt_logp: int = 0,
                 work: tuple[int, int] | None = None):
    """Log probabilities of given tokens, entropies and best alternatives of rows of logits (mz_token_scores). work: as of
    Kv8.attention."""
    a = L.ScoreArgs(dtype, rows, vocab, alts, logits, ld or vocab, mask, tokens, token_stride, at, at_add, logp, entropy,
                    out_stride, alt_ids, alt_logp)
    a.work, a.work_bytes = work or ctx.workspace(scores_bytes(ctx, a))
    check(L.lib().mz_token_scores(ctx.h, C.byref(a)))
