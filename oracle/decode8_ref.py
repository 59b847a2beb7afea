"""The 8-bit key/value caches, the attention over them and the token scores from their definitions, in numpy and 64
bits: what tests hold the kernels to."""
from __future__ import annotations

import numpy as np

BLK, HD = 32, 64
TOP = {"i8": 127.0, "e4m3": 448.0}


def to_code(v, fmt):
    """v (64 bits) rounded to the numbers that codes stand for, halves to even."""
    if fmt == "i8":
        return np.rint(v) + 0.0  # (whole numbers have one zero)
    _, e = np.frexp(v)
    unit = np.ldexp(1.0, np.maximum(e - 4, -9))
    return np.rint((v + 0.0) / unit) * unit  # (a zero of either sign is +0; what rounds to zero keeps its sign)


def code_bytes(c, fmt):
    if fmt == "i8":
        return c.astype(np.int8).view(np.uint8)
    a = np.abs(c)
    _, e = np.frexp(a)
    e = np.maximum(e - 1, -6)  # 2^e <= a < 2^(e + 1), or subnormal
    m = a / np.ldexp(1.0, e - 3)  # 8 .. 15, below 8: subnormal
    b = np.where(m >= 8, (e + 7) * 8 + (m - 8), m).astype(np.uint8)
    return b | np.where(np.signbit(c), 128, 0).astype(np.uint8)


def block(x, fmt):
    """(codes as numbers, scale f32, f16 values they stand for) of a block x f16 [32][64]."""
    x = x.astype(np.float64)
    if not np.isfinite(x).all():
        return np.zeros_like(x), np.float32(np.nan), np.full(x.shape, np.nan, np.float16)
    top = np.abs(x).max()
    if top == 0:
        return np.zeros_like(x), np.float32(0), np.zeros(x.shape, np.float16)
    c = to_code(TOP[fmt] * x / top, fmt)
    s = np.float32(top / TOP[fmt])
    return c, s, (c.astype(np.float32) * s).astype(np.float16)


def value_order(x):
    """Blocks [..., 32 positions, 64 channels] in the order of v: [..., 32][4][2][8]."""
    x = x.reshape(*x.shape[:-2], 4, 8, 32, 2)
    n = x.ndim
    return np.ascontiguousarray(np.moveaxis(x, (n - 2, n - 4, n - 1, n - 3), (n - 4, n - 3, n - 2, n - 1)))


class Cache:
    """One cache: raw arrays as the library lays them out, and what every position stands for, f16."""

    def __init__(self, slots, heads, max_tokens, fmt):
        self.slots, self.heads, self.fmt = slots, heads, fmt
        self.blocks = -(-max_tokens // BLK)
        self.cap = self.blocks * BLK
        sh = (slots, heads)
        self.code = [np.zeros(sh + (self.blocks, BLK, HD)) for _ in "kv"]
        self.scale = [np.zeros(sh + (self.blocks,), np.float32) for _ in "kv"]
        self.opened = [np.zeros(sh + (BLK, HD), np.float16) for _ in "kv"]
        self.open = np.zeros(sh, np.int32)

    def stands_for(self, side):
        """[slots][heads][positions][64] f16."""
        x = (self.code[side].astype(np.float32) * self.scale[side][..., None, None]).astype(np.float16)
        for s, h in zip(*np.nonzero(self.open)):
            x[s, h, self.open[s, h] - 1] = self.opened[side][s, h]
        return x.reshape(self.slots, self.heads, self.cap, HD)

    def exact(self, side):
        """The same in 64 bits, codes times scales not rounded."""
        x = self.code[side] * self.scale[side][..., None, None].astype(np.float64)
        for s, h in zip(*np.nonzero(self.open)):
            x[s, h, self.open[s, h] - 1] = self.opened[side][s, h]
        return x.reshape(self.slots, self.heads, self.cap, HD)

    def write(self, k, v, slot=None, pos=None, count=None):
        """k, v f16 [rows][tokens][heads][64]."""
        rows, tokens = k.shape[:2]
        todo = {}  # slot: its row, position and tokens
        for r in range(rows):
            s = r if slot is None else int(slot[r])
            p = 0 if pos is None else int(pos[r])
            n = tokens if count is None else min(max(int(count[r]), 0), tokens)
            if 0 <= s < self.slots and n > 0 and p >= 0 and p + n <= self.cap:
                todo[s] = r, p, n
        for s, (r, p, n) in todo.items():
            for h in range(self.heads):
                was, last = int(self.open[s, h]) - 1, (p + n - 1) // BLK
                for side, src in enumerate((k, v)):
                    for b in range(p // BLK, last + 1):
                        off, end = max(p - b * BLK, 0), min(p + n - b * BLK, BLK)
                        x = np.zeros((BLK, HD), np.float16)
                        old = self.opened[side][s, h] if was == b else (
                            self.code[side][s, h, b].astype(np.float32) * self.scale[side][s, h, b]).astype(np.float16)
                        x[:off] = old[:off]
                        x[off:end] = src[r, b * BLK + off - p:b * BLK + end - p, h]
                        if end == BLK:
                            self.code[side][s, h, b], self.scale[side][s, h, b], _ = block(x, self.fmt)
                        else:
                            self.opened[side][s, h, :end] = x[:end]
                self.open[s, h] = last + 1 if (p + n) % BLK else 0


def attention(cache, q, causal, length, slot=None, first=None, count=None, scale=0.125):
    """q [rows][tokens][heads][64] -> (out, lse, probabilities [rows][tokens][heads][positions], spread of the rounding
    terms): length[r] positions for token 0. The last output holds sum p |v| and max sum |q k| * scale for bounds."""
    rows, tokens, heads = q.shape[:3]
    grp = heads // cache.heads
    kk, vv = cache.exact(0), cache.exact(1)
    out = np.zeros(q.shape)
    lse = np.full((rows, tokens, heads), -np.inf)
    prob = np.zeros((rows, tokens, heads, cache.cap))
    av, aq = np.zeros(q.shape), np.zeros((rows, tokens, heads))
    for r in range(rows):
        s = r if slot is None else int(slot[r])
        if not 0 <= s < cache.slots:
            continue
        lo = 0 if first is None else max(int(first[r]), 0)
        for i in range(tokens):
            hi = min(max(int(length[r]) + (i if causal else 0), 0), cache.cap)
            if hi <= lo:
                continue
            for h in range(heads):
                k, v = kk[s, h // grp, lo:hi], vv[s, h // grp, lo:hi]
                qd = q[r, i, h].astype(np.float64)
                x = k @ qd * scale
                m = x.max()
                e = np.exp(x - m)
                z = e.sum()
                out[r, i, h] = (e / z) @ v
                lse[r, i, h] = m + np.log(z)
                prob[r, i, h, lo:hi] = e / z
                av[r, i, h] = (e / z) @ np.abs(v)
                aq[r, i, h] = (np.abs(k) @ np.abs(qd)).max() * scale
    return out, lse, prob, (av, aq)


def scores(x, tokens, mask=None, alts=0):
    """x [rows][vocab] -> (logp, entropy, ids, logp of ids) as mz_token_scores defines them."""
    x = x.astype(np.float64).copy()
    if mask is not None:
        x[:, mask != 0] = -np.inf
    rows, vocab = x.shape
    logp, ent = np.zeros(rows), np.zeros(rows)
    ids, best = np.full((rows, alts), -1, np.int32), np.full((rows, alts), -np.inf)
    for r in range(rows):
        t = int(tokens[r])
        if np.isnan(x[r]).any() or (x[r] == np.inf).any():
            logp[r] = 0.0 if t < 0 else np.nan
            ent[r] = np.nan
            best[r] = np.nan
            continue
        m = x[r].max()
        if m == -np.inf:
            logp[r] = 0.0 if t < 0 else np.nan if t >= vocab else -np.inf
            continue
        a = int(x[r].argmax())
        d = x[r] - m
        e = np.exp(d)
        e[a] = 0.0
        z = np.log1p(e.sum())
        logp[r] = 0.0 if t < 0 else np.nan if t >= vocab else d[t] - z
        ent[r] = z - (e * np.maximum(d, -1e6)).sum() / (1.0 + e.sum())
        order = np.argsort(-x[r], kind="stable")[:alts]
        for k, i in enumerate(order):
            if x[r, i] > -np.inf:
                ids[r, k], best[r, k] = i, d[i] - z
    return logp, ent, ids, best
