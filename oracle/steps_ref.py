"""Products with 4-bit weights, attention over an encoder's output and the choice of the next token from their definitions,
in numpy and 64 bits: what tests hold the kernels to."""
from __future__ import annotations

import math

import numpy as np
from scipy.special import ndtr

HD = 64


# ---------------------------------------------------------------- weights in 4 bits


def w4_codes(w, group):
    """(codes as whole numbers [n][k], scales f16 [n][k / group]) of weights f16 [n][k]."""
    n, k = w.shape
    x = w.astype(np.float64).reshape(n, k // group, group)
    bad = ~np.isfinite(x).all(-1)
    x = np.where(bad[..., None], 0.0, x)
    hi, lo = x.max(-1), x.min(-1)
    s = (np.where(hi > -lo, hi, lo) / -8.0).astype(np.float16)
    d = s.astype(np.float64)[..., None]
    c = np.clip(np.rint(np.divide(x, d, out=np.zeros_like(x), where=d != 0)), -8, 7)
    s = np.where(bad, np.float16(np.nan), s)
    return c.reshape(n, k), s


def w4_bytes_of(codes, scales, group):
    """The two arrays as the header lays them out: u8 [tiles][k / 128][64][16], f16 [tiles][k / 128][16][128 / group]."""
    n, k = codes.shape
    tiles, chunks, groups = -(-n // 16), k // 128, 128 // group
    c = np.zeros((tiles * 16, k), np.int64)
    c[:n] = codes
    words = np.zeros((tiles, chunks, 4, 16, 4), np.uint32)  # [tile][chunk][j][row][s]
    v = (c + 8).reshape(tiles, 16, chunks, 4, 4, 8).astype(np.uint32)  # [tile][row][chunk][s][j][e]
    for e in range(8):
        words |= v[..., e].transpose(0, 2, 4, 1, 3) << np.uint32(4 * (e // 2) + 16 * (e % 2))
    s = np.zeros((tiles * 16, k // group), np.float16)
    s[:n] = scales
    s = s.reshape(tiles, 16, chunks, groups).transpose(0, 2, 1, 3)
    return np.ascontiguousarray(words).view(np.uint8).reshape(tiles, chunks, 64, 16), np.ascontiguousarray(s)


def w4_values(codes, scales, group):
    """What codes stand for, in 64 bits."""
    return codes * np.repeat(scales.astype(np.float64), group, axis=1)


def w4_linear(x, w, bias=None):
    """(x . w^T + bias, the sum of the magnitudes) in 64 bits."""
    y, size = x.astype(np.float64) @ w.T, np.abs(x.astype(np.float64)) @ np.abs(w).T
    if bias is not None:
        y, size = y + bias.astype(np.float64), size + np.abs(bias.astype(np.float64))
    return y, size


def gelu(y):
    return y * ndtr(y)


# ---------------------------------------------------------------- attention


def cross(q, k, v, scale=0.125, slot=None, first=None, length=None, count=None):
    """q f16 [rows][tokens][heads][64], k and v f16 [slots][positions][kv_heads][64] -> dict of out [rows][tokens][heads][64],
    lse [rows][tokens][heads], p [rows][tokens][heads][positions], and of what tolerances need: size (sum of p |v|), ds (the
    largest scale sum |q k| of what a query sees), n (the positions it sees). Tokens from count on are NaN."""
    rows, tokens, heads, _ = q.shape
    slots, pos, kvh, _ = k.shape
    r = {"out": np.zeros(q.shape), "lse": np.full((rows, tokens, heads), -np.inf), "p": np.zeros((rows, tokens, heads, pos)),
         "size": np.zeros(q.shape), "ds": np.zeros((rows, tokens, heads)), "n": np.zeros((rows, 1, 1))}
    for i in range(rows):
        s = i if slot is None else int(slot[i])
        lo = 0 if first is None else max(int(first[i]), 0)
        hi = pos if length is None else min(int(length[i]), pos)
        if 0 <= s < slots and hi > lo:
            r["n"][i] = hi - lo
            for h in range(heads):
                kk, vv = (x[s, lo:hi, h // (heads // kvh)].astype(np.float64) for x in (k, v))
                qq = q[i, :, h].astype(np.float64)
                x = qq @ kk.T * scale
                r["ds"][i, :, h] = (np.abs(qq) @ np.abs(kk).T * scale).max(-1)
                m = x.max(-1, keepdims=True)
                e = np.exp(x - m)
                z = e.sum(-1, keepdims=True)
                r["lse"][i, :, h] = (m + np.log(z))[:, 0]
                p = e / z
                r["p"][i, :, h, lo:hi] = p
                r["out"][i, :, h] = p @ vv
                r["size"][i, :, h] = p @ np.abs(vv)
        if count is not None:
            for name in ("out", "lse", "p"):
                r[name][i, max(int(count[i]), 0):] = np.nan
    return r


# ---------------------------------------------------------------- the next token


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mask=None):
    """One row of logits -> (token, logp, kept, how near u is to a border of the token's share, and the limits to a border of
    theirs, as a share of the sum)."""
    x = np.asarray(x, np.float64).copy()
    if mask is not None:
        x[mask.astype(bool)] = -np.inf
    t, p, low = float(temperature), float(top_p), float(min_p)
    if np.isnan(x).any() or (x == np.inf).any() or not 0 <= t < math.inf or math.isnan(p) or math.isnan(low):
        return -1, math.nan, 0, 1.0
    ids = np.nonzero(x > -np.inf)[0]
    if not len(ids):
        return -1, -math.inf, 0, 1.0
    order = ids[np.argsort(-x[ids], kind="stable")]
    if t == 0:
        return int(order[0]), 0.0, 1, 1.0
    if 0 < top_k < len(order):
        order = order[:top_k]
    w = np.exp((x[order] - x[order[0]]) / t)
    near = 1.0
    keep = len(order)
    if p < 1:
        run = np.cumsum(w)
        need = max(p, 0.0) * run[-1]
        keep = max(1, int(np.searchsorted(run, need)) + 1)
        near = min(near, np.abs(run - need).min() / run[-1]) if p > 0 else near
    if low > 0:
        keep = min(keep, max(1, int((w >= low).sum())))
        near = min(near, np.abs(w[1:] - low).min()) if low < 1 and len(w) > 1 else near  # (the largest weight is exactly 1)
    order, w = order[:keep], w[:keep]
    by_id = np.argsort(order)
    run = np.cumsum(w[by_id])
    u = 0.0 if not u >= 0 else min(float(u), 1.0 - 2.0 ** -24)
    i = min(int(np.searchsorted(run, u * run[-1], side="right")), keep - 1)
    near = min(near, np.abs(np.concatenate([run[:-1], [np.inf]]) / run[-1] - u).min())
    tok = order[by_id[i]]
    return int(tok), float((x[tok] - x[order[0]]) / t - np.log(run[-1])), keep, near
