"""Attention over 8-bit caches, their reading and token scores where their definitions are easily missed. Against
oracle/decode8_ref.py (numpy, 64 bits); helpers and the counting of roundings as in test_gpu_decode8.py."""
import numpy as np
import pytest
from test_gpu_decode8 import FMT, Both, H, U, check_scores, ctx, dev, f16, i32, run_attention, run_scores  # noqa: F401

from oracle import decode8_ref as R

pytestmark = pytest.mark.gpu


def filled_with(ctx, dev, fmt, k, v):
    """A cache whose one slot holds the sequence k, v [positions][heads][64]."""
    b = Both(ctx, 1, k.shape[1], k.shape[0], fmt)
    b.write(dev, k.astype(np.float16)[None], v.astype(np.float16)[None])
    return b


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("rows,heads,tokens", [(1, 2, 1), (1, 2, 9), (1, 2, 24), (17, 16, 1), (40, 20, 24)])
@pytest.mark.parametrize("what", ["key", "value", "open value", "open key"])
def test_a_query_that_sees_nothing_of_a_block_with_nan(ctx, dev, fmt, rows, heads, tokens, what):
    """Padding in front: a row's first position lies inside a block and its first tokens end before it, in the same block, which
    holds a NaN: out 0 and lse -inf. A later token that sees the block gets what it holds."""
    rng = np.random.default_rng(tokens)
    n = 60 if what.startswith("open") else 64
    k, v = f16(rng, (n, heads, 64)), f16(rng, (n, heads, 64))
    (k if what.endswith("key") else v)[45, :, 5] = np.nan  # block 1
    b = Both(ctx, 1, heads, 64, fmt)
    b.write(dev, k[None], v[None])
    q = f16(rng, (rows, tokens, heads, 64), 1.5)
    first, length = 44, 34  # token i sees positions 44 .. 33 + i
    for causal in (False, True):
        end = length + (np.arange(tokens) if causal else np.zeros(tokens, int))
        out, lse, _ = run_attention(ctx, dev, b, q, causal, [length] * rows, slot=[0] * rows, first=[first] * rows)
        none = end <= first
        assert none.any()
        assert (out[:, none] == 0).all() and (lse[:, none] == -np.inf).all()
        if what in ("key", "value"):
            assert np.isnan(out[:, ~none, :, 5]).all()  # the block is none as a whole
    b.free()


def expected(b, q, causal, length, **kw):
    """Outputs and lse in 64 bits, and how far an output may be from them. Probabilities are carried with 16 bits or more (2^-16
    relative, of two roundings to 8 bits each) whatever their size, sums are of 32-bit numbers in any order (a score's error
    ds and n + 16 roundings u, relative to sum p |v|), the output is rounded once: h relative, or half its smallest step."""
    w, lse, prob, (av, aq) = R.attention(b.r, q, causal, length, **kw)
    rel = 2 * 80 * U * aq + ((prob > 0).sum(-1) + 16) * U + 2.0 ** -16
    return w, lse, rel[..., None] * av + H * np.abs(w) + 2.0 ** -25


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("rows,heads,tokens", [(1, 1, 1), (32, 10, 1), (1, 2, 20), (40, 8, 20), (90, 10, 20)])
@pytest.mark.parametrize("n", [20, 1500, 15990])
def test_a_long_tail_far_below_the_peak(ctx, dev, fmt, rows, heads, tokens, n):
    """A sequence whose first block has large values and next to no weight, a peak whose own value is 0 in some channels, and
    all other positions `down` powers of two below it, with values 1/120 of the first block's: what these channels get comes
    from the tail alone. 20 positions: all of them in the open block, with values of thousands."""
    rng = np.random.default_rng(n)
    at = 40 if n > 40 else 3  # the peak
    k = np.zeros((n, heads, 64))
    k[..., 1:] = rng.standard_normal((n, heads, 63)) * 0.3
    v = (0.3 + 0.2 * rng.random((n, heads, 64))) * (1 if n > 32 else 20000)
    if n > 32:
        v[:32] = 60.0 * rng.standard_normal((32, heads, 64))
        k[:32, :, 0] = -1.0
    k[at, :, 0] = 1.0
    v[at, :, :32] = 0.0
    b = filled_with(ctx, dev, fmt, k, v)
    for down in (6, 12, 18, 40):
        q = np.zeros((rows, tokens, heads, 64), np.float16)  # (a score is the first channel's product alone)
        q[..., 0] = down * np.log(2) / 0.125
        for first in (0, 32) if n > 32 else (0,):  # (without the first block no large values are met)
            out, lse, _ = run_attention(ctx, dev, b, q, False, [n] * rows, slot=[0] * rows, first=[first] * rows)
            w, wl, tol = expected(b, q[:1, :1], False, [n], slot=[0], first=[first])
            err = np.abs(out.astype(np.float64) - w)
            assert (err <= tol).all(), f"{down}: {(err / tol).max():.3g} x the bound, {(err / np.abs(w))[..., :32].max():.2g} of the output"
            assert (np.abs(lse - wl) <= 160 * U * down + (n + 8) * U + 4 * U * np.abs(wl)).all()
    b.free()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("rows,heads,kvh,tokens", [(2, 2, 2, 1), (2, 4, 4, 16), (2, 4, 4, 17), (3, 8, 2, 5), (20, 16, 16, 65), (8, 20, 20, 224)])
def test_outputs_are_as_exact_for_prompts_as_for_single_tokens(ctx, dev, fmt, rows, heads, kvh, tokens):
    """The output's own rounding to fp16 and little else, whatever the number of queries."""
    rng = np.random.default_rng(rows + tokens)
    past = [(37 * r) % 150 for r in range(rows)]
    t = max(past) + tokens
    b = Both(ctx, rows, kvh, t, fmt)
    b.write(dev, f16(rng, (rows, t, kvh, 64)), f16(rng, (rows, t, kvh, 64)), count=[p + tokens for p in past])
    q = f16(rng, (rows, tokens, heads, 64), 1.5)
    out = run_attention(ctx, dev, b, q, True, [p + 1 for p in past])[0]
    w, _, tol = expected(b, q, True, [p + 1 for p in past])
    err = np.abs(out.astype(np.float64) - w)
    assert (err <= tol).all(), f"{(err / tol).max():.3g} x the bound at {np.argwhere(err > tol)[:3].tolist()}, {(err > tol).mean():.2g} of them"
    b.free()


# ---------------------------------------------------------------- token scores


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows", [1, 40, 1100])
@pytest.mark.parametrize("alts", [1, 5, 16])
def test_zeros_of_either_sign_are_one_value(ctx, dev, dtype, rows, alts):
    """The best logits are zeros, -0 at some ids and +0 at others, in one lane, in lanes, waves and workgroups of their own, a
    few of them and (through the network) many: the lowest ids come first."""
    rng = np.random.default_rng(rows + alts)
    v = 20011
    x = -1.0 - np.abs(rng.standard_normal((rows, v)))
    for r in range(rows):
        # (neighbours share a lane; 16 on another lane, 1024 on another wave, 8192 on another workgroup of a split row)
        step = [1, 3, 16, 64, 1024, 5000, 8192, 700][r % 8] if rows > 1 else 5000
        ids = (np.arange(3, v, step) if r % 3 else np.arange(v - 1, -1, -step))[:[2, 3, 9, 40][r // 8 % 4]]
        x[r, ids] = np.where(rng.random(len(ids)) < 0.5, 0.0, -0.0)
        x[r, ids.min()] = -0.0
        x[r, ids.max()] = 0.0
    x = x.astype(dtype)
    tokens = rng.integers(0, v, rows)
    mask = (rng.random(v) < 0.01).astype(np.uint8)
    for m in (None, mask):
        check_scores(x, tokens, run_scores(ctx, dev, x, tokens, m, alts), m, alts)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("vocab", [2, 70, 5000])
def test_rows_of_zeros_of_either_sign(ctx, dev, dtype, vocab):
    rng = np.random.default_rng(vocab)
    x = np.where(rng.random((6, vocab)) < 0.5, 0.0, -0.0).astype(dtype)
    x[:, 0], x[:, -1] = -0.0, 0.0
    tokens = np.full(6, vocab - 1)
    for alts in (1, 2, 16):
        check_scores(x, tokens, run_scores(ctx, dev, x, tokens, None, alts), None, alts)


# ---------------------------------------------------------------- reading


@pytest.mark.parametrize("fmt", FMT)
def test_read_from_before_the_cache(ctx, dev, fmt):
    """Tokens at negative positions are left as they were, the others of their row are read."""
    rng = np.random.default_rng(8)
    b = Both(ctx, 2, 3, 128, fmt)
    b.write(dev, f16(rng, (2, 128, 3, 64)), f16(rng, (2, 128, 3, 64)), count=[128, 77])
    pos, count = [-5, -1, -40, -32, -70, -71, -(2 ** 31), -64, -3, 100, 127, 128], [10, 1, 70, 33, 70, 70, 70, 70, 0, 70, 70, 70]
    n, t = len(pos), 70
    slot = [r % 2 for r in range(n)]
    init = f16(rng, (n, 3, t, 64))
    for add in (0, 7, -(2 ** 31)):
        ok, ov = dev(init), dev(init)
        b.d.read(ok, ov, n, t, strides=(3 * t * 64, 64, t * 64), slot=dev(i32(slot)), pos=dev(i32(pos)), pos_add=add, count=dev(i32(count)))
        for at, side in ((ok, 0), (ov, 1)):
            want, src = init.copy(), b.r.stands_for(side)
            for r in range(n):
                for i in range(count[r]):
                    p = pos[r] + add + i
                    if 0 <= p < 128:
                        want[r, :, i] = src[slot[r], :, p]
            np.testing.assert_array_equal(ctx.download(at, init.shape, np.float16).view(np.uint16), want.view(np.uint16))
    # without an array: pos_add alone, all tokens
    o = dev(init[:2])
    b.d.read(o, 0, 2, t, strides=(3 * t * 64, 64, t * 64), pos_add=-33)
    want = init[:2].copy()
    want[:, :, 33:] = b.r.stands_for(0)[:, :, :t - 33]
    np.testing.assert_array_equal(ctx.download(o, want.shape, np.float16).view(np.uint16), want.view(np.uint16))
    b.free()
