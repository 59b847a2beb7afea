"""GPU parity of the parts of a decoder step, products with 4-bit weights, attention over an encoder's output and the choice
of the next token, through the C ABI, against oracle/steps_ref.py (numpy, 64 bits).

What is packed is compared bit for bit, and so are the tokens drawn (wherever no sum lies within 1e-11 of a border: weights are
multiples of 2^-46 or less of the largest, at most 2^17 of them) and the number kept. Tolerances of the rest count roundings,
u = 2^-24 in 32 bits and h = 2^-11 in fp16 (half a step each):
  a product's sum       2 (k + 16) u sum |c s x| (a matrix instruction may cut instead of rounding: twice a rounding)
  its output            h |y| + 2^-25 (fp16), u |y| (fp32); GELU, whose slope is at most 1.13, 1.13 times the sum's error and
                        0.505 steps: 1.01 h |y| + 2^-25
  a score's exponent    (64 products and sums + 16 for the scale, the maximum and exp2) u sum |q k| scale = ds
  lse                   ds + (n + 8) u (a sum of n terms, in any order) + 4 u |lse|
  a probability         relative 2 ds + (n + 16) u, and 2^-120 for those at the bottom of the range
  attention's output    the probabilities' error, 2^-20 and n 2^-31 of the largest for their two fp16 parts, times sum p |v|; h
                        for the output's own; 2^-24 for numbers below fp16's normal range
  a drawn token's logp  u |logp| + 2^-40
"""
import ctypes as C

import numpy as np
import pytest

from mimizuku_amd import _lib as L
from mimizuku_amd import model, steps
from oracle import steps_ref as R

pytestmark = pytest.mark.gpu
U, H = 2.0 ** -24, 2.0 ** -11


@pytest.fixture(scope="module")
def ctx():
    c = model.Context(0)
    yield c
    c.close()


class Dev:
    """Device copies of arrays, freed together."""

    def __init__(self, ctx):
        self.ctx, self.at = ctx, []

    def __call__(self, a):
        if a is None:
            return 0
        self.at.append(self.ctx.upload_new(np.ascontiguousarray(a)))
        return self.at[-1]

    def free(self):
        for p in self.at:
            self.ctx.free(p)


@pytest.fixture
def dev(ctx):
    d = Dev(ctx)
    yield d
    d.free()


def i32(v):
    return None if v is None else np.asarray(v, np.int32)


def f32(v):
    return None if v is None else np.asarray(v, np.float32)


def f16(rng, shape, scale=0.7):
    return (rng.standard_normal(shape, dtype=np.float32) * scale).astype(np.float16)


# ---------------------------------------------------------------- weights in 4 bits


def packed(ctx, dev, w, group, ld=0):
    n, k = w.shape
    src = w
    if ld:
        src = np.full((n, ld), 7, np.float16)
        src[:, :k] = w
    p = steps.W4(ctx, n, k, group, at=dev(np.zeros(steps.w4_bytes(n, k, group) + 256, np.uint8)))
    p.pack(dev(src), ld)
    return p


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k,ld", [(1, 128, 0), (16, 128, 136), (40, 384, 0), (77, 1280, 1288), (1000, 256, 0)])
def test_w4_pack_and_unpack(ctx, dev, n, k, ld, group):
    rng = np.random.default_rng(n + k + group)
    w = f16(rng, (n, k), 0.05)
    w[0, :group] = 0
    w[n // 2, :3] = 60000, -65504, 1e-7
    w[n - 1, 3:6] = 2.0, -2.0, 1.0  # alike in size, and a quotient halfway
    w[n - 1, group - 1] = 0.125
    w[n // 3, k - group:] = np.float16(6e-8) * np.arange(group) % 1e-6  # scales below fp16's range
    if n > 3:
        w[1, k - 1], w[2, 0], w[2, k - 1] = np.nan, np.inf, -np.inf
    p = packed(ctx, dev, w, group, ld)
    c, s = R.w4_codes(w, group)
    words, scales = R.w4_bytes_of(c, s, group)
    np.testing.assert_array_equal(ctx.download(p.w.codes, words.shape, np.uint8), words)
    got = ctx.download(p.w.scales, scales.shape, np.float16)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(scales))
    np.testing.assert_array_equal(got[~np.isnan(got)], scales[~np.isnan(got)])
    out = dev(np.full((n, k + 8), 9, np.float16))
    p.unpack(out, k + 8)
    y = ctx.download(out, (n, k + 8), np.float16)
    assert (y[:, k:] == 9).all()
    with np.errstate(invalid="ignore"):
        want = (c.astype(np.float32) * np.repeat(s, group, 1).astype(np.float32)).astype(np.float16)
    np.testing.assert_array_equal(y[:, :k], want)


def check_linear(x, w64, bias, epilogue, got, before=None):
    y, size = R.w4_linear(x, w64, bias)
    err = 2 * (x.shape[1] + 16) * U * size
    if epilogue == L.EPI_GELU_F16:
        g = R.gelu(y)
        tol = 1.13 * err + 1.01 * H * np.abs(g) + 2.0 ** -25
        y = g
    elif epilogue == L.EPI_F16:
        tol = err + H * (np.abs(y) + err) + 2.0 ** -25
    else:
        if before is not None:
            y = y + before
        tol = err + U * (np.abs(y) + err)
    bad = ~(np.abs(got - y) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], y[bad][:4], tol[bad][:4])


def run_linear(ctx, dev, p, x, bias, epilogue, ldx=0, ldo=0, off=0):
    """x and out with rows ldx and ldo apart, out `off` elements behind an aligned address."""
    m, n = x.shape[0], p.w.n
    if ldx:
        xs = np.full((m, ldx), np.nan, np.float16)
        xs[:, :x.shape[1]] = x
        x = xs
    half = epilogue in (L.EPI_F16, L.EPI_GELU_F16)
    dtype, o = (np.float16 if half else np.float32), ldo or n
    rng = np.random.default_rng(5)
    before = rng.standard_normal(off + m * o).astype(dtype)
    out = dev(before)
    p.linear(dev(x), out + off * before.itemsize, m, epilogue, dev(bias), ldx, ldo)
    after = ctx.download(out, before.shape, dtype)
    rows = lambda a: a[off:].reshape(m, o)  # noqa: E731
    np.testing.assert_array_equal(after[:off], before[:off])
    np.testing.assert_array_equal(rows(after)[:, n:], rows(before)[:, n:])
    return rows(after)[:, :n], rows(before)[:, :n]


EPI = [L.EPI_F16, L.EPI_GELU_F16, L.EPI_RESID_F32, L.EPI_F32]


@pytest.mark.parametrize("m", [1, 2, 5, 8, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 129, 224, 300])
@pytest.mark.parametrize("n,k,group", [(1, 128, 128), (37, 384, 32), (512, 512, 64), (1283, 256, 128), (333, 1280, 64)])
def test_w4_linear(ctx, dev, m, n, k, group):
    rng = np.random.default_rng(m * 7 + n)
    w, x = f16(rng, (n, k), k ** -0.5), f16(rng, (m, k), 1.0)
    p = packed(ctx, dev, w, group)
    w64 = R.w4_values(*R.w4_codes(w, group), group)
    epilogue = EPI[(m + n) % 4]
    bias = f16(rng, (n,), 0.3) if m % 3 else None
    got, before = run_linear(ctx, dev, p, x, bias, epilogue)
    check_linear(x, w64, bias, epilogue, got, before if epilogue == L.EPI_RESID_F32 else None)


@pytest.mark.parametrize("epilogue", EPI)
@pytest.mark.parametrize("m,n,k,group,ldx,ldo,off", [(3, 45, 256, 32, 264, 47, 1), (19, 64, 128, 64, 0, 67, 3), (40, 130, 640, 128, 648, 136, 4),
                                                     (1, 4096, 128, 32, 0, 0, 2), (70, 51, 384, 32, 400, 0, 0),
                                                     (150, 200, 256, 64, 0, 203, 5)])
def test_w4_linear_layouts(ctx, dev, epilogue, m, n, k, group, ldx, ldo, off):
    rng = np.random.default_rng(m + n)
    w, x, bias = f16(rng, (n, k), k ** -0.5), f16(rng, (m, k), 1.0), f16(rng, (n,), 0.3)
    p = packed(ctx, dev, w, group)
    got, before = run_linear(ctx, dev, p, x, bias, epilogue, ldx, ldo, off)
    check_linear(x, R.w4_values(*R.w4_codes(w, group), group), bias, epilogue, got, before if epilogue == L.EPI_RESID_F32 else None)


@pytest.mark.parametrize("m,n,k,group", [(1, 1536, 384, 32), (1, 1280, 5120, 64), (8, 1280, 5120, 128), (32, 1280, 5120, 32),
                                         (4, 384, 1536, 32), (2, 51865, 384, 64), (32, 51866, 512, 32), (200, 1280, 1280, 64),
                                         (1, 80, 16384, 128), (20, 33, 20480, 32), (448, 5120, 1280, 128), (1100, 640, 256, 32)])
def test_w4_linear_of_model_sizes(ctx, dev, m, n, k, group):
    rng = np.random.default_rng(m + n + k)
    w, x, bias = f16(rng, (n, k), k ** -0.5), f16(rng, (m, k), 1.0), f16(rng, (n,), 0.3)
    p = packed(ctx, dev, w, group)
    got, _ = run_linear(ctx, dev, p, x, bias, L.EPI_F32)
    check_linear(x, R.w4_values(*R.w4_codes(w, group), group), bias, L.EPI_F32, got)
    again, _ = run_linear(ctx, dev, p, x, bias, L.EPI_F32)
    np.testing.assert_array_equal(got, again)


@pytest.mark.parametrize("m", [1, 9, 40, 200])
@pytest.mark.parametrize("group", [32, 128])
def test_w4_linear_of_unusual_numbers(ctx, dev, m, group):
    """Rows of x and of weights that are no numbers stay to themselves; large, tiny and zero ones."""
    rng = np.random.default_rng(m)
    n, k = 70, 256
    w, x = f16(rng, (n, k), 0.1), f16(rng, (m, k), 1.0)
    w[3, 200], w[66, 0] = np.nan, np.inf
    w[10] *= 1000
    w[11] = 0
    w[12] *= np.float16(1e-4)
    x[0, 7] = np.inf if m > 1 else 30000.0
    if m > 1:
        x[m - 1] *= 200
    p = packed(ctx, dev, w, group)
    got, _ = run_linear(ctx, dev, p, x, None, L.EPI_F32)
    w64 = R.w4_values(*R.w4_codes(w, group), group)
    good = np.ones((m, n), bool)
    good[:, [3, 66]] = False
    assert np.isnan(got[:, [3, 66]]).all()
    if m > 1:
        assert not np.isfinite(got[0][w64[:, 7] != 0]).any()
        good[0] = False
    xs, ws = np.where(np.isfinite(x), x, 0).astype(np.float16), np.where(np.isnan(w64), 0, w64)
    y, size = R.w4_linear(xs, ws)
    tol = 2 * (k + 16) * U * size + U * np.abs(y)
    assert (np.abs(got - y) <= tol)[good].all()
    assert (got[1:, 11] == 0).all()


def test_w4_linear_past_32_bits(ctx, dev):
    """Rows of x and of the output more than 2^32 bytes apart, and weights whose codes pass 2^31 bytes are not needed for it."""
    rng = np.random.default_rng(0)
    m, n, k = 3, 20, 128
    w, x = f16(rng, (n, k), 0.1), f16(rng, (m, k), 1.0)
    p = packed(ctx, dev, w, 32)
    ldx, ldo = (1 << 31) + 64, (1 << 30) + 3  # halves, floats
    xs, out = ctx.alloc((m - 1) * ldx * 2 + k * 2), ctx.alloc((m - 1) * ldo * 4 + n * 4)
    try:
        for i in range(m):
            ctx.upload(xs + i * ldx * 2, x[i])
        p.linear(xs, out, m, L.EPI_F32, 0, ldx, ldo)
        got = np.stack([ctx.download(out + i * ldo * 4, (n,), np.float32) for i in range(m)])
        check_linear(x, R.w4_values(*R.w4_codes(w, 32), 32), None, L.EPI_F32, got)
    finally:
        ctx.free(xs)
        ctx.free(out)


# ---------------------------------------------------------------- attention


def run_cross(ctx, dev, q, k, v, slot=None, first=None, length=None, count=None, scale=0.125, head_slot=None, align_heads=0,
              align_cols=0, **kw):
    """k, v [slots][positions][kv_heads][64] as they lie."""
    rows, tokens, heads, _ = q.shape
    slots, pos, kvh, _ = k.shape
    out0, lse0 = np.full(q.shape, 3, np.float16), np.full((rows, tokens, heads), 5, np.float32)
    out, lse = dev(out0), dev(lse0)
    al = dev(np.full((rows, tokens, align_heads, align_cols), 7, np.float32)) if align_heads else 0
    steps.cross_attention(ctx, dev(q), out, dev(k), dev(v), rows, tokens, heads, pos, slots, kvh,
                          k_strides=(pos * kvh * 64, kvh * 64, 64), scale=scale, slot=dev(i32(slot)), count=dev(i32(count)),
                          first=dev(i32(first)), len=dev(i32(length)), lse=lse, head_slot=dev(i32(head_slot)), align=al,
                          align_heads=align_heads, align_cols=align_cols, **kw)
    got = {"out": ctx.download(out, q.shape, np.float16), "lse": ctx.download(lse, lse0.shape, np.float32)}
    if align_heads:
        got["align"] = ctx.download(al, (rows, tokens, align_heads, align_cols), np.float32)
    return got


def check_cross(q, k, v, got, head_slot=None, **kw):
    r = R.cross(q, k, v, **{x: y for x, y in kw.items() if x in ("slot", "first", "length", "count", "scale")})
    gone = np.isnan(r["lse"])
    assert (got["out"][gone] == 3).all() and (got["lse"][gone] == 5).all()
    ok = ~gone
    none = np.isneginf(r["lse"]) & ok
    assert (got["lse"][none] == -np.inf).all() and (got["out"][none] == 0).all()
    some = ok & ~none
    ds = (64 + 16) * U * r["ds"]
    n = np.broadcast_to(r["n"], ds.shape)
    err = ds + (n + 8) * U + 4 * U * np.abs(np.where(some, r["lse"], 0))
    bad = ~(np.abs(got["lse"] - np.where(some, r["lse"], 0)) <= err) & some
    assert not bad.any(), (np.argwhere(bad)[:4], got["lse"][bad][:4], r["lse"][bad][:4])
    rel = (2 * ds + (n + 16) * U + 2.0 ** -20)[..., None]
    far = np.abs(v.astype(np.float64)).max()
    tol = rel * r["size"] + (n * 2.0 ** -31)[..., None] * far + H * (1 + rel) * np.abs(r["out"]) + 2.0 ** -24
    bad = ~(np.abs(got["out"] - r["out"]) <= tol) & some[..., None]
    assert not bad.any(), (np.argwhere(bad)[:4], got["out"][bad][:4], r["out"][bad][:4], tol[bad][:4])
    if head_slot is None:
        return
    rows, tokens, ah, cols = got["align"].shape
    want = np.full(got["align"].shape, np.nan)
    tol = np.zeros(got["align"].shape)
    for h in reversed(range(len(head_slot))):
        s = head_slot[h]
        if not 0 <= s < ah:
            continue
        p = np.zeros((rows, tokens, cols))
        m = min(cols, r["p"].shape[-1])
        p[..., :m] = r["p"][:, :, h, :m]
        p[gone[:, :, h]] = np.nan
        want[:, :, s] = p
        tol[:, :, s] = ((2 * ds + (n + 16) * U)[:, :, h, None] * p + 2.0 ** -120) * (p > 0)
    left = np.isnan(want)
    assert (got["align"][left] == 7).all()
    bad = ~(np.abs(got["align"] - want) <= tol) & ~left
    assert not bad.any(), (np.argwhere(bad)[:4], got["align"][bad][:4], want[bad][:4], tol[bad][:4])


def cross_case(ctx, dev, seed, rows, tokens, heads, kvh, pos, slots=None, std=1.0, **kw):
    rng = np.random.default_rng(seed)
    q, (k, v) = f16(rng, (rows, tokens, heads, 64), 1.5), (f16(rng, (slots or rows, pos, kvh, 64), std) for _ in range(2))
    got = run_cross(ctx, dev, q, k, v, **kw)
    check_cross(q, k, v, got, **{x: y for x, y in kw.items() if x not in ("align_heads", "align_cols", "work")})
    return got


@pytest.mark.parametrize("pos", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 250, 257, 700, 1500])
@pytest.mark.parametrize("rows,tokens,heads,kvh", [(1, 1, 6, 6), (3, 5, 4, 2), (2, 40, 2, 2)])
def test_cross_lengths(ctx, dev, rows, tokens, heads, kvh, pos):
    cross_case(ctx, dev, pos, rows, tokens, heads, kvh, pos)


@pytest.mark.parametrize("tokens", [1, 2, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 129, 224])
def test_cross_tokens(ctx, dev, tokens):
    cross_case(ctx, dev, tokens, 2, tokens, 3, 3, 333, first=[0, 21], length=[333, 300], count=[tokens, (tokens + 1) // 2])


@pytest.mark.parametrize("heads,kvh,tokens", [(1, 1, 1), (8, 1, 1), (64, 1, 1), (6, 2, 5), (20, 4, 3), (16, 8, 30), (128, 2, 1), (12, 1, 9)])
def test_cross_shared_heads(ctx, dev, heads, kvh, tokens):
    cross_case(ctx, dev, heads, 2, tokens, heads, kvh, 210, length=[210, 77])


@pytest.mark.parametrize("tokens", [1, 6, 40, 130])
def test_cross_rows_that_see_little_or_nothing(ctx, dev, tokens):
    cross_case(ctx, dev, tokens, 9, tokens, 4, 4, 200, slots=4, slot=[0, 1, 2, 3, 4, -1, 0, 3, 1],
               first=[0, 5, 199, 200, 0, 0, -7, 31, 90], length=[0, 6, 200, 500, 9, 9, 1, 64, 50],
               count=[tokens, 99999, tokens, tokens, tokens, tokens, 0, -3, tokens])


@pytest.mark.parametrize("tokens", [1, 24, 130])
@pytest.mark.parametrize("rows,heads", [(1, 2), (14, 20)])
def test_cross_what_is_not_seen_is_not_looked_at(ctx, dev, tokens, rows, heads):
    rng = np.random.default_rng(2)
    q = f16(rng, (rows, tokens, heads, 64), 1.5)
    k, v = (f16(rng, (rows, 150, heads, 64)) for _ in range(2))
    first, length = [13] * rows, [101] * rows
    kw = dict(first=first, length=length)
    clean = run_cross(ctx, dev, q, k, v, **kw)
    for x, bad in ((k, np.nan), (v, np.inf)):
        x[:, :13], x[:, 101:] = bad, -bad
    got = run_cross(ctx, dev, q, k, v, **kw)
    np.testing.assert_array_equal(got["out"], clean["out"])
    np.testing.assert_array_equal(got["lse"], clean["lse"])


def test_cross_a_row_that_is_no_number_stays_alone(ctx, dev):
    rng = np.random.default_rng(6)
    for tokens in (1, 3, 40):
        q = f16(rng, (3, tokens, 4, 64), 1.5)
        k, v = (f16(rng, (3, 90, 4, 64)) for _ in range(2))
        q[0, tokens - 1, 1, 5], k[1, 40, 2, 0], v[2, 89, 3, 9] = np.nan, np.nan, np.nan
        got = run_cross(ctx, dev, q, k, v)
        bad = np.zeros((3, tokens, 4, 64), bool)
        bad[0, tokens - 1, 1] = bad[1, :, 2] = bad[2, :, 3, 9] = True
        np.testing.assert_array_equal(np.isnan(got["out"]), bad)


@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("scale,size", [(0.125, 30.0), (8.0, 1.0), (0.001, 1.0), (1.0, 0.01), (1048576.0, 0.5)])
def test_cross_sharp_and_flat_rows(ctx, dev, tokens, scale, size):
    rng = np.random.default_rng(8)
    q, k, v = f16(rng, (2, tokens, 2, 64), size), f16(rng, (2, 400, 2, 64), size), f16(rng, (2, 400, 2, 64), 100.0)
    got = run_cross(ctx, dev, q, k, v, scale=scale)
    if scale < 1000:
        check_cross(q, k, v, got, scale=scale)
    else:  # one position takes all of it
        x = np.einsum("rthd,rphd->rthp", q.astype(np.float64), k.astype(np.float64))
        top = x.argmax(-1)
        second = np.sort(x, -1)[..., -2]
        sure = x.max(-1) - second > 0.01
        want = np.stack([[[v[r, top[r, i, h], h] for h in range(2)] for i in range(tokens)] for r in range(2)])
        np.testing.assert_array_equal(got["out"][sure], want[sure])


@pytest.mark.parametrize("tokens", [1, 40])
def test_cross_a_long_tail_far_below_the_peak(ctx, dev, tokens):
    """1,499 positions 2^-18 each of one: 0.57% of the sum, which is not lost, with values that only they have."""
    q = np.zeros((1, tokens, 1, 64), np.float16)
    q[..., 0] = 8.0
    k = np.zeros((1, 1500, 1, 64), np.float16)
    v = np.zeros((1, 1500, 1, 64), np.float16)
    k[0, 700, 0, 0] = 12.4766  # 8 * 12.4766 / 8 = 18 ln 2
    v[0, :, 0, 1] = 100.0
    v[0, 700, 0, 1] = 0.0
    got = run_cross(ctx, dev, q, k, v)
    check_cross(q, k, v, got)
    r = R.cross(q, k, v)["out"][..., 1]
    assert (np.abs(got["out"][..., 1] / r - 1) < 2.0 ** -10).all() and 0.5 < r[0, 0, 0] < 0.6


@pytest.mark.parametrize("pos", [40, 65, 300, 1500])
@pytest.mark.parametrize("rows,tokens,heads,kvh", [(1, 1, 6, 6), (3, 1, 20, 20), (2, 5, 4, 2), (2, 33, 4, 4), (40, 1, 20, 20), (1, 100, 2, 2)])
def test_cross_alignment_rows(ctx, dev, rows, tokens, heads, kvh, pos):
    head_slot = [[-1, 3, 0, 3, 9, 1][h % 6] if h < 12 else -1 for h in range(heads)]
    length = [pos - (7 * i) % (pos // 2) for i in range(rows)]
    cross_case(ctx, dev, pos, rows, tokens, heads, kvh, pos, length=length, first=[(3 * i) % 9 for i in range(rows)],
               count=[tokens - (i % 2) * (tokens // 2) for i in range(rows)], head_slot=head_slot, align_heads=4,
               align_cols=pos + (3 if rows == 2 else -5))


@pytest.mark.parametrize("rows,heads,tokens,pos", [(8, 20, 100, 150), (30, 20, 1, 130), (13, 20, 3, 90), (64, 20, 1, 64), (2, 20, 224, 700),
                                                   (2, 8, 1, 16000), (1, 4, 3, 9001), (1, 16, 90, 4000), (300, 6, 2, 33)])
def test_cross_many_rows_and_long_sequences(ctx, dev, rows, heads, tokens, pos):
    length = [max(1, pos - 11 * (i % 12)) for i in range(rows)]
    cross_case(ctx, dev, rows, rows, tokens, heads, heads, pos, length=length)


def test_cross_layouts(ctx, dev):
    """The engine's tiles, rows of a fused product, queries and outputs head by head: the same bits as the dense form."""
    rng = np.random.default_rng(4)
    for tokens in (1, 30):
        rows, heads, pos = 3, 4, 90
        q = f16(rng, (rows, tokens, heads, 64), 1.5)
        k, v = (f16(rng, (rows, pos, heads, 64)) for _ in range(2))
        want = run_cross(ctx, dev, q, k, v)
        tiles = np.full((rows, 2, 2, heads, 96, 64), np.nan, np.float16)  # layer 1 of two
        tiles[:, 1, 0, :, :pos], tiles[:, 1, 1, :, :pos] = k.transpose(0, 2, 1, 3), v.transpose(0, 2, 1, 3)
        fused = np.stack([k, v], 2)  # [row][t][2][head][64]
        t, f = dev(tiles), dev(fused)
        ts, fs = (4 * heads * 96 * 64, 64, 96 * 64), (pos * 2 * heads * 64, 2 * heads * 64, 64)
        qt = dev(q.transpose(2, 0, 1, 3))  # [head][row][token]
        by_head = (tokens * 64, 64, rows * tokens * 64)
        for ks, vs, kat, vat in ((ts, ts, t + 2 * 2 * heads * 96 * 64, t + 2 * 3 * heads * 96 * 64), (fs, fs, f, f + 2 * heads * 64),
                                 (ts, fs, t + 2 * 2 * heads * 96 * 64, f + 2 * heads * 64)):
            out = dev(np.zeros((heads, rows, tokens, 64), np.float16))
            steps.cross_attention(ctx, qt, out, kat, vat, rows, tokens, heads, pos, k_strides=ks, v_strides=vs, q_strides=by_head,
                                  out_strides=by_head)
            got = ctx.download(out, (heads, rows, tokens, 64), np.float16).transpose(1, 2, 0, 3)
            np.testing.assert_array_equal(got, want["out"])


def test_cross_past_32_bits(ctx, dev):
    """Positions and slots whose offsets pass 2^32 bytes."""
    rng = np.random.default_rng(9)
    pos, heads, far = 140, 2, 1 << 24  # positions 2^25 bytes apart: 4.4 GiB
    k, v, q = f16(rng, (1, pos, heads, 64)), f16(rng, (1, pos, heads, 64)), f16(rng, (1, 1, heads, 64), 1.5)
    base = ctx.alloc(pos * far * 2 + 4096)
    try:
        for p in range(pos):
            ctx.upload(base + p * far * 2, np.concatenate([k[0, p].reshape(-1), v[0, p].reshape(-1)]))
        for tokens in (1, 20):
            qq = np.repeat(q, tokens, 1)
            out, lse = dev(np.full(qq.shape, 3, np.float16)), dev(np.full(qq.shape[:3], 5, np.float32))
            steps.cross_attention(ctx, dev(qq), out, base, base + 2 * heads * 64, 1, tokens, heads, pos,
                                  k_strides=(0, far, 64), lse=lse)
            check_cross(qq, k, v, {"out": ctx.download(out, qq.shape, np.float16), "lse": ctx.download(lse, qq.shape[:3], np.float32)})
    finally:
        ctx.free(base)


# ---------------------------------------------------------------- the next token


def logits(rng, n, v, dtype, spread=2.5, likely=12):
    x = rng.standard_normal((n, v), dtype=np.float32) * spread
    for r in range(n):
        x[r, rng.integers(0, v, likely)] += rng.random(likely, dtype=np.float32) * 16
    return x.astype(dtype)


def run_sample(ctx, dev, x, u, mask=None, pad=0, off=0, **kw):
    n, v = x.shape
    full = np.full((n, v + pad), 99, x.dtype)
    full[:, :v] = x
    flat = np.concatenate([np.zeros(off, x.dtype), full.reshape(-1)])
    arrays = {name: dev((i32 if name == "top_ks" else f32)(kw.pop(name))) for name in ("temperatures", "top_ks", "top_ps", "min_ps")
              if kw.get(name) is not None}
    out = [dev(np.full(n, 77, t)) for t in (np.int32, np.float32, np.int32)]
    steps.sample(ctx, dev(flat) + off * x.itemsize, n, v, dev(f32(u)), out[0], L.DT_F16 if x.dtype == np.float16 else L.DT_F32,
                 v + pad, dev(mask), logp=out[1], kept=out[2], **arrays, **kw)
    return [ctx.download(p, (n,), t) for p, t in zip(out, (np.int32, np.float32, np.int32))]


SETTINGS = [("temperature", "temperatures", 1.0), ("top_k", "top_ks", 0), ("top_p", "top_ps", 1.0), ("min_p", "min_ps", 0.0)]


def check_sample(x, u, got, mask=None, **kw):
    """Returns how many rows had a sum too near to a border to tell."""
    unsure = 0
    for r in range(len(x)):
        t, k, p, m = (kw[each][r] if kw.get(each) is not None else kw.get(name, usual) for name, each, usual in SETTINGS)
        tok, logp, kept, near = R.sample(x[r], np.float32(u[r]), np.float32(t), int(k), np.float32(p), np.float32(m), mask)
        if near < 1e-11:
            unsure += 1
            continue
        assert (got[0][r], got[2][r]) == (tok, kept), (r, got[0][r], tok, got[2][r], kept, near)
        if np.isfinite(logp):
            assert abs(got[1][r] - logp) <= U * abs(logp) + 2.0 ** -40, (r, got[1][r], logp)
        else:
            np.testing.assert_array_equal(got[1][r], np.float32(logp))
    return unsure


LIMITS = [dict(), dict(temperature=0.0), dict(temperature=0.3), dict(temperature=3.0), dict(top_k=1), dict(top_k=7), dict(top_k=300),
          dict(top_p=0.9), dict(top_p=0.3, temperature=1.5), dict(top_p=0.0), dict(min_p=0.05), dict(min_p=1.0),
          dict(top_p=0.999, temperature=2.0), dict(top_k=50, top_p=0.95, min_p=0.02, temperature=0.8), dict(top_k=5000, top_p=0.8, temperature=4.0)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 1025, 4097, 51865])
@pytest.mark.parametrize("limits", LIMITS, ids=lambda d: "-".join(f"{k}{v}" for k, v in d.items()) or "none")
def test_sample(ctx, dev, dtype, vocab, limits):
    rng = np.random.default_rng(vocab)
    n = 6
    x, u = logits(rng, n, vocab, dtype), rng.random(n, dtype=np.float32)
    mask = (rng.random(vocab) < 0.1).astype(np.uint8) if vocab > 60 and vocab % 2 else None
    got = run_sample(ctx, dev, x, u, mask, pad=vocab % 3, off=vocab % 4, **limits)
    assert check_sample(x, u, got, mask, **limits) == 0


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,vocab", [(40, 51866), (300, 5000), (700, 700)])
def test_sample_of_many_rows_with_settings_of_their_own(ctx, dev, dtype, rows, vocab):
    rng = np.random.default_rng(rows)
    x, u = logits(rng, rows, vocab, dtype), rng.random(rows, dtype=np.float32)
    pick = lambda *v: np.array([v[i % len(v)] for i in range(rows)])  # noqa: E731
    kw = dict(temperatures=pick(0.0, 0.2, 0.7, 1.0, 1.3, 5.0, 50.0), top_ks=pick(0, 1, 40, -3, 400, vocab, vocab + 9), top_ps=pick(1.0, 0.9, 0.5, 2.0),
              min_ps=pick(0.0, 0.0, 0.05, -1.0, 0.0))
    got = run_sample(ctx, dev, x, u, **kw)
    assert check_sample(x, u, got, **kw) <= 1
    again = run_sample(ctx, dev, x, u, **kw)
    for a, b in zip(got, again):
        np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("vocab", [300000, 60000])
@pytest.mark.parametrize("limits", [dict(), dict(top_k=900, temperature=2.0), dict(top_p=0.97, temperature=2.0), dict(min_p=0.01)], ids=str)
def test_sample_of_large_vocabularies(ctx, dev, vocab, limits):
    rng = np.random.default_rng(1)
    x, u = logits(rng, 3, vocab, np.float32), rng.random(3, dtype=np.float32)
    assert check_sample(x, u, run_sample(ctx, dev, x, u, **limits), **limits) == 0


@pytest.mark.parametrize("vocab", [50, 3000, 51865])
@pytest.mark.parametrize("limits", [dict(), dict(top_k=3), dict(top_k=40), dict(top_p=0.5), dict(min_p=0.5), dict(top_p=0.77, top_k=41),
                                    dict(temperature=0.0)], ids=str)
def test_sample_of_equal_logits(ctx, dev, vocab, limits):
    """Ties: everything, two values, few values, zeros of either sign."""
    rng = np.random.default_rng(2)
    x = np.zeros((6, vocab), np.float32)
    x[1] = rng.integers(0, 2, vocab)
    x[2] = rng.integers(-3, 4, vocab)
    x[3, ::2] = -0.0
    x[4] = -np.inf
    x[4, [7, 30, 41]] = -1.5
    x[5, 1:] = -3.0e38
    u = np.array([0.37, 0.81, 0.11, 0.73, 0.9, 0.5], np.float32)
    got = run_sample(ctx, dev, x, u, **limits)
    # sums of whole weights are exact: also where a limit is met exactly
    for r in range(6):
        tok, logp, kept, near = R.sample(x[r], u[r], np.float32(limits.get("temperature", 1.0)), limits.get("top_k", 0), np.float32(limits.get("top_p", 1.0)),
                                         np.float32(limits.get("min_p", 0.0)))
        if near < 1e-11 and r in (1, 2):
            continue
        assert (got[0][r], got[2][r]) == (tok, kept), (r, got[0][r], tok, got[2][r], kept, near)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("vocab", [70, 51866])
def test_sample_of_unusual_rows(ctx, dev, dtype, vocab):
    rng = np.random.default_rng(3)
    x = logits(rng, 14, vocab, dtype)
    mask = np.zeros(vocab, np.uint8)
    mask[[3, vocab - 1]] = 1, 255
    x[0, 5] = np.nan
    x[1, vocab - 2] = np.inf
    x[2] = -np.inf
    x[3, 3], x[3, vocab - 1] = np.nan, np.inf  # masked
    x[4] = -np.inf
    x[4, 3] = 4.0  # only a masked one left
    x[5, :] = -np.inf
    x[5, vocab - 3] = -60000.0
    x[6, 9] = 60000.0  # sure
    t = np.array([1, 1, 1, 1, 1, 1, 1, -1, np.nan, np.inf, 1, 1, 1e-30, 1e30])
    p = np.array([1, 1, 1, .9, 1, .9, .9, 1, 1, 1, np.nan, 1, .9, .9])
    m = np.array([0, 0, 0, 0, 0, .1, 0, 0, 0, 0, 0, np.nan, 0, .5])
    u = np.array([.5, .5, .5, .5, .5, .5, .5, .5, .5, .5, .5, .5, np.nan, 7.0], np.float32)
    kw = dict(temperatures=t, top_ps=p, min_ps=m)
    got = run_sample(ctx, dev, x, u, mask, **kw)
    assert check_sample(x, u, got, mask, **kw) == 0
    assert (got[0][[0, 1, 2, 4, 7, 8, 9, 10, 11]] == -1).all() and (got[2][[0, 1, 2, 4, 7, 8, 9, 10, 11]] == 0).all()
    assert got[0][5] == vocab - 3 and got[0][6] == 9


@pytest.mark.parametrize("limits", [dict(), dict(top_p=0.8), dict(top_k=20)], ids=str)
def test_sample_follows_the_distribution(ctx, dev, limits):
    """Evenly spread numbers u draw each token in its share: the counts are within one of it."""
    rng = np.random.default_rng(4)
    n, v = 4000, 500
    x = np.repeat(logits(rng, 1, v, np.float32, 1.0, 3), n, 0)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = run_sample(ctx, dev, x, u, **limits)
    assert (np.diff(got[0]) >= 0).all()  # in the order of ids
    w = np.exp(x[0].astype(np.float64) - x[0].max())
    order = np.argsort(-x[0], kind="stable")
    keep = got[2][0]
    share = np.zeros(v)
    share[order[:keep]] = w[order[:keep]] / w[order[:keep]].sum()
    assert (np.abs(np.bincount(got[0], minlength=v) - n * share) <= 1.001).all()


def test_sample_at_a_step(ctx, dev):
    """Random numbers, tokens, log probabilities and counts beside those of other steps; rows out of range write nothing."""
    rng = np.random.default_rng(5)
    n, v, st = 5, 900, 7
    x, u = logits(rng, n, v, np.float32), rng.random((n, st), dtype=np.float32)
    at = dev(i32([3]))
    d = dev(x), dev(u)
    for add, col in ((0, 3), (2, 5), (-3, 0), (3, 6), (4, None), (-4, None)):
        out = [dev(np.full((n, st), 77, t)) for t in (np.int32, np.float32, np.int32)]
        steps.sample(ctx, d[0], n, v, d[1], out[0], logp=out[1], kept=out[2], stride=st, at=at, at_add=add, top_p=0.9)
        got = [ctx.download(p, (n, st), t) for p, t in zip(out, (np.int32, np.float32, np.int32))]
        for g in got:
            rest = np.delete(g, col, 1) if col is not None else g
            assert (rest == 77).all()
        if col is not None:
            assert check_sample(x, u[:, col], [g[:, col] for g in got], top_p=0.9) == 0
    tok = dev(np.full(n, 77, np.int32))
    steps.sample(ctx, d[0], n, v, dev(u[:, 0]), tok, top_p=0.9)  # nothing else wanted
    np.testing.assert_array_equal(ctx.download(tok, (n,), np.int32), [R.sample(x[r], u[r, 0], top_p=np.float32(0.9))[0] for r in range(n)])


# ---------------------------------------------------------------- together


def test_a_captured_decoding_step(ctx, dev):
    """A small decoder's cross-attention block, feed-forward block and logits with 4-bit weights, and the next token, captured
    once and replayed for several steps with work of other kinds between: each step equals the same calls made eagerly, and
    the eager ones the oracle fed with the device's inputs of each call."""
    rng = np.random.default_rng(11)
    rows, heads, d, ff, v, pos, n_steps, group = 4, 6, 384, 1536, 5000, 300, 6, 64
    wq, wo, w1, w2, wv = (f16(rng, s, s[1] ** -0.5) for s in ((d, d), (d, d), (ff, d), (d, ff), (v, d)))
    W = [packed(ctx, dev, w, group) for w in (wq, wo, w1, w2, wv)]
    bq, b1 = f16(rng, (d,), 0.1), f16(rng, (ff,), 0.1)
    k, ev = (f16(rng, (rows, pos, heads, 64)) for _ in range(2))
    length = [300, 120, 1, 0]
    emb, u = f16(rng, (v, d), 1.0), rng.random((rows, n_steps), dtype=np.float32)
    temps = f32([0.0, 0.7, 1.0, 1.3])
    mask = (rng.random(v) < 0.02).astype(np.uint8)
    D = {name: dev(a) for name, a in dict(bq=bq, b1=b1, k=k, v=ev, len=i32(length), u=u, t=temps, mask=mask).items()}
    buf = lambda shape, t: dev(np.zeros(shape, t))  # noqa: E731

    def buffers():
        return dict(h=buf((rows, d), np.float16), q=buf((rows, d), np.float16), o=buf((rows, d), np.float16),
                    x=buf((rows, d), np.float32), f=buf((rows, ff), np.float16), g=buf((rows, d), np.float16),
                    logits=buf((rows, v), np.float32), tok=buf((rows, n_steps), np.int32), logp=buf((rows, n_steps), np.float32),
                    kept=buf((rows, n_steps), np.int32), ctr=buf((1,), np.int32))

    def step(b):
        W[0].linear(b["h"], b["q"], rows, L.EPI_F16, D["bq"])
        steps.cross_attention(ctx, b["q"], b["o"], D["k"], D["v"], rows, 1, heads, pos, k_strides=(pos * d, d, 64), len=D["len"])
        W[1].linear(b["o"], b["x"], rows, L.EPI_RESID_F32)
        W[2].linear(b["o"], b["f"], rows, L.EPI_GELU_F16, D["b1"])
        W[3].linear(b["f"], b["g"], rows, L.EPI_F16)
        W[4].linear(b["g"], b["logits"], rows, L.EPI_F32)
        steps.sample(ctx, b["logits"], rows, v, D["u"], b["tok"], mask=D["mask"], temperatures=D["t"], top_p=0.9, top_k=200, logp=b["logp"],
                     kept=b["kept"], stride=n_steps, at=b["ctr"])

    def begin(b, i, tokens):
        ctx.upload(b["ctr"], i32([i]))
        ctx.upload(b["h"], emb[tokens])

    eager, graph = buffers(), buffers()
    begin(eager, 0, [0] * rows)
    step(eager)  # the workspace is there before the capture
    ctx.upload(eager["x"], np.zeros((rows, d), np.float32))
    g = C.c_void_p()
    L.check(L.lib().mz_graph_begin(ctx.h))
    step(graph)
    L.check(L.lib().mz_graph_end(ctx.h, C.byref(g)))
    tokens = [1, 2, 3, 4]
    for i in range(n_steps):
        for b in (eager, graph):
            begin(b, i, tokens)
        step(eager)
        L.check(L.lib().mz_graph_launch(ctx.h, g))
        for name, shape, t in (("x", (rows, d), np.float32), ("logits", (rows, v), np.float32), ("tok", (rows, n_steps), np.int32),
                               ("logp", (rows, n_steps), np.float32), ("kept", (rows, n_steps), np.int32)):
            np.testing.assert_array_equal(ctx.download(graph[name], shape, t), ctx.download(eager[name], shape, t), err_msg=f"{name} {i}")
        get = lambda name, shape, t=np.float16: ctx.download(eager[name], shape, t)  # noqa: E731
        val = lambda w: R.w4_values(*R.w4_codes(w, group), group)  # noqa: E731
        q, o = get("q", (rows, d)), get("o", (rows, d))
        check_linear(emb[tokens], val(wq), bq, L.EPI_F16, q)
        r = R.cross(q.reshape(rows, 1, heads, 64), k, ev, length=length)
        assert np.abs(o - r["out"].reshape(rows, d)).max() <= 2 * H * np.abs(ev).max()
        check_linear(o, val(w1), b1, L.EPI_GELU_F16, get("f", (rows, ff)))
        check_linear(get("f", (rows, ff)), val(w2), None, L.EPI_F16, get("g", (rows, d)))
        x = get("logits", (rows, v), np.float32)
        check_linear(get("g", (rows, d)), val(wv), None, L.EPI_F32, x)
        got = [get(name, (rows, n_steps), t)[:, i] for name, t in (("tok", np.int32), ("logp", np.float32), ("kept", np.int32))]
        check_sample(x, u[:, i], got, mask, temperatures=temps, top_p=0.9, top_k=200)
        tokens = got[0].tolist()
    L.check(L.lib().mz_graph_free(g))


# ---------------------------------------------------------------- limits of the choices between variants


@pytest.mark.parametrize("m,n,k,group", [(1000, 5129, 128, 64), (1800, 5100, 128, 128), (1025, 4099, 256, 32), (700, 2050, 128, 64),
                                         (448, 5121, 128, 128), (385, 6150, 256, 64), (4097, 1281, 128, 32), (100, 8200, 128, 64),
                                         (65, 16384, 128, 128), (2049, 513, 128, 32), (65, 30000, 128, 32), (31, 17000, 256, 64)])
@pytest.mark.parametrize("epilogue", [L.EPI_RESID_F32, L.EPI_GELU_F16])
def test_w4_linear_in_tiles(ctx, dev, epilogue, m, n, k, group):
    """Numbers of rows of either side that fill tiles of every width and leave their last ones ragged; as many workgroups as there
    are CUs, some more, and several times as many."""
    rng = np.random.default_rng(m + n)
    w, x, bias = f16(rng, (n, k), k ** -0.5), f16(rng, (m, k), 1.0), f16(rng, (n,), 0.3)
    got, before = run_linear(ctx, dev, packed(ctx, dev, w, group), x, bias, epilogue, ldo=n + 1)
    check_linear(x, R.w4_values(*R.w4_codes(w, group), group), bias, epilogue, got, before if epilogue == L.EPI_RESID_F32 else None)


@pytest.mark.parametrize("rows,tokens,heads,pos", [(4, 64, 64, 40), (4, 65, 64, 70), (8, 200, 34, 33), (5, 250, 64, 65), (20, 129, 64, 31),
                                                   (40, 128, 33, 40), (33, 64, 40, 5), (1, 17, 256, 96), (129, 1, 1, 400), (257, 16, 1, 161)])
def test_cross_where_the_card_fills(ctx, dev, rows, tokens, heads, pos):
    """As many groups of queries as there are CUs, some more, and several times as many; rows of unequal lengths, none among them."""
    length = [(pos * (1 + 7 * r % 11)) // 11 for r in range(rows)]
    length[rows // 2] = 0
    cross_case(ctx, dev, rows + tokens, rows, tokens, heads, heads, pos, length=length, count=[tokens - (r % 3 == 2) * (tokens // 2) for r in range(rows)])


def test_cross_rows_that_share_a_slot(ctx, dev):
    """The same slot for every row, seen from other places each, is as good as slots of their own; every call again is bit for bit
    the same."""
    rng = np.random.default_rng(21)
    rows, heads, pos = 9, 6, 700
    k, v = (f16(rng, (2, pos, heads, 64)) for _ in range(2))
    for tokens in (1, 20, 300):
        q = f16(rng, (rows, tokens, heads, 64), 1.5)
        kw = dict(slot=[1] * rows, first=[0, 5, 31, 32, 33, 200, 699, 0, 700], length=[700, 6, 700, 33, 100, 700, 700, 1, 700])
        got = run_cross(ctx, dev, q, k, v, **kw)
        check_cross(q, k, v, got, **kw)
        again = run_cross(ctx, dev, q, k, v, **kw)
        for name in got:
            np.testing.assert_array_equal(got[name], again[name])


@pytest.mark.parametrize("vocab", [30000, 51866])
@pytest.mark.parametrize("temperature", [0.05, 1.0, 3.0])
@pytest.mark.parametrize("top_k", [0, 65, 512, 513, 1000, 1024, 1025, 2000, 20000])
def test_sample_where_long_lists_end(ctx, dev, vocab, temperature, top_k):
    rng = np.random.default_rng(top_k + vocab)
    n = 9
    x, u = logits(rng, n, vocab, np.float32), rng.random(n, dtype=np.float32)
    kw = dict(temperature=temperature, top_k=top_k, top_ps=f32([1, .999, .97, .9, .7, .5, .3, .05, .9999]), min_ps=f32([0, 0, 0, .001, 0, 0, 1e-6, 0, 1e-9]))
    assert check_sample(x, u, run_sample(ctx, dev, x, u, **dict(kw)), **kw) <= 1


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("values", [[0.0], [0.0, -1.0], [3.0, 2.5, -7.0], [-0.0, 0.0, 2.0 ** -20], [1.0, -60000.0]], ids=str)
@pytest.mark.parametrize("limits", [dict(), dict(top_k=1500), dict(top_p=0.5), dict(top_k=1025, top_p=0.9), dict(top_p=0.999, temperature=5.0),
                                    dict(min_p=0.3), dict(top_k=1023, min_p=0.5, top_p=0.25)], ids=str)
def test_sample_of_more_equal_logits_than_a_list_holds(ctx, dev, dtype, values, limits):
    rng = np.random.default_rng(len(values))
    x = rng.choice(np.array(values, np.float64), (4, 20011)).astype(dtype)
    u = np.array([0.0, 0.3, 0.777, 1.0 - 2.0 ** -24], np.float32)
    got = run_sample(ctx, dev, x, u, **limits)
    assert check_sample(x, u, got, **limits) <= 2  # (where all weights but equal ones are 0, sums end on borders)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("t", [1e-44, 0.01, 1.0, 1e6, 1e38])
def test_sample_of_lowest_logits(ctx, dev, dtype, t):
    """The type's lowest number is a logit like others: rows of nothing else, rows that have it instead of a mask, rows with one
    or two tokens above it; so is its least one, next to zeros."""
    low = np.finfo(dtype).min
    rng = np.random.default_rng(4)
    x = np.full((7, 3001), low, dtype)
    x[1, 5:] = rng.standard_normal(2996).astype(dtype)
    x[2, 2999] = 0
    x[3, [7, 8]] = 0.5, 0.25
    x[4, ::2] = -np.inf
    x[5, :] = np.finfo(dtype).max
    x[5, ::3] = low
    x[6] = -np.finfo(dtype).smallest_subnormal
    x[6, ::2] = 0
    u = np.array([.1, .3, .5, .7, .9, .37, .61], np.float32)
    for limits in (dict(), dict(top_p=0.9), dict(top_k=30), dict(min_p=0.1)):
        kw = dict(temperature=np.float32(t), **limits)
        check_sample(x, u, run_sample(ctx, dev, x, u, **kw), **kw)


def test_contexts_at_once(ctx):
    """Contexts of two threads, each with its own stream and workspace, while both are at work: the results of one alone."""
    import threading
    rng = np.random.default_rng(8)
    heads, pos, n, k, v = 6, 1500, 500, 256, 20000
    w, x = f16(rng, (n, k), 0.1), f16(rng, (9, k))
    q, (ek, ev) = f16(rng, (2, 1, heads, 64), 1.5), (f16(rng, (2, pos, heads, 64)) for _ in range(2))
    lg, u = logits(rng, 8, v, np.float32), rng.random(8, dtype=np.float32)

    def work(c, times):
        d, out = Dev(c), []
        try:
            p = packed(c, d, w, 32)
            for _ in range(times):
                lin, _ = run_linear(c, d, p, x, None, L.EPI_F32)
                cr = run_cross(c, d, q, ek, ev, length=[1500, 700])
                out.append([lin, cr["out"], cr["lse"], *run_sample(c, d, lg, u, top_p=0.95, top_k=700)])
        finally:
            d.free()
        return out

    want, got = work(ctx, 1)[0], {}

    def thread(i):
        c = model.Context(0)
        try:
            got[i] = work(c, 12)
        finally:
            c.close()

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 2
    for runs in got.values():
        for run in runs:
            for a, b in zip(run, want):
                np.testing.assert_array_equal(a, b)


def test_graphs_that_share_a_workspace(ctx, dev):
    """Two captured calls whose workgroups share rows, and a captured choice of tokens, replayed in turns with eager calls of other
    sizes between: every replay equals the eager result."""
    rng = np.random.default_rng(9)
    heads, pos = 6, 1500
    k, v = (f16(rng, (3, pos, heads, 64)) for _ in range(2))
    D = {"k": dev(k), "v": dev(v), "len": dev(i32([1500, 900, 40]))}
    x, u = logits(rng, 5, 30000, np.float32), rng.random(5, dtype=np.float32)
    dx, du = dev(x), dev(u)

    def attend(rows, tokens, q, out):
        steps.cross_attention(ctx, q, out, D["k"], D["v"], rows, tokens, heads, pos, k_strides=(pos * heads * 64, heads * 64, 64), len=D["len"])

    calls = []
    for rows, tokens in ((1, 1), (3, 12)):
        q, shape = dev(f16(rng, (rows, tokens, heads, 64), 1.5)), (rows, tokens, heads, 64)
        calls.append((lambda o, rows=rows, tokens=tokens, q=q: attend(rows, tokens, q, o), shape, np.float16))
    calls.append((lambda o: steps.sample(ctx, dx, 5, 30000, du, o, top_k=600, top_p=0.9), (5,), np.int32))
    want, outs, graphs = [], [], []
    for f, shape, t in calls:
        o = dev(np.zeros(shape, t))
        f(o)
        want.append(ctx.download(o, shape, t))
    for f, shape, t in calls:
        outs.append(dev(np.zeros(shape, t)))
        g = C.c_void_p()
        L.check(L.lib().mz_graph_begin(ctx.h))
        f(outs[-1])
        L.check(L.lib().mz_graph_end(ctx.h, C.byref(g)))
        graphs.append(g)
    other = dev(np.zeros((2, 1, heads, 64), np.float16))
    oq = dev(f16(rng, (2, 1, heads, 64)))
    for i in range(6):
        for j in ((0, 1, 2), (2, 1, 0), (1, 0, 2))[i % 3]:
            ctx.upload(outs[j], np.zeros(calls[j][1], calls[j][2]))
            L.check(L.lib().mz_graph_launch(ctx.h, graphs[j]))
            if i % 2:
                attend(2, 1, oq, other)
        for (f, shape, t), o, w in zip(calls, outs, want):
            np.testing.assert_array_equal(ctx.download(o, shape, t), w)
    for g in graphs:
        L.check(L.lib().mz_graph_free(g))


# ---------------------------------------------------------------- where the pieces' largest logits stop lying in LDS


def check_sample_of_all_numbers(x, u, got, **kw):
    """check_sample with a bound that holds for any number of tokens; returns how many rows were too near to a border to tell.

    n tokens as multiples of 2^-s, s = min(51, 62 - ceil(log2 n)), are off by n 2^-(s + 1) at most, and by 2e-12 of each weight. The
    sum is 1 or more (the largest weight is 1), so its logarithm is off by no more than that, and no limit or share whose border
    is farther away than twice that falls on the other side: 2^-25.9 for 2^18 tokens. The logarithm is compared in 64 bits (a
    difference of a numpy float32 and a Python float is one of 32 bits: it rounds the oracle's to a neighbour first)."""
    unsure, n = 0, x.shape[1]
    off = n * 2.0 ** (-1 - min(51, 62 - int(np.ceil(np.log2(n))))) + 4e-12
    for r in range(len(x)):
        t, k, p, m = (kw[each][r] if kw.get(each) is not None else kw.get(name, usual) for name, each, usual in SETTINGS)
        tok, logp, kept, near = R.sample(x[r], np.float32(u[r]), np.float32(t), int(k), np.float32(p), np.float32(m))
        if near < 2 * off:
            unsure += 1
            continue
        assert (got[0][r], got[2][r]) == (tok, kept), (r, got[0][r], tok, got[2][r], kept, near)
        assert got[1][r] == logp if np.isinf(logp) else abs(float(got[1][r]) - logp) <= U * abs(logp) + off, (r, got[1][r], logp, off)
    return unsure


@pytest.mark.parametrize("dtype,vocabs", [(np.float32, range(122876, 122885)), (np.float16, range(245752, 245765))], ids=["f32", "f16"])
@pytest.mark.parametrize("limits", [dict(), dict(temperature=0.0), dict(top_k=40, temperature=0.8), dict(top_p=0.9, temperature=0.6), dict(min_p=0.05),
                                    dict(top_k=700, top_p=0.95, temperature=1.5)], ids=str)
def test_sample_at_the_most_pieces_with_a_word(ctx, dev, dtype, vocabs, limits):
    """Lengths on either side of 30 pieces a thread, rows that begin at every offset from 16 bytes; largest logits above 0."""
    per = 16 // np.dtype(dtype).itemsize
    for vocab in vocabs:
        rng = np.random.default_rng(vocab)
        x, u = logits(rng, per, vocab, dtype), rng.random(per, dtype=np.float32)
        assert (x.max(1) > 0).all()
        for pad in {1 - vocab % 2, 0}:  # rows an odd number of elements apart; all at the same offset, where vocab is even
            got = run_sample(ctx, dev, x, u, pad=pad, **limits)
            assert check_sample_of_all_numbers(x, u, got, **limits) <= 1


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("limits", [dict(), dict(top_k=3), dict(top_k=3000, top_p=0.9), dict(top_p=0.5, temperature=4.0)], ids=str)
@pytest.mark.parametrize("vocab", [60, 20011])
def test_sample_of_a_share_that_no_token_has(ctx, dev, dtype, vocab, limits):
    """min_p above 1 keeps the first of several largest logits, min_p 1 all of them: a row's own and for all rows."""
    rng = np.random.default_rng(vocab)
    x = rng.choice(np.array([0.0, 2.0, 1.0]), (6, vocab)).astype(dtype)
    x[4:, 3::7] = 2.0
    x[5, ::2] = -np.inf
    u = np.array([0.0, 0.4, 0.6, 0.8, 0.99, 0.7], np.float32)
    above = np.nextafter(np.float32(1), np.float32(2))
    kw = dict(min_ps=f32([above, 2.0, 1.0, np.inf, above, 1e30]), **limits)
    got = run_sample(ctx, dev, x, u, **dict(kw))
    assert check_sample(x, u, got, **kw) == 0
    alone = [0, 1, 3, 4, 5]
    assert (got[2][alone] == 1).all() and (got[1][alone] == 0).all() and (got[0][alone] == x.argmax(1)[alone]).all()
    assert got[2][2] > 1
    kw = dict(min_p=3.0, **limits)
    got = run_sample(ctx, dev, x, u, **kw)
    assert check_sample(x, u, got, **kw) == 0 and (got[0] == x.argmax(1)).all() and (got[2] == 1).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("t", [1e-44, 0.01, 1.0, 1e6, 1e38])
def test_sample_of_lowest_logits_row_by_row(ctx, dev, dtype, t):
    """Rows of the type's lowest number and of its least one: every row is far enough from a border to tell, but one."""
    low = np.finfo(dtype).min
    rng = np.random.default_rng(12)
    x = np.full((7, 3001), low, dtype)
    x[1, 5:] = rng.standard_normal(2996).astype(dtype)
    x[2, 2999] = 0
    x[3, [7, 8]] = 0.5, 0.25
    x[4, ::2] = -np.inf
    x[5, :] = np.finfo(dtype).max
    x[5, ::3] = low
    x[6] = -np.finfo(dtype).smallest_subnormal
    x[6, ::2] = 0
    u = np.array([.1, .3, .5, .7, .9, .37, .61], np.float32)
    for limits in (dict(), dict(top_p=0.9), dict(top_k=30), dict(min_p=0.1)):
        kw = dict(temperature=np.float32(t), **limits)
        assert check_sample_of_all_numbers(x, u, run_sample(ctx, dev, x, u, **kw), **kw) <= 1


@pytest.mark.parametrize("vocab", [50, 3000, 51865])
@pytest.mark.parametrize("limits", [dict(), dict(top_k=3), dict(top_k=40), dict(top_p=0.45), dict(min_p=0.5), dict(top_p=0.77, top_k=41),
                                    dict(temperature=0.0)], ids=str)
def test_sample_of_equal_logits_all_numbers(ctx, dev, vocab, limits):
    """Ties, their logarithms of shares too."""
    rng = np.random.default_rng(3)
    x = np.zeros((5, vocab), np.float32)
    x[1] = rng.integers(0, 2, vocab)
    x[2] = rng.integers(-3, 4, vocab)
    x[3, ::2] = -0.0
    x[4] = -np.inf
    x[4, [7, 30, 41]] = -1.5
    u = np.array([0.3712, 0.8134, 0.1151, 0.7351, 0.9], np.float32)
    assert check_sample_of_all_numbers(x, u, run_sample(ctx, dev, x, u, **limits), **limits) == 0


@pytest.mark.parametrize("m,k,group", [(3, 5120, 128), (16, 5120, 32), (17, 2560, 64), (32, 2560, 128), (40, 1280, 64), (64, 1280, 32),
                                       (1, 5248, 64), (20, 2688, 32), (64, 1408, 128)])
def test_w4_linear_of_many_rows_as_long_as_lds(ctx, dev, m, k, group):
    """Weights of more than four tiles a CU: rows of x that fill the 160 KB of LDS, and rows that are one entry too long for it."""
    rng = np.random.default_rng(m + k)
    n = 16385
    w, x, bias = f16(rng, (n, k), k ** -0.5), f16(rng, (m, k), 1.0), f16(rng, (n,), 0.3)
    p = packed(ctx, dev, w, group)
    for epilogue in (L.EPI_F32, L.EPI_GELU_F16):
        got, _ = run_linear(ctx, dev, p, x, bias, epilogue)
        check_linear(x, R.w4_values(*R.w4_codes(w, group), group), bias, epilogue, got)
