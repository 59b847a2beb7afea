"""GPU parity of the 8-bit key/value caches, the attention over them and the token scores, through the C ABI, against
oracle/decode8_ref.py (numpy, 64 bits).

What is written and read back is compared bit for bit: codes, scales and open blocks are defined exactly. Tolerances of
the rest count roundings, u = 2^-24 in 32 bits and h = 2^-11 in fp16 (half a step each):
  a score's exponent    (64 products and sums + 16 for the scales, the maximum and exp2) u sum |q k| scale = ds
  lse                   ds + (n + 8) u (a sum of n terms, in any order) + 4 u |lse|
  a probability         relative 2 ds + (n + 16) u, and 2^-120 for those at the bottom of the range
  attention's output    the probabilities' error and h for their rounding, times sum p |v|; h for the output's own; 2^-24
                        for numbers below fp16's normal range, once for the output and once a position for p
  a log probability     4 u |x - m| + relative ((n + 8) u + 6 u min(|x - m|, 104)) of what is summed, below S / (1 + S)
"""
import numpy as np
import pytest

from mimizuku_amd import _lib as L
from mimizuku_amd import decode8, model
from oracle import decode8_ref as R

pytestmark = pytest.mark.gpu
U, H = 2.0 ** -24, 2.0 ** -11
FMT = ["i8", "e4m3"]


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


def f16(rng, shape, scale=0.7):
    return (rng.standard_normal(shape, dtype=np.float32) * scale).astype(np.float16)


class Both:
    """A cache on the device and the same in the oracle."""

    def __init__(self, ctx, slots, heads, max_tokens, fmt):
        self.ctx, self.d, self.r = ctx, decode8.Kv8(ctx, slots, heads, max_tokens, fmt), R.Cache(slots, heads, max_tokens, fmt)

    def write(self, dev, k, v, slot=None, pos=None, count=None, **kw):
        self.r.write(k, v, slot, pos, count)
        self.d.write(dev(k), dev(v), k.shape[0], k.shape[1], slot=dev(i32(slot)), pos=dev(i32(pos)), count=dev(i32(count)), **kw)

    def check(self):
        """The raw arrays, bit for bit (open blocks only where they are open)."""
        r, kv = self.r, self.d.kv
        sh = (r.slots, r.heads)
        op = self.ctx.download(kv.open, sh, np.int32)
        np.testing.assert_array_equal(op, r.open)
        for side, (c, s, o) in enumerate(((kv.k, kv.k_scale, kv.k_open), (kv.v, kv.v_scale, kv.v_open))):
            order = R.value_order if side else (lambda x: x)
            want = R.code_bytes(order(r.code[side]), r.fmt).reshape(sh + (r.blocks, 2048))
            got = self.ctx.download(c, sh + (r.blocks, 2048), np.uint8)
            # (-0 is 0 as a whole number and has a byte of its own in e4m3)
            np.testing.assert_array_equal(got, want, err_msg="kv"[side] + " codes")
            np.testing.assert_array_equal(self.ctx.download(s, sh + (r.blocks,), np.float32), r.scale[side])
            got = self.ctx.download(o, sh + (2048,), np.float16)
            want = order(r.opened[side]).reshape(sh + (2048,))
            # (a position's places in the order of the array)
            place = order(np.broadcast_to(np.arange(32)[:, None], (32, 64))).reshape(-1)
            for a, b in zip(*np.nonzero(op)):
                held = place < self.held(a)
                np.testing.assert_array_equal(got[a, b][held].view(np.uint16), want[a, b][held].view(np.uint16))
        return self

    def held(self, slot):
        return self.end[slot] % 32 if hasattr(self, "end") else 32

    def free(self):
        self.d.free()


# ---------------------------------------------------------------- writing and reading


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("tokens", [1, 2, 31, 32, 33, 64, 65, 200])
def test_write_from_the_start(ctx, dev, fmt, tokens):
    rng = np.random.default_rng(tokens)
    b = Both(ctx, 3, 2, 224, fmt)
    b.end = [tokens] * 3
    b.write(dev, f16(rng, (3, tokens, 2, 64)), f16(rng, (3, tokens, 2, 64), 3.0))
    b.check().free()


@pytest.mark.parametrize("fmt", FMT)
def test_write_in_pieces_is_write_at_once(ctx, dev, fmt):
    """Pieces of every size up to 70, each row at its own position, single tokens among them: after each the raw arrays
    are the oracle's, and what full blocks hold is what one write of everything leaves."""
    rng = np.random.default_rng(5)
    b, whole = Both(ctx, 2, 3, 320, fmt), Both(ctx, 2, 3, 320, fmt)
    k, v = f16(rng, (2, 320, 3, 64)), f16(rng, (2, 320, 3, 64))
    b.end = np.array([0, 0])
    for n in [1, 1, 29, 1, 1, 3, 40, 64, 1, 70, 37]:
        cnt = np.array([n, max(n - 2, 0)])
        kk, vv = np.zeros((2, n, 3, 64), np.float16), np.zeros((2, n, 3, 64), np.float16)
        for r in range(2):
            kk[r, :cnt[r]], vv[r, :cnt[r]] = k[r, b.end[r]:b.end[r] + cnt[r]], v[r, b.end[r]:b.end[r] + cnt[r]]
            kk[r, cnt[r]:] = np.nan  # what is not there is not looked at
        pos, b.end = b.end.copy(), b.end + cnt
        b.write(dev, kk, vv, pos=pos, count=cnt)
        b.check()
    whole.end = b.end
    whole.write(dev, k, v, count=b.end)
    whole.check()
    for side in range(2):
        for r in range(2):
            n = b.end[r] // 32
            np.testing.assert_array_equal(b.r.code[side][r, :, :n], whole.r.code[side][r, :, :n])
    b.free()
    whole.free()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("rows,heads,tokens", [(24, 20, 500), (3, 20, 333)])
def test_write_of_many_blocks(ctx, dev, fmt, rows, heads, tokens):
    """Rows at every place of a block, with one block a wave and with two; read back whole."""
    rng = np.random.default_rng(tokens)
    b = Both(ctx, rows, heads, 640, fmt)
    pos, cnt = [(11 * r) % 35 for r in range(rows)], [tokens - 17 * (r % 7) for r in range(rows)]
    b.end = pos
    b.write(dev, *(f16(rng, (rows, 35, heads, 64)) for _ in "kv"), count=pos)
    b.end = [p + c for p, c in zip(pos, cnt)]
    b.write(dev, *(f16(rng, (rows, tokens, heads, 64)) for _ in "kv"), pos=pos, count=cnt)
    b.check().free()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("back", [5, 32, 33, 50, 63, 64, 70])
def test_write_behind_the_end_opens_a_block_again(ctx, dev, fmt, back):
    rng = np.random.default_rng(back)
    b = Both(ctx, 1, 2, 160, fmt)
    b.end = [100]
    b.write(dev, f16(rng, (1, 100, 2, 64)), f16(rng, (1, 100, 2, 64)))
    b.end = [back + 3]
    b.write(dev, f16(rng, (1, 3, 2, 64)), f16(rng, (1, 3, 2, 64)), pos=[back])
    b.check()
    for _ in range(2):  # the same write again changes nothing
        b.write(dev, *(f16(np.random.default_rng(9), (1, 40, 2, 64)) for _ in "kv"), pos=[back])
        b.end = [back + 40]
        b.check()
    b.free()


def special_blocks():
    """Blocks whose rounding is at its limits: halfway quotients, one magnitude, the smallest and largest numbers."""
    out = [np.zeros((32, 64)), np.full((32, 64), -65504.0), np.full((32, 64), 2.0 ** -24)]
    x = np.zeros((32, 64))
    x.reshape(-1)[:254] = np.arange(-127, 127) + 0.5
    x[-1, -1] = 127.0
    out.append(x)  # every halfway quotient of whole numbers
    g = np.arange(0, 448.5, 0.5)
    x = np.zeros(2048)
    x[:g.size] = g
    x[1000:1000 + 600] = 2.0 ** -10 * np.arange(600)
    x[-1] = 448.0
    out.append(x.reshape(32, 64))  # e4m3: halfway among normals and subnormals
    x = np.full((32, 64), 2.0 ** -24)
    x[3, 7] = 65504.0
    out.append(x)
    rng = np.random.default_rng(2)
    out += [rng.standard_normal((32, 64)) * s for s in (1e-6, 1e-3, 30.0, 9000.0)]
    return np.stack(out).astype(np.float16)


@pytest.mark.parametrize("fmt", FMT)
def test_write_at_the_limits_of_rounding(ctx, dev, fmt):
    x = special_blocks()
    b = Both(ctx, 1, 1, 32 * len(x), fmt)
    b.end = [32 * len(x)]
    b.write(dev, x.reshape(1, -1, 1, 64), -x.reshape(1, -1, 1, 64))
    b.check().free()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_number_that_is_none_makes_its_block_none(ctx, dev, fmt, bad):
    rng = np.random.default_rng(3)
    k = f16(rng, (1, 96, 1, 64))
    k[0, 40, 0, 11] = bad
    b = Both(ctx, 1, 1, 96, fmt)
    b.write(dev, k, f16(rng, (1, 96, 1, 64)))
    b.check()
    out = dev(np.zeros((96, 64), np.float16))
    b.d.read(out, 0, 1, 96)
    got = ctx.download(out, (96, 64), np.float16)
    assert np.isnan(got[32:64]).all() and np.isfinite(got[:32]).all() and np.isfinite(got[64:]).all()
    b.free()


def test_rows_outside_the_cache_write_nothing(ctx, dev):
    """Slots and positions outside, empty rows, and of rows with one slot the last."""
    rng = np.random.default_rng(6)
    b = Both(ctx, 5, 2, 64, "i8")
    b.end = [0, 0, 20, 20, 40]
    slot, pos, cnt = [-1, 5, 2, 3, 0, 3, 4, 1, 1 << 30], [0, 0, 0, 0, 60, 0, 20, -3, 0], [20, 20, 20, 20, 20, 20, 20, 20, 20]
    k, v = f16(rng, (9, 20, 2, 64)), f16(rng, (9, 20, 2, 64))
    b.write(dev, k, v, slot=slot, pos=pos, count=cnt)
    b.check()
    assert (b.r.open[:, 0] > 0).tolist() == [False, False, True, True, True]
    b.write(dev, k, v, slot=slot, pos=pos, count=[0, -3, 0, 0, 0, 0, -1, 0, 0])
    b.check()
    huge = [2 ** 31 - 1] * 9
    b.write(dev, k, v, slot=slot, pos=huge, count=cnt)
    b.check()
    # more tokens than a slot has positions, of which a few are there
    b.d.write(dev(k), dev(v), 1, 2 ** 31 - 1, strides=(0, 128, 64), pos=dev(i32([3])), count=dev(i32([17])))
    b.r.write(k[:1, :17], v[:1, :17], pos=[3])
    b.end[0] = 20
    b.check()
    out = dev(np.zeros((64, 2, 64), np.float16))
    b.d.read(out, 0, 1, 2 ** 31 - 1, strides=(0, 128, 64), slot=dev(i32([4])), count=dev(i32([2 ** 31 - 1])))
    np.testing.assert_array_equal(ctx.download(out, (64, 2, 64), np.float16)[:40], b.r.stands_for(0)[4, :, :40].transpose(1, 0, 2))
    b.free()


def test_padding_rows_do_not_take_a_slot(ctx, dev):
    """Rows behind the last sequence name slot 0 and have no tokens, or tokens outside the cache: slot 0's own row writes.
    More rows than a wave looks at in one go."""
    rng = np.random.default_rng(7)
    n = 200
    b = Both(ctx, 3, 2, 96, "e4m3")
    slot, pos, cnt = [0, 1, 2, 1] + [0] * (n - 4), [0] * n, [40, 33, 10, 64] + [0] * (n - 4)
    cnt[150], pos[150] = 40, 57
    cnt[180], pos[180] = -3, 5
    k, v = f16(rng, (n, 64, 2, 64)), f16(rng, (n, 64, 2, 64))
    b.end = [40, 64, 10]
    b.write(dev, k, v, slot=slot, pos=pos, count=cnt)
    b.check()
    assert b.r.open[:, 0].tolist() == [2, 0, 1]
    # one of them writes after all
    cnt[150], pos[150] = 7, 40
    b.end = [47, 64, 10]
    b.write(dev, k, v, slot=slot, pos=pos, count=cnt)
    b.check()
    b.free()


@pytest.mark.parametrize("fmt", FMT)
def test_source_layouts(ctx, dev, fmt):
    """Rows of a fused projection, per-head tiles as the engine's cross keys and values, a broadcast row."""
    rng = np.random.default_rng(7)
    n, t, h = 2, 50, 3
    k, v = f16(rng, (n, t, h, 64)), f16(rng, (n, t, h, 64))
    fused = np.zeros((n, t, 3, h, 64), np.float16)
    fused[:, :, 1], fused[:, :, 2] = k, v
    at = dev(fused)
    tiles = np.zeros((n, 2, h, 72, 64), np.float16)
    tiles[:, 0, :, :t], tiles[:, 1, :, :t] = k.transpose(0, 2, 1, 3), v.transpose(0, 2, 1, 3)
    tat = dev(tiles)
    for ka, va, strides in ((at + h * 128, at + 2 * h * 128, (t * 3 * h * 64, 3 * h * 64, 64)),
                            (tat, tat + h * 72 * 128, (2 * h * 72 * 64, 64, 72 * 64))):
        b = Both(ctx, n, h, 64, fmt)
        b.end = [t] * n
        b.r.write(k, v)
        b.d.write(ka, va, n, t, strides=strides)
        b.check().free()
    b = Both(ctx, n, h, 64, fmt)
    b.end = [t] * n
    b.r.write(np.stack([k[0]] * n), np.stack([v[0]] * n))
    b.d.write(dev(k), dev(v), n, t, strides=(0, h * 64, 64))
    b.check().free()


@pytest.mark.parametrize("fmt", FMT)
def test_read_back(ctx, dev, fmt):
    """Any range, shared slots, other layouts, one of the two, and what is left as it was."""
    rng = np.random.default_rng(8)
    b = Both(ctx, 3, 2, 128, fmt)
    cnt = [128, 77, 40]
    b.write(dev, f16(rng, (3, 128, 2, 64)), f16(rng, (3, 128, 2, 64)), count=cnt)
    k64, v64 = b.r.stands_for(0), b.r.stands_for(1)
    slot, pos, count, t = [1, 1, 0, 2, 9, -1, 0], [0, 30, 5, 39, 0, 0, 100], [70, 47, 64, 1, 10, 10, 70], 70
    n = len(slot)
    init = f16(rng, (n, 2, t, 64))
    ok, ov = dev(init), dev(init)
    args = dict(strides=(2 * t * 64, 64, t * 64), slot=dev(i32(slot)), pos=dev(i32(pos)), count=dev(i32(count)))
    b.d.read(ok, ov, n, t, **args)
    for got, src in ((ctx.download(ok, init.shape, np.float16), k64), (ctx.download(ov, init.shape, np.float16), v64)):
        want = init.copy()
        for r in range(n):
            if 0 <= slot[r] < 3:
                m = min(count[r], 128 - pos[r])
                want[r, :, :m] = src[slot[r], :, pos[r]:pos[r] + m]
        np.testing.assert_array_equal(got.view(np.uint16), want.view(np.uint16))
    o = dev(init)
    b.d.read(0, o, n, t, **args)
    np.testing.assert_array_equal(ctx.download(o, init.shape, np.float16), ctx.download(ov, init.shape, np.float16))
    b.free()


# ---------------------------------------------------------------- attention


def filled(ctx, dev, rng, slots, heads, lens, fmt, cap=None):
    b = Both(ctx, slots, heads, cap or max(max(lens), 1), fmt)
    t = max(max(lens), 1)
    b.end = list(lens)
    b.write(dev, f16(rng, (slots, t, heads, 64)), f16(rng, (slots, t, heads, 64)), count=lens)
    return b


def run_attention(ctx, dev, b, q, causal, length, slot=None, first=None, count=None, scale=0.125, head_slot=None,
                  align_heads=0, align_cols=0, out=None, **kw):
    n, t, h = q.shape[:3]
    init = np.full((n, t, h, 64), 7.0, np.float16)
    o, l = dev(init), dev(np.full((n, t, h), 5.0, np.float32))
    al = dev(np.full((n, t, align_heads, align_cols), 3.0, np.float32)) if align_heads else 0
    b.d.attention(dev(q), o, n, t, h, causal=causal, scale=scale, slot=dev(i32(slot)), count=dev(i32(count)),
                  len=dev(i32(length)), first=dev(i32(first)), lse=l, head_slot=dev(i32(head_slot)), align=al,
                  align_heads=align_heads, align_cols=align_cols, **kw)
    return (ctx.download(o, init.shape, np.float16), ctx.download(l, (n, t, h), np.float32),
            ctx.download(al, (n, t, align_heads, align_cols), np.float32) if al else None)


def check_attention(b, q, got, causal, length, slot=None, first=None, count=None, scale=0.125, head_slot=None):
    out, lse, align = got
    n, t, h = q.shape[:3]
    w, wl, prob, (av, aq) = R.attention(b.r, q, causal, length, slot, first, count, scale)
    there = np.arange(t)[None] < (np.full(n, t) if count is None else np.asarray(count))[:, None]
    assert (out[~there] == 7.0).all() and (lse[~there] == 5.0).all()
    seen = (prob > 0).sum(-1)
    ds = 80 * U * aq
    rel = 2 * ds + (seen + 16) * U
    tol = (rel + H)[..., None] * av + H * np.abs(w) + 2.0 ** -24
    vmax = np.abs(b.r.exact(1)).max() if np.isfinite(b.r.exact(1)).all() else 10.0
    tol += (seen * 2.0 ** -24 * vmax)[..., None]
    err = np.abs(out.astype(np.float64) - w)
    bad = there[..., None, None] & ~(err <= tol)
    assert not bad.any(), f"{bad.sum()} outputs off, worst {np.nanmax(err / tol):.3g} x the bound at {np.argwhere(bad)[:4].tolist()}"
    fin = np.isfinite(wl)
    assert (np.isfinite(lse) == fin)[there].all() and (lse[there & (~fin).all(-1)] == -np.inf).all()
    e = np.abs(lse.astype(np.float64) - np.where(fin, wl, 0))
    lt = ds + (seen + 8) * U + 4 * U * np.abs(np.where(fin, wl, 0))
    assert (e[fin & there[..., None]] <= lt[fin & there[..., None]]).all(), np.nanmax((e / lt)[fin & there[..., None]])
    if align is not None:
        cols = align.shape[-1]
        done = set()
        for a, s in enumerate(head_slot):
            if 0 <= s < align.shape[2] and s not in done:
                done.add(s)
                p = np.zeros((n, t, cols))
                m = min(cols, prob.shape[-1])
                p[..., :m] = prob[:, :, a, :m]
                g = align[:, :, s].astype(np.float64)
                tol = rel[:, :, a, None] * p + 2.0 ** -120
                assert (np.abs(g - p)[there] <= tol[there]).all()
                assert (g[there][p[there] == 0] <= 2.0 ** -120).all()
        for s in set(range(align.shape[2])) - done:
            assert (align[:, :, s] == 3.0).all()
        assert (align[~there] == 3.0).all()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("length", [1, 2, 31, 32, 33, 63, 64, 65, 127, 129, 448, 1500])
def test_attention_of_single_tokens(ctx, dev, fmt, length):
    rng = np.random.default_rng(length)
    lens = [length, max(1, length - 1), max(1, length // 2)]
    b = filled(ctx, dev, rng, 3, 2, lens, fmt)
    q = f16(rng, (3, 1, 2, 64), 1.5)
    check_attention(b, q, run_attention(ctx, dev, b, q, False, lens), False, lens)
    b.free()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("tokens", [1, 2, 5, 15, 16, 17, 32, 33, 64, 65, 97])
def test_attention_of_prompts(ctx, dev, fmt, tokens):
    """Causal, each row behind another past; the shorter rows' padding is left as it was."""
    rng = np.random.default_rng(tokens)
    past = [0, 30, 61]
    cnt = [tokens, max(tokens - 3, 0), (tokens + 1) // 2]
    b = filled(ctx, dev, rng, 3, 2, [p + c for p, c in zip(past, cnt)], fmt, cap=200)
    q = f16(rng, (3, tokens, 2, 64), 1.5)
    length = [p + 1 for p in past]
    check_attention(b, q, run_attention(ctx, dev, b, q, True, length, count=cnt), True, length, count=cnt)
    b.free()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("heads,kvh,tokens", [(4, 2, 1), (6, 2, 1), (8, 1, 1), (16, 1, 1), (20, 1, 1), (64, 1, 1),
                                              (6, 2, 3), (10, 2, 7), (34, 2, 2), (64, 1, 5)])
def test_attention_of_shared_heads(ctx, dev, fmt, heads, kvh, tokens):
    rng = np.random.default_rng(heads + tokens)
    b = filled(ctx, dev, rng, 2, kvh, [100, 70], fmt)
    q = f16(rng, (2, tokens, heads, 64), 1.5)
    length = [101 - tokens, 71 - tokens]
    check_attention(b, q, run_attention(ctx, dev, b, q, True, length), True, length)
    b.free()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("tokens", [1, 4, 20])
def test_attention_of_rows_that_see_little_or_nothing(ctx, dev, fmt, tokens):
    """Lengths of zero and below, a first position at or behind the end, slots outside the cache, lengths past it."""
    rng = np.random.default_rng(11)
    b = filled(ctx, dev, rng, 3, 2, [96, 50, 33], fmt, cap=96)
    slot = [0, 1, 2, 0, 1, 2, 0, 3, -1, 0, 1, 0]
    length = [0, -7, 1, 40, 50, 33, 96, 50, 50, 5000, 50, 2 ** 31 - 1]
    first = [0, 0, 0, 40, 49, -9, 95, 0, 0, 64, 2 ** 31 - 1, 3]
    n = len(slot)
    q = f16(rng, (n, tokens, 2, 64), 1.5)
    for causal in (False, True):
        # (beyond what a slot was given the cache stands for what lies there)
        for f in (None, first):
            got = run_attention(ctx, dev, b, q, causal, length, slot=slot, first=f)
            check_attention(b, q, got, causal, length, slot=slot, first=f)
    b.free()


@pytest.mark.parametrize("fmt", FMT)
def test_what_is_not_seen_is_not_looked_at(ctx, dev, fmt):
    """NaN and infinities behind the length and before the first position: in coded blocks (scale NaN), in the open block,
    and in positions of the open block that earlier tokens of a prompt do not see yet. A block that is seen at all
    counts as a whole."""
    rng = np.random.default_rng(12)
    for where, length, first, cnt in (("behind", 64, 0, 100), ("open", 70, 0, 96 - 26), ("before", 100, 32, 100)):
        b = Both(ctx, 1, 1, 128, fmt)
        k, v = f16(rng, (1, 100, 1, 64)), f16(rng, (1, 100, 1, 64))
        if where == "behind":
            k[0, 66, 0, 3], v[0, 80, 0, 5], v[0, 98, 0, 1] = np.nan, np.inf, np.nan
        elif where == "open":
            k, v = k[:, :96], v[:, :96]
            k[0, 80], v[0, 80] = np.nan, np.inf
        else:
            k[0, 20, 0, 3], v[0, 5, 0, 5] = np.inf, np.nan
        if where == "open":  # stale numbers of an earlier sequence in the open block
            b.write(dev, k[:, :95], v[:, :95])
            b.write(dev, k[:, 64:70], v[:, 64:70], pos=[64])
        else:
            b.write(dev, k, v)
        clean = Both(ctx, 1, 1, 128, fmt)
        clean.write(dev, np.nan_to_num(k, nan=0, posinf=0, neginf=0)[:, :cnt], np.nan_to_num(v, nan=0, posinf=0, neginf=0)[:, :cnt])
        for tokens in (1, 6):
            q = f16(rng, (1, tokens, 1, 64), 1.5)
            got = run_attention(ctx, dev, b, q, False, [length], first=[first])
            assert np.isfinite(got[0]).all() and np.isfinite(got[1]).all()
            want = run_attention(ctx, dev, clean, q, False, [length], first=[first])
            for x, y in zip(got[:2], want[:2]):
                np.testing.assert_array_equal(x, y)
        b.free()
        clean.free()
    # a prompt that reaches a block with a NaN: the tokens before it are not touched by it
    b = Both(ctx, 1, 1, 128, fmt)
    for n in (90, 96):  # the block open, and coded
        k, v = f16(rng, (1, n, 1, 64)), f16(rng, (1, n, 1, 64))
        v[0, 70, 0, 9] = np.nan
        for kbad in (False, True):
            if kbad:
                k[0, 71, 0, 5] = np.inf
            b.write(dev, k, v)
            q = f16(rng, (1, 30, 1, 64), 1.5)
            out, lse, _ = run_attention(ctx, dev, b, q, True, [50])  # token i sees 50 + i
            assert np.isfinite(out[0, :15]).all() and np.isfinite(lse[0, :15]).all()
            assert np.isnan(out[0, 22:, :, 9]).all()
            # (in an open block an infinite key alone: a score of -inf where the query's channel is negative)
            assert not kbad or np.isnan(lse[0, 22:][(q[0, 22:, :, 5] > 0) | (n == 96)]).all()
    b.free()


@pytest.mark.parametrize("fmt", FMT)
def test_a_query_that_is_no_number_stays_alone(ctx, dev, fmt):
    rng = np.random.default_rng(13)
    b = filled(ctx, dev, rng, 1, 1, [70], fmt)
    q = f16(rng, (1, 20, 2, 64), 1.5)
    want = run_attention(ctx, dev, b, q, False, [70])
    q[0, 3, 1, 5] = np.nan
    q[0, 11, 0, 5] = np.inf
    got = run_attention(ctx, dev, b, q, False, [70])
    hit = np.zeros((1, 20, 2), bool)
    hit[0, 3, 1] = hit[0, 11, 0] = True
    assert np.isnan(got[0][hit]).all()
    np.testing.assert_array_equal(got[0][~hit], want[0][~hit])
    np.testing.assert_array_equal(got[1][~hit], want[1][~hit])
    b.free()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("scale,size", [(1.0, 8.0), (0.125, 40.0), (1e-4, 1.0), (0.125, 0.0)])
def test_attention_of_sharp_and_flat_rows(ctx, dev, fmt, scale, size):
    """Scores up to thousands (one position takes all, wherever it lies) and none at all (a plain mean)."""
    rng = np.random.default_rng(14)
    b = filled(ctx, dev, rng, 2, 2, [300, 290], fmt)
    q = f16(rng, (2, 3, 2, 64), size)
    check_attention(b, q, run_attention(ctx, dev, b, q, False, [300, 290], scale=scale), False, [300, 290], scale=scale)
    b.free()


@pytest.mark.parametrize("fmt", FMT)
def test_attention_over_blocks_of_very_different_scales(ctx, dev, fmt):
    rng = np.random.default_rng(15)
    t = 32 * 9 + 7
    size = np.repeat(10.0 ** np.array([0, -4, 2, -6, 3, 0, -5, 1, 4, 0]), 32)[:t, None, None]
    k, v = f16(rng, (1, t, 1, 64)), (rng.standard_normal((1, t, 1, 64)) * size).astype(np.float16)
    b = Both(ctx, 1, 1, t, fmt)
    b.end = [t]
    b.write(dev, k, v)
    for first in (0, 32 * 5, 32 * 6):
        q = f16(rng, (1, 2, 1, 64), 1.5)
        check_attention(b, q, run_attention(ctx, dev, b, q, False, [t], first=[first]), False, [t], first=[first])
    b.free()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("tokens,heads,kvh", [(1, 5, 5), (3, 4, 2), (20, 3, 3)])
@pytest.mark.parametrize("cols", [70, 96, 131])
def test_alignment_rows(ctx, dev, fmt, tokens, heads, kvh, cols):
    """Chosen heads' probabilities, cropped or padded to the row's columns; of two heads with one index the first."""
    rng = np.random.default_rng(cols + tokens)
    b = filled(ctx, dev, rng, 3, kvh, [96, 90, 50], fmt, cap=96)
    head_slot = [2, -1, 0, 0, 4][:heads]
    q = f16(rng, (3, tokens, heads, 64), 1.5)
    length, first = [96 - tokens, 80 - tokens, 0], [0, 37, 0]
    cnt = [tokens, max(tokens - 1, 1), tokens]
    for causal in (False, True):
        got = run_attention(ctx, dev, b, q, causal, length, first=first, count=cnt, head_slot=head_slot, align_heads=3, align_cols=cols)
        check_attention(b, q, got, causal, length, first=first, count=cnt, head_slot=head_slot)
    b.free()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("rows,heads,tokens", [(10, 16, 5), (3, 7, 1), (20, 16, 1), (17, 16, 3), (10, 16, 6), (1, 2, 30),
                                               (9, 15, 33), (11, 12, 16), (9, 15, 16)])
def test_alignment_rows_of_long_caches(ctx, dev, fmt, rows, heads, tokens):
    """The encoder's 1500 positions: scores kept by a workgroup (the most that are) or in their rows, by one workgroup or
    several that share the blocks, of four and of eight waves."""
    rng = np.random.default_rng(rows)
    lens = [1500 - 7 * (r % 5) for r in range(rows)]
    b = filled(ctx, dev, rng, rows, heads, lens, fmt)
    q = f16(rng, (rows, tokens, heads, 64), 1.5)
    head_slot = [(5 * h) % heads if h % 3 == 0 else -1 for h in range(heads)]
    n = max(head_slot) + 1
    got = run_attention(ctx, dev, b, q, False, lens, head_slot=head_slot, align_heads=n, align_cols=1500)
    check_attention(b, q, got, False, lens, head_slot=head_slot)
    b.free()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("rows,heads,kvh,tokens", [(16, 16, 16, 17), (13, 20, 20, 40), (16, 32, 16, 33), (17, 16, 16, 1),
                                                   (4, 8, 4, 130)])
def test_attention_of_many_rows(ctx, dev, fmt, rows, heads, kvh, tokens):
    """Workgroups enough for every CU: queries of a wave's own (more than 16 of a cache head), or four waves a tile."""
    rng = np.random.default_rng(rows + tokens)
    past = [(13 * r) % 60 for r in range(rows)]
    cnt = [max(1, tokens - r % 4) for r in range(rows)]
    b = filled(ctx, dev, rng, rows, kvh, [p + c for p, c in zip(past, cnt)], fmt, cap=200)
    q = f16(rng, (rows, tokens, heads, 64), 1.5)
    length, first = [p + 1 for p in past], [r % 3 for r in range(rows)]
    for causal in (True, False):
        check_attention(b, q, run_attention(ctx, dev, b, q, causal, length, first=first, count=cnt), causal, length, first=first, count=cnt)
    b.free()


@pytest.mark.parametrize("fmt", FMT)
@pytest.mark.parametrize("rows,heads,tokens,length", [(16, 16, 1, 15700), (17, 16, 1, 8000), (17, 8, 20, 8000), (16, 16, 20, 2600)])
def test_attention_over_more_blocks_than_a_wave_has_scales_of(ctx, dev, fmt, rows, heads, tokens, length):
    """More than 60 blocks a wave, of eight and four waves and of waves with queries of their own; rows that share a slot."""
    rng = np.random.default_rng(length)
    b = filled(ctx, dev, rng, 1, heads, [length], fmt)
    q = f16(rng, (rows, tokens, heads, 64), 1.5)
    lens, slot = [length - 37 * r - tokens + 1 for r in range(rows)], [0] * rows
    for first in (None, [61 * r for r in range(rows)]):
        got = run_attention(ctx, dev, b, q, True, lens, slot=slot, first=first)
        check_attention(b, q, got, True, lens, slot=slot, first=first)
    b.free()


@pytest.mark.parametrize("fmt", FMT)
def test_attention_layouts_and_shared_counter(ctx, dev, fmt):
    """Queries inside a fused projection's rows, the output per head, lse not wanted, one counter for all rows."""
    rng = np.random.default_rng(16)
    n, t, h = 3, 2, 4
    b = filled(ctx, dev, rng, n, h, [60, 60, 60], fmt)
    q = f16(rng, (n, t, h, 64), 1.5)
    fused = np.full((n, t, 3, h, 64), np.nan, np.float16)
    fused[:, :, 0] = q
    o = dev(np.zeros((n, h, t, 64), np.float16))
    b.d.attention(dev(fused), o, n, t, h, q_strides=(t * 3 * h * 64, 3 * h * 64, 64), out_strides=(h * t * 64, 64, t * 64),
                  causal=True, len=dev(i32([58])), len_stride=0, len_add=1)
    got = ctx.download(o, (n, h, t, 64), np.float16).transpose(0, 2, 1, 3)
    want = run_attention(ctx, dev, b, q, True, [59] * n)[0]
    np.testing.assert_array_equal(got, want)
    b.free()


def test_attention_needs_its_workspace(ctx, dev):
    rng = np.random.default_rng(17)
    b = filled(ctx, dev, rng, 1, 1, [1500], "i8")
    q, o = dev(f16(rng, (1, 1, 1, 64))), dev(np.zeros((1, 64), np.float16))
    a = L.Kv8Attention(q=q, out=o, q_row=64, q_token=64, q_head=64, out_row=64, out_token=64, out_head=64, rows=1,
                       tokens=1, heads=1, scale=0.125, len_add=1500)
    need = decode8.attention_bytes(ctx, b.d.kv, a)
    if need:
        for work, n in ((0, need), (ctx.workspace(need)[0], need - 1), (ctx.workspace(need)[0] + 64, need)):
            a.work, a.work_bytes = work, n
            with pytest.raises(L.MzError, match="workspace"):
                L.check(L.lib().mz_kv8_attention(ctx.h, b.d.kv, a))
    b.free()


def test_one_workspace_for_calls_of_every_size(ctx, dev):
    """Attention and scores of different sizes one after the other in one workspace, twice: the same bits as each in one of
    its own, which is zero before and whose head is zero afterwards."""
    rng = np.random.default_rng(19)
    caches = [filled(ctx, dev, rng, r, h, [n] * r, "i8") for r, h, n in ((1, 2, 1500), (5, 7, 1400), (2, 20, 700))]
    qs = [f16(rng, (b.r.slots, 1, b.r.heads, 64), 1.5) for b in caches]
    xs = [logits(rng, n, v, np.float32) for n, v in ((1, 51865), (30, 20000), (200, 9000))]
    size = 32 << 20
    shared = ctx.alloc(size)

    def attend(i, work):
        b, q = caches[i], qs[i]
        return run_attention(ctx, dev, b, q, False, [b.end[0]] * len(q), head_slot=[0] + [-1] * (b.r.heads - 1), align_heads=1,
                             align_cols=1500, work=work)

    def score(i, work):
        x = xs[i]
        o = [dev(np.zeros((len(x), 3), t)) for t in (np.float32, np.int32)]
        decode8.token_scores(ctx, dev(x), *x.shape, entropy=o[0], alts=3, alt_ids=o[1], work=work)
        return ctx.download(o[0], (len(x),), np.float32), ctx.download(o[1], (len(x), 3), np.int32)

    calls = [(attend, 0), (score, 0), (attend, 1), (score, 1), (attend, 2), (score, 2), (attend, 0), (score, 0)]
    for _ in range(2):
        for f, i in calls:
            own = ctx.alloc(size)
            want, got = f(i, (own, size)), f(i, (shared, size))
            for a, b in zip(want, got):
                np.testing.assert_array_equal(a, b)
            for p in (own, shared):
                assert not ctx.download(p, (4096,), np.uint32).any()
            ctx.free(own)
    ctx.free(shared)
    for b in caches:
        b.free()


@pytest.mark.parametrize("fmt", FMT)
def test_offsets_past_32_bits(ctx, dev, fmt):
    """A cache whose codes alone are 5 GB for the keys and as much for the values: the last slot's last blocks written,
    read and attended to."""
    slots, heads, blocks = 2, 8, 153000
    kv = decode8.Kv8(ctx, slots, heads, blocks * 32, fmt)
    rng = np.random.default_rng(18)
    small = Both(ctx, 1, heads, 96, fmt)
    k, v = f16(rng, (1, 75, heads, 64)), f16(rng, (1, 75, heads, 64))
    small.end = [75]
    small.write(dev, k, v)
    p0 = (blocks - 3) * 32
    kv.write(dev(k), dev(v), 1, 75, slot=dev(i32([1])), pos=dev(i32([p0])))
    out = dev(np.zeros((75, heads, 64), np.float16))
    for side in range(2):
        kv.read(0 if side else out, out if side else 0, 1, 75, slot=dev(i32([1])), pos=dev(i32([p0])))
        np.testing.assert_array_equal(ctx.download(out, (75, heads, 64), np.float16),
                                      small.r.stands_for(side)[0, :, :75].transpose(1, 0, 2))
    q = f16(rng, (1, 2, heads, 64), 1.5)
    want = run_attention(ctx, dev, small, q, True, [74])
    check_attention(small, q, want, True, [74])
    big = Both.__new__(Both)
    big.d = kv
    got = run_attention(ctx, dev, big, q, True, [p0 + 74], slot=[1], first=[p0])
    # (the same numbers, split over workgroups in another way)
    np.testing.assert_allclose(got[0].astype(np.float32), want[0].astype(np.float32), rtol=4 * H, atol=2.0 ** -10)
    np.testing.assert_allclose(got[1], want[1], rtol=1e-5)
    small.free()
    kv.free()


# ---------------------------------------------------------------- token scores


def run_scores(ctx, dev, x, tokens, mask=None, alts=0, pad=0, off=0):
    """Rows of x with `pad` elements between them, the first at element `off` of its buffer."""
    n, v = x.shape
    buf = np.full(off + n * (v + pad), np.nan, x.dtype)
    for r in range(n):
        buf[off + r * (v + pad):off + r * (v + pad) + v] = x[r]
    o = [dev(np.full((n, max(w, 1)), 9, t)) for w, t in ((1, np.float32), (1, np.float32), (alts, np.int32), (alts, np.float32))]
    decode8.token_scores(ctx, dev(buf) + off * x.itemsize, n, v, dtype=L.DT_F32 if x.dtype == np.float32 else L.DT_F16,
                         ld=v + pad, mask=dev(mask), tokens=dev(i32(tokens)), logp=o[0], entropy=o[1], alts=alts,
                         alt_ids=o[2], alt_logp=o[3])
    return (ctx.download(o[0], (n,), np.float32), ctx.download(o[1], (n,), np.float32),
            ctx.download(o[2], (n, alts), np.int32), ctx.download(o[3], (n, alts), np.float32))


def check_scores(x, tokens, got, mask=None, alts=0):
    logp, ent, ids, best = R.scores(x, tokens, mask, alts)
    np.testing.assert_array_equal(got[2], ids)
    z = x.astype(np.float64).copy()
    if mask is not None:
        z[:, mask != 0] = -np.inf
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        m = z.max(-1, keepdims=True)
        d = np.where(np.isfinite(z) & np.isfinite(m), z - m, 0)
        e = np.where(np.isfinite(z) & np.isfinite(m), np.exp(d), 0)
        for r in range(len(x)):
            if np.isfinite(m[r, 0]):
                e[r, z[r].argmax()] = 0
        part = U * (z.shape[1] + 8 + 6 * np.minimum(np.abs(d), 104))
        dz = (part * e).sum(-1) / (1 + e.sum(-1))
        dent = (part * e * (2 + np.abs(d))).sum(-1) / (1 + e.sum(-1)) + dz * (1 + np.abs(e * d).sum(-1) / (1 + e.sum(-1)))
    for g, w, t in ((got[0], logp, dz), (got[1], ent, dent)):
        np.testing.assert_array_equal(np.isnan(g), np.isnan(w))
        np.testing.assert_array_equal(g == -np.inf, w == -np.inf)
        f = np.isfinite(w)
        err = np.abs(g[f] - w[f])
        assert (err <= t[f] + 6 * U * np.abs(w[f]) + 2.0 ** -140).all(), (err / (t[f] + 6 * U * np.abs(w[f]) + 2.0 ** -140)).max()
    np.testing.assert_array_equal(np.isnan(got[3]), np.isnan(best))
    f = np.isfinite(best)
    np.testing.assert_array_equal(got[3][~f & ~np.isnan(best)], best[~f & ~np.isnan(best)])
    t = np.broadcast_to(dz[:, None], best.shape)[f] + 6 * U * np.abs(best[f])
    assert (np.abs(got[3][f] - best[f]) <= t).all()


def logits(rng, n, v, dtype, sure=8.0):
    x = rng.standard_normal((n, v)) * 2.5
    x[np.arange(n), rng.integers(0, v, n)] += rng.uniform(0, sure, n)
    return x.astype(dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 63, 64, 65, 255, 1000, 1024, 1025, 4099, 16384, 51864, 51865, 51866])
@pytest.mark.parametrize("rows", [1, 3])
def test_scores(ctx, dev, dtype, vocab, rows):
    rng = np.random.default_rng(vocab + rows)
    x = logits(rng, rows, vocab, dtype)
    tokens = rng.integers(0, vocab, rows)
    mask = (rng.random(vocab) < 0.3).astype(np.uint8)
    for alts, m, pad, off in ((0, None, 0, 0), (5, mask, 3, 1), (16, None, 0, 3), (1, None, 5, 2), (8, mask, 1, 7)):
        check_scores(x, tokens, run_scores(ctx, dev, x, tokens, m, alts, pad, off), m, alts)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows", [17, 300, 1100])
def test_scores_of_many_rows(ctx, dev, dtype, rows):
    rng = np.random.default_rng(rows)
    x = logits(rng, rows, 3001, dtype)
    tokens = rng.integers(-1, 3001, rows)
    mask = (rng.random(3001) < 0.1).astype(np.uint8)
    check_scores(x, tokens, run_scores(ctx, dev, x, tokens, mask, 4, 1, 1), mask, 4)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("vocab", [40, 5000, 51866])
def test_scores_of_unusual_rows(ctx, dev, dtype, vocab):
    """Ties everywhere, one number only, lowest numbers, -inf in places and throughout, NaN, +inf, sorted rows, sure rows."""
    rng = np.random.default_rng(20)
    low = np.finfo(dtype).min
    rows = []
    rows.append(np.zeros(vocab))
    rows.append(np.full(vocab, low))
    rows.append(np.full(vocab, -np.inf))
    rows.append(np.where(np.arange(vocab) == vocab - 1, 3.0, -np.inf))
    rows.append(np.where(np.arange(vocab) % 7 == 3, 2.0, low))
    rows.append(np.where(rng.random(vocab) < 0.5, rng.standard_normal(vocab), -np.inf))
    rows.append(np.arange(vocab) / vocab * 9)
    rows.append(-np.arange(vocab) / vocab * 9)
    rows.append(rng.integers(0, 3, vocab).astype(float))
    rows.append(np.where(np.arange(vocab) == 11, 30.0, rng.standard_normal(vocab)))
    rows.append(np.where(np.arange(vocab) == 11, 30.0, -20.0 + rng.standard_normal(vocab)))
    rows.append(np.full(vocab, np.finfo(dtype).max))
    r = rng.standard_normal(vocab)
    r[vocab // 2] = np.nan
    rows.append(r)
    r = rng.standard_normal(vocab)
    r[vocab - 1] = np.inf
    rows.append(r)
    rows.append(np.full(vocab, np.nan))
    rows.append(np.where(np.arange(vocab) < 3, [1.0] * 3 + [0.0] * (vocab - 3), -np.inf))
    x = np.stack(rows).astype(dtype)
    n = len(x)
    for tokens in (np.full(n, 11), np.full(n, vocab - 1), np.full(n, -1), np.full(n, vocab), np.full(n, 2 ** 31 - 1)):
        for alts in (0, 7):
            check_scores(x, tokens, run_scores(ctx, dev, x, tokens, None, alts), None, alts)
    mask = np.zeros(vocab, np.uint8)
    mask[[0, 11, vocab // 2, vocab - 1]] = [1, 7, 255, 128]  # NaN and +inf masked: the row is an ordinary one
    for tokens in (np.full(n, 11), np.full(n, 5)):
        check_scores(x, tokens, run_scores(ctx, dev, x, tokens, mask, 5, 1, 1), mask, 5)
    check_scores(x, np.full(n, 3), run_scores(ctx, dev, x, np.full(n, 3), np.ones(vocab, np.uint8), 3), np.ones(vocab, np.uint8), 3)


def test_scores_at_a_step(ctx, dev):
    """Tokens and results kept [rows][steps], the step's index on the device; an index outside writes nothing."""
    rng = np.random.default_rng(21)
    n, v, steps, alts = 3, 700, 6, 2
    x = logits(rng, n, v, np.float32)
    tok = rng.integers(0, v, (n, steps))
    dx, dt, at = dev(x), dev(i32(tok)), dev(i32([0]))
    for step, add in ((0, 0), (3, 0), (2, 3), (6, 0), (0, -1), (2 ** 31 - 1, 2 ** 31 - 1), (-(2 ** 31), 0)):
        o = [dev(np.full((n, steps, w), 9, t)) for w, t in ((1, np.float32), (1, np.float32), (alts, np.int32), (alts, np.float32))]
        ctx.upload(at, i32([step]))
        decode8.token_scores(ctx, dx, n, v, tokens=dt, token_stride=steps, at=at, at_add=add, logp=o[0], entropy=o[1],
                             out_stride=steps, alts=alts, alt_ids=o[2], alt_logp=o[3])
        got = [ctx.download(p, (n, steps, w), t) for p, w, t in zip(o, (1, 1, alts, alts), (np.float32, np.float32, np.int32, np.float32))]
        s = step + add
        if 0 <= s < steps:
            check_scores(x, tok[:, s], (got[0][:, s, 0], got[1][:, s, 0], got[2][:, s], got[3][:, s]), None, alts)
            got = [np.delete(g, s, 1) for g in got]
        assert all((g == 9).all() for g in got)
    # no token at an index outside the tokens' stride; results not wanted
    o = dev(np.full((n, steps), 9, np.float32))
    ctx.upload(at, i32([4]))
    decode8.token_scores(ctx, dx, n, v, tokens=dt, token_stride=4, at=at, logp=o, out_stride=steps)
    assert (ctx.download(o, (n, steps), np.float32)[:, 4] == 0).all()
    e = dev(np.full((n,), 9, np.float32))
    decode8.token_scores(ctx, dx, n, v, entropy=e)
    assert np.abs(ctx.download(e, (n,), np.float32) - R.scores(x, tok[:, 0])[1]).max() < 1e-4


# ---------------------------------------------------------------- together, in a captured step


@pytest.mark.parametrize("fmt", FMT)
def test_a_captured_decoding_step(ctx, dev, fmt):
    """A step as a program would capture it: the position's keys and values into the cache, attention over it and over
    a second cache that beams share, a product for logits, their scores beside the tokens, the counter moved on by a
    copy. Every replay, with eager calls on other caches between them, gives the bits of the same calls made eagerly, and
    those are right."""
    rng = np.random.default_rng(22)
    n, h, v, steps, kx = 4, 2, 512, 40, 70
    d = h * 64
    xs = [f16(rng, (n, 3, h, 64), 1.0) for _ in range(steps)]  # q, k, v of each step
    cross_kv = filled(ctx, dev, rng, 2, h, [kx, kx - 9], fmt)
    slot = dev(i32([0, 0, 1, 1]))
    xlen = dev(i32([kx, kx, kx - 9, kx - 9]))
    w = dev(f16(rng, (v, d), 0.2))
    tok = rng.integers(0, v, (n, steps))
    dtok, counts = dev(i32(tok)), dev(np.arange(1, steps + 1, dtype=np.int32))
    src = dev(np.stack(xs))
    mask = dev((rng.random(v) < 0.05).astype(np.uint8))

    class Program:
        def __init__(self):
            self.kv = decode8.Kv8(ctx, n, h, steps, fmt)
            self.x, self.ctr = dev(xs[0]), dev(i32([0]))
            self.a, self.o, self.y = (dev(np.zeros((n, d), np.float16)) for _ in range(3))
            self.logits = dev(np.zeros((n, v), np.float16))
            self.al = dev(np.zeros((n, 1, 1, kx), np.float32))
            self.lp, self.en = dev(np.zeros((n, steps), np.float32)), dev(np.zeros((n, steps), np.float32))
            self.ids = dev(np.zeros((n, steps, 3), np.int32))

        def step(self):
            x = self.x
            self.kv.write(x + d * 2, x + 2 * d * 2, n, 1, strides=(3 * d, d, 64), pos=self.ctr, pos_stride=0)
            self.kv.attention(x, self.a, n, 1, h, q_strides=(3 * d, d, 64), causal=True, len=self.ctr, len_stride=0, len_add=1)
            cross_kv.d.attention(self.a, self.o, n, 1, h, causal=False, slot=slot, len=xlen, scale=2.0,
                                 head_slot=hs, align=self.al, align_heads=1, align_cols=kx)
            L.check(L.lib().mz_gemm(ctx.h, self.o, d, w, self.logits, v, n, v, d, 0))
            decode8.token_scores(ctx, self.logits, n, v, dtype=L.DT_F16, mask=mask, tokens=dtok, token_stride=steps,
                                 at=self.ctr, logp=self.lp, entropy=self.en, out_stride=steps, alts=3, alt_ids=self.ids)

        def feed(self, i):
            L.check(L.lib().mz_copy(ctx.h, self.x, src + i * n * 3 * d * 2, n * 3 * d * 2))
            if i:
                L.check(L.lib().mz_copy(ctx.h, self.ctr, counts + (i - 1) * 4, 4))

        def results(self):
            return [ctx.download(self.lp, (n, steps), np.float32), ctx.download(self.en, (n, steps), np.float32),
                    ctx.download(self.ids, (n, steps, 3), np.int32), ctx.download(self.o, (n, d), np.float16),
                    ctx.download(self.al, (n, kx), np.float32), ctx.download(self.logits, (n, v), np.float16)]

    import ctypes as C
    hs = dev(i32([-1, 0]))
    eager, captured = Program(), Program()
    eager.step()  # workspaces exist before the capture
    ctx.sync()
    L.check(L.lib().mz_graph_begin(ctx.h))
    captured.step()
    g = C.c_void_p()
    L.check(L.lib().mz_graph_end(ctx.h, C.byref(g)))
    last, ref = None, R.Cache(n, h, steps, fmt)
    for i in range(steps):
        eager.feed(i)
        captured.feed(i)
        L.check(L.lib().mz_graph_launch(ctx.h, g))
        eager.step()
        if i % 7 == 3:
            ctx.sync()
        a, b = eager.results(), captured.results()
        for x, y in zip(a, b):
            np.testing.assert_array_equal(x, y, err_msg=f"step {i}")
        last = a
        ref.write(xs[i][:, 1:2].reshape(n, 1, h, 64), xs[i][:, 2:3].reshape(n, 1, h, 64), pos=[i] * n)
        wo = R.attention(ref, xs[i][:, :1].reshape(n, 1, h, 64), True, [i + 1] * n)[0]
        got = ctx.download(eager.a, (n, 1, h, 64), np.float16)
        assert np.abs(got - wo).max() < 8e-3
        xo = R.attention(cross_kv.r, got, False, [kx, kx, kx - 9, kx - 9], slot=[0, 0, 1, 1], scale=2.0)
        assert np.abs(a[3].reshape(n, 1, h, 64) - xo[0]).max() < 8e-3
        np.testing.assert_allclose(a[4], xo[2][:, 0, 1, :kx], rtol=2e-4, atol=1e-30)
        lp, en, ids, _ = R.scores(a[5], tok[:, i], ctx.download(mask, (v,), np.uint8), 3)
        np.testing.assert_allclose(a[0][:, i], lp, atol=2e-5)
        np.testing.assert_allclose(a[1][:, i], en, atol=2e-4)
        np.testing.assert_array_equal(a[2][:, i], ids)
    L.check(L.lib().mz_graph_free(g))
    for p in (eager, captured):
        p.kv.free()
    cross_kv.free()
    assert np.isfinite(last[0]).all() or (last[0] == -np.inf).any()


def test_captured_calls_that_share_rows_and_a_workspace(ctx, dev):
    """Two graphs, each of an attention and scores whose work is shared by workgroups, in one workspace, replayed in turn with
    eager calls between them while a second context runs the same on its own stream with its own: always the bits of the
    eager calls."""
    import ctypes as C
    rng = np.random.default_rng(23)
    lens = (1500, 1311)
    caches = [filled(ctx, dev, rng, 1, 2, [n], "i8") for n in lens]
    qs = [dev(f16(rng, (1, 2, 64), 1.5)) for _ in lens]
    xs = [dev(logits(rng, 1, 51866, np.float32)) for _ in lens]
    other = model.Context(0)
    work = other.alloc(4 << 20)

    class Calls:
        def __init__(self, c, i, work=None):
            self.c, self.i, self.work = c, i, work
            self.o, self.l, self.e = dev(np.zeros((2, 64), np.float16)), dev(np.zeros(2, np.float32)), dev(np.zeros(1, np.float32))
            self.ids = dev(np.zeros((1, 5), np.int32))
            self.kv = decode8.Kv8.__new__(decode8.Kv8)
            self.kv.ctx, self.kv.kv = c, caches[i].d.kv

        def run(self):
            self.kv.attention(qs[self.i], self.o, 1, 1, 2, causal=False, len_add=lens[self.i], lse=self.l, work=self.work)
            decode8.token_scores(self.c, xs[self.i], 1, 51866, entropy=self.e, alts=5, alt_ids=self.ids, work=self.work)

        def results(self):
            self.c.sync()
            return [ctx.download(*x) for x in ((self.o, (2, 64), np.float16), (self.l, (2,), np.float32),
                                               (self.e, (1,), np.float32), (self.ids, (1, 5), np.int32))]

    want, graphs = [], []
    for i in range(2):
        eager = Calls(ctx, i)
        eager.run()
        want.append(eager.results())
        held = Calls(ctx, i)
        L.check(L.lib().mz_graph_begin(ctx.h))
        held.run()
        g = C.c_void_p()
        L.check(L.lib().mz_graph_end(ctx.h, C.byref(g)))
        graphs.append((held, g))
    for n in range(6):
        beside = Calls(other, n % 2, (work, 4 << 20))
        between = Calls(ctx, 1 - n % 2)
        for _ in range(3):
            beside.run()
            for held, g in graphs:
                L.check(L.lib().mz_graph_launch(ctx.h, g))
            between.run()
        for c in (graphs[0][0], graphs[1][0], between, beside):
            for a, b in zip(c.results(), want[c.i]):
                np.testing.assert_array_equal(a, b, err_msg=f"replay {n}")
    for _, g in graphs:
        L.check(L.lib().mz_graph_free(g))
    other.free(work)
    other.close()
    for b in caches:
        b.free()


def test_engine_buffers(ctx, dev):
    """An engine's own buffers: the cross keys and values of its encoder into a cache, and the logits of its step scored
    where they lie, the step's chosen token the best alternative."""
    from mimizuku_amd import synth
    g = synth.TINY
    dims = model.Dims(g.d, g.ff, g.nh, g.enc_layers, g.dec_layers, g.n_mels, g.vocab, g.max_t)
    gc = model.GenCfg.from_dict(synth.generation_config(g), dims)
    e = model.Engine(ctx, dims, gc, bmax=2, eg=2)
    e.load(synth.random_weights(g, seed=0))
    e.encode(synth.synthetic_mel(2, g.n_mels, seed=1), 0)
    xkv, _ = e.buffer(L.BUF_XKV)
    tile = 1536 * 64
    layer = 1
    kv = Both(ctx, 2, g.nh, 1500, "i8")
    kv.end = [1500, 1500]
    strides = (g.dec_layers * 2 * g.nh * tile, 64, tile)
    at = xkv + layer * 2 * g.nh * tile * 2
    kv.d.write(at, at + g.nh * tile * 2, 2, 1500, strides=strides)
    host = e.xkv()[:, layer, :, :, :1500]
    kv.r.write(host[:, 0].transpose(0, 2, 1, 3), host[:, 1].transpose(0, 2, 1, 3))
    kv.check()
    prompt = [gc.sot, 50259, 50359, gc.no_timestamps]
    e.reset([prompt] * 2)
    tok, _ = e.buffer(L.BUF_TOK)
    ctr, _ = e.buffer(L.BUF_CTR)
    lg, _ = e.buffer(L.BUF_LOGITS)
    lp, en, ids = dev(np.zeros((2, g.max_t), np.float32)), dev(np.zeros((2, g.max_t), np.float32)), dev(np.zeros((2, g.max_t, 1), np.int32))
    sup = np.zeros(g.vocab, np.uint8)
    sup[gc.suppress] = 1
    sup1 = sup.copy()
    sup1[gc.begin_suppress] = 1
    m, m1 = dev(sup), dev(sup1)
    for i in range(6):
        e.step(2, False, len(prompt))  # leaves the counter at the chosen token's position
        decode8.token_scores(ctx, lg, 2, g.vocab, mask=m1 if i == len(prompt) - 1 else m, tokens=tok, token_stride=g.max_t, at=ctr,
                             logp=lp, entropy=en, out_stride=g.max_t, alts=1, alt_ids=ids)
    t, got = e.tokens(), ctx.download(ids, (2, g.max_t), np.int32)
    p = ctx.download(lp, (2, g.max_t), np.float32)
    assert (got[:, 4:7] == t[:, 4:7]).all() and (p[:, 1:7] < 0).all() and (p[:, 7:] == 0).all()
    want = R.scores(e.logits(), t[:, 6], sup)[0]
    np.testing.assert_allclose(p[:, 6], want, atol=1e-5)
    kv.free()
    e.close()
