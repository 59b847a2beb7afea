"""CPU checks of the parts of a decoder step: the layout of 4-bit weights, the structs as a C compiler sees them, the
refusals (none of which touches the device), and the definitions in oracle/steps_ref.py."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

from mimizuku_amd import _lib as L
from mimizuku_amd import steps
from oracle import steps_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOME = 0x10000  # an address that no refused call reads
NOBODY = C.create_string_buffer(4096)  # stands for a context: a refused call does not look at it


def test_struct_layouts_match_the_header(tmp_path):
    """Offsets of every field as gcc lays the header's structs out against the Python mirror's."""
    pairs = [("mz_w4", L.W4), ("mz_w4_linear_args", L.W4LinearArgs), ("mz_cross_attention_args", L.CrossArgs),
             ("mz_sample_args", L.SampleArgs)]
    lines, want = [], []
    for name, cls in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {f}));')
            want.append(getattr(cls, f).offset)
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "mimizuku.h"\nint main(void){%s return 0;}' % "".join(lines))
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == want


# ---------------------------------------------------------------- weights in 4 bits


def place(n=40, k=256, group=32, base=SOME):
    w, b = L.W4(), C.c_size_t()
    L.check(L.lib().mz_w4_place(n, k, group, base, C.byref(w), C.byref(b)))
    return w, b.value


@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_place(group):
    w, b = place(group=group)
    assert (w.n, w.k, w.group, w.codes) == (40, 256, group, SOME)
    assert w.scales >= w.codes + 48 * 256 // 2 and w.scales % 256 == 0
    assert SOME + b >= w.scales + 48 * 256 // group * 2
    assert steps.w4_bytes(40, 256, group) == b
    w, b = place(n=1 << 22, k=1 << 14, group=group)  # past 32 bits
    assert w.scales - w.codes == 1 << 35 and b == (1 << 35) + (1 << 37) // group


@pytest.mark.parametrize("bad", [dict(n=0), dict(n=-1), dict(n=(1 << 25) + 1), dict(k=0), dict(k=64), dict(k=200), dict(k=-128),
                                 dict(k=1 << 25), dict(group=16), dict(group=0), dict(group=256), dict(group=96),
                                 dict(base=SOME + 128), dict(n=1 << 25, k=1 << 12)])
def test_w4_place_refuses(bad):
    with pytest.raises(L.MzError, match="mz_w4_place"):
        place(**bad)


BAD_W4 = [dict(n=0), dict(k=100), dict(group=48), dict(codes=0), dict(codes=SOME + 8), dict(scales=0), dict(scales=SOME + 2)]


@pytest.mark.parametrize("fn", ["mz_w4_pack", "mz_w4_unpack"])
def test_w4_pack_refuses(fn):
    call = lambda w, p=SOME, ld=256: L.check(getattr(L.lib(), fn)(C.byref(NOBODY), C.byref(w), p, ld))  # noqa: E731
    for bad in BAD_W4:
        w, _ = place()
        for f, v in bad.items():
            setattr(w, f, v)
        with pytest.raises(L.MzError, match=fn):
            call(w)
    w, _ = place()
    for p, ld in ((0, 256), (SOME + 8, 256), (SOME, 255), (SOME, 260), (SOME, 128), (SOME, -256), (SOME, 1 << 50)):
        with pytest.raises(L.MzError, match=fn):
            call(w, p, ld)
    assert getattr(L.lib(), fn)(None, C.byref(w), SOME, 256) == 2
    assert getattr(L.lib(), fn)(C.byref(NOBODY), None, SOME, 256) == 2


LINEAR = dict(epilogue=L.EPI_F16, m=3, x=SOME, ldx=256, bias=SOME, out=SOME, ldo=40)


def test_w4_linear_refuses():
    def call(change=None, **weights):
        w, _ = place()
        for f, v in weights.items():
            setattr(w, f, v)
        L.check(L.lib().mz_w4_linear(C.byref(NOBODY), C.byref(w), C.byref(L.W4LinearArgs(**{**LINEAR, **(change or {})}))))

    for bad in BAD_W4:
        with pytest.raises(L.MzError, match="mz_w4_linear"):
            call(**bad)
    for bad in (dict(epilogue=-1), dict(epilogue=L.EPI_GELU_POS), dict(epilogue=L.EPI_HEADS), dict(epilogue=6), dict(m=-1),
                dict(m=(1 << 20) + 1), dict(x=0), dict(x=SOME + 8), dict(ldx=248), dict(ldx=260), dict(ldx=1 << 46),
                dict(bias=SOME + 1), dict(out=0), dict(out=SOME + 1), dict(out=SOME + 2, epilogue=L.EPI_F32),
                dict(out=SOME + 2, epilogue=L.EPI_RESID_F32), dict(ldo=39), dict(ldo=1 << 46)):
        with pytest.raises(L.MzError, match="mz_w4_linear"):
            call(bad)
    call(dict(m=0))  # nothing to do is no error
    assert L.lib().mz_w4_linear(None, C.byref(place()[0]), C.byref(L.W4LinearArgs(**LINEAR))) == 2


def test_linear_epilogues_stay_apart():
    """mz_linear has no plain fp32 epilogue."""
    a = L.LinearArgs(epilogue=L.EPI_F32, a=SOME, lda=64, w=SOME, m=64, n=64, k=64, out=SOME, ldo=64)
    with pytest.raises(L.MzError, match="mz_linear: bad epilogue"):
        L.check(L.lib().mz_linear(C.byref(NOBODY), C.byref(a)))


@pytest.mark.parametrize("group", [32, 64, 128])
def test_w4_definition(group):
    """Codes are the nearest, the extreme is met but for its scale's rounding, what is stored is what it stands for."""
    rng = np.random.default_rng(group)
    w = (rng.standard_normal((20, 256)) * 0.05).astype(np.float16)
    w[3, :group] = 0
    w[4, 0], w[5, 1] = np.nan, -np.inf
    w[6, :group] = 0.5
    w[7, 0], w[7, 1] = 2.0, -2.0  # alike in size: the negative one
    c, s = R.w4_codes(w, group)
    assert np.isnan(s[4, 0]) and np.isnan(s[5, 0]) and s[3, 0] == 0 and (c[6, :group] == -8).all() and s[7, 0] == 0.25
    assert (c[7, :2] == [7, -8]).all()
    v, x = R.w4_values(c, s, group), w.astype(np.float64)
    d = np.repeat(np.abs(s.astype(np.float64)), group, 1)
    ok = ~np.isnan(v)
    assert (np.abs(v - x)[ok] <= np.where(c == 7, 1.01, 0.5 * (1 + 2.0 ** -40))[ok] * d[ok]).all()
    words, scales = R.w4_bytes_of(c, s, group)
    for n, k in ((0, 0), (7, 1), (19, 255), (16, 128), (13, 77)):
        t, i, ch, sw, j, e = n // 16, n % 16, k // 128, k % 128 // 32, k % 32 // 8, k % 8
        word = int.from_bytes(words[t, ch, 16 * j + i, 4 * sw:4 * sw + 4].tobytes(), "little")
        assert (word >> (4 * (e // 2) + 16 * (e % 2)) & 15) - 8 == c[n, k]
        assert scales[t, ch, i, k % 128 // group] == s[n, k // group]
    assert (words.reshape(2, 2, 4, 16, 16)[1, :, :, 4:] == 0x88).all()  # rows that pad


# ---------------------------------------------------------------- attention


CROSS = dict(q=SOME, out=SOME, q_row=512, q_token=512, q_head=64, out_row=512, out_token=512, out_head=64, k=SOME, v=SOME,
             k_slot=64 * 4 * 10, k_pos=64, k_head=640, v_slot=64 * 4 * 10, v_pos=64, v_head=640, rows=2, tokens=1, heads=8,
             kv_heads=4, slots=2, positions=10, scale=0.125)


@pytest.mark.parametrize("fn", ["mz_cross_attention", "mz_cross_attention_bytes"])
def test_cross_refuses(fn):
    def call(**change):
        a, n = L.CrossArgs(**{**CROSS, **change}), C.c_size_t(5)
        more = (C.byref(n),) if fn.endswith("bytes") else ()
        L.check(getattr(L.lib(), fn)(C.byref(NOBODY), C.byref(a), *more))
        assert not more or n.value == 0

    for bad in (dict(rows=-1), dict(tokens=-1), dict(slots=-1), dict(positions=-1), dict(heads=0), dict(kv_heads=0),
                dict(heads=6), dict(heads=4 * 65), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(q=0), dict(out=0), dict(q=SOME + 8), dict(out=SOME + 2), dict(k=0), dict(v=0),
                dict(k=SOME + 8), dict(v=SOME + 4), dict(slot=SOME + 1), dict(count=SOME + 2), dict(first=SOME + 3),
                dict(len=SOME + 1), dict(lse=SOME + 2), dict(align=SOME + 1), dict(q_head=60), dict(q_row=-8),
                dict(k_pos=60), dict(k_slot=-64), dict(v_head=4), dict(v_slot=1 << 47), dict(k_pos=1 << 44, positions=100),
                dict(k_pos=(1 << 24) + 8), dict(v_pos=(1 << 24) + 8),
                dict(out_row=0), dict(out_head=32), dict(out_token=64, tokens=2, out_row=4096), dict(align=SOME),
                dict(align=SOME, head_slot=SOME, align_heads=0, align_cols=4),
                dict(align=SOME, head_slot=SOME, align_heads=2, align_cols=0), dict(out_row=1 << 47),
                dict(tokens=1 << 30, rows=1 << 30), dict(rows=1 << 21), dict(tokens=1 << 20)):
        with pytest.raises(L.MzError, match=fn):
            call(**bad)
    call(rows=0)
    call(tokens=0)
    call(rows=0, k=0, v=0, positions=0)
    assert L.lib().mz_cross_attention(None, C.byref(L.CrossArgs(**CROSS))) == 2


@pytest.mark.parametrize("fn", ["mz_cross_attention", "mz_cross_attention_bytes"])
@pytest.mark.parametrize("positions", [(1 << 30) + 1, (1 << 31) - 1])
def test_cross_refuses_more_positions_than_it_can_count(fn, positions):
    a = L.CrossArgs(**{**CROSS, "positions": positions, "k_pos": 0, "v_pos": 0})
    with pytest.raises(L.MzError, match=fn):
        L.check(getattr(L.lib(), fn)(C.byref(NOBODY), C.byref(a), *((C.byref(C.c_size_t()),) if fn.endswith("bytes") else ())))


def test_cross_definition():
    rng = np.random.default_rng(3)
    q = rng.standard_normal((2, 3, 4, 64)).astype(np.float16)
    k, v = (rng.standard_normal((2, 9, 2, 64)).astype(np.float16) for _ in range(2))
    r = R.cross(q, k, v, slot=[1, 0], first=[2, 0], length=[8, 20], count=[3, 1])
    t = lambda x: torch.from_numpy(x.astype(np.float64))  # noqa: E731
    kk, vv = (t(x[1, 2:8]).repeat_interleave(2, 1).transpose(0, 1) for x in (k, v))
    want = torch.nn.functional.scaled_dot_product_attention(t(q[0]).transpose(0, 1), kk, vv).transpose(0, 1)
    np.testing.assert_allclose(r["out"][0], want.numpy(), rtol=1e-12)
    assert np.isnan(r["out"][1, 1:]).all() and np.isfinite(r["out"][1, 0]).all() and (r["p"][0, ..., :2] == 0).all()


# ---------------------------------------------------------------- the next token


SAMPLE = dict(dtype=L.DT_F32, rows=2, vocab=100, logits=SOME, ld=100, temperature=1.0, top_p=1.0, u=SOME, tokens=SOME, stride=1)


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(rows=-1), dict(rows=1 << 22), dict(vocab=0), dict(vocab=(1 << 30) + 1, ld=1 << 31),
                                 dict(ld=99), dict(ld=1 << 50), dict(logits=0), dict(logits=SOME + 2),
                                 dict(dtype=L.DT_F16, logits=SOME + 1), dict(u=0), dict(u=SOME + 1), dict(tokens=0),
                                 dict(tokens=SOME + 2), dict(logp=SOME + 1), dict(kept=SOME + 3), dict(at=SOME + 1),
                                 dict(temperatures=SOME + 2), dict(top_ks=SOME + 1), dict(top_ps=SOME + 1),
                                 dict(min_ps=SOME + 2), dict(temperature=-0.5), dict(temperature=float("nan")),
                                 dict(temperature=float("inf")), dict(top_p=float("nan")), dict(min_p=float("nan")),
                                 dict(stride=0), dict(stride=-1), dict(stride=1 << 46)])
def test_sample_refuses(bad):
    a, n = L.SampleArgs(**{**SAMPLE, **bad}), C.c_size_t()
    for call in (lambda: L.lib().mz_sample(C.byref(NOBODY), C.byref(a)),
                 lambda: L.lib().mz_sample_bytes(C.byref(NOBODY), C.byref(a), C.byref(n))):
        with pytest.raises(L.MzError, match="mz_sample"):
            L.check(call())


def test_sample_of_no_rows():
    a, n = L.SampleArgs(**{**SAMPLE, "rows": 0}), C.c_size_t(3)
    assert L.lib().mz_sample(C.byref(NOBODY), C.byref(a)) == 0
    assert L.lib().mz_sample_bytes(C.byref(NOBODY), C.byref(a), C.byref(n)) == 0 and n.value == 0
    assert L.lib().mz_sample(None, C.byref(a)) == 2


def test_sample_definition():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.2, 0.1]))
    got = lambda u, **kw: R.sample(x, u, **kw)[:3:2]  # (token, kept)  # noqa: E731
    assert [got(u)[0] for u in (0.0, 0.05, 0.11, 0.49, 0.51, 0.71, 0.91)] == [0, 0, 1, 1, 2, 3, 4]
    assert got(0.99, temperature=0.0) == (1, 1)
    assert got(0.99, top_k=2) == (2, 2) and got(0.6, top_k=2) == (1, 2)  # the lower of two equal ones
    assert got(0.9, top_p=0.5) == (2, 2) and got(0.9, top_p=0.3) == (1, 1) and got(0.1, top_p=0.0) == (1, 1)
    assert got(0.9, top_k=3, top_p=0.7) == (2, 2)  # 0.4 + 0.2 of 0.8: three quarters
    assert got(0.9, min_p=0.4) == (3, 3) and got(0.9, min_p=7.0) == (1, 1)
    assert R.sample(x, 0.4, mask=np.array([0, 1, 0, 0, 0]))[0] == 2
    assert R.sample(np.full(4, -np.inf), 0.5)[:3] == (-1, -np.inf, 0)
    assert R.sample([0.0, np.nan], 0.5)[0] == -1 and R.sample([0.0, 1.0], 0.5, temperature=-1)[0] == -1
    np.testing.assert_allclose(R.sample(x, 0.2, top_k=2)[1], np.log(2 / 3))


@pytest.mark.parametrize("min_p", [np.nextafter(np.float32(1), np.float32(2)), 2.0, np.inf])
def test_sample_definition_of_a_share_that_no_token_has(min_p):
    """Above 1 there is no token of weight min_p or more, also not where several are the largest: the first alone is kept."""
    assert R.sample([1.0, 1.0, 0.0], 0.9, min_p=min_p)[:3] == (0, 0.0, 1)
    assert R.sample([0.0, 1.0, 1.0, 1.0], 0.9, min_p=min_p, top_k=2, top_p=0.99)[:3] == (1, 0.0, 1)
    assert R.sample([1.0, 1.0, 0.0], 0.9, min_p=1.0)[::2][:2] == (1, 2)
