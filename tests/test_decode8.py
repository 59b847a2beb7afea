"""CPU checks of the 8-bit caches and the token scores: the layout, the structs' sizes as a C compiler sees them, the
refusals (none of which touches the device), and the definitions in oracle/decode8_ref.py against torch's own types."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest
import torch

from mimizuku_amd import _lib as L
from oracle import decode8_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOME = 0x10000  # an address that no refused call reads
NOBODY = C.create_string_buffer(4096)  # stands for a context: a refused call does not look at it


def place(fmt=L.KV8_I8, slots=2, heads=4, max_tokens=100, base=SOME):
    kv, n = L.Kv8(), C.c_size_t()
    L.check(L.lib().mz_kv8_place(fmt, slots, heads, max_tokens, base, C.byref(kv), C.byref(n)))
    return kv, n.value


def test_struct_layouts_match_the_header(tmp_path):
    """Offsets of every field as gcc lays the header's structs out against the Python mirror's."""
    pairs = [("mz_kv8", L.Kv8), ("mz_kv8_io", L.Kv8Io), ("mz_kv8_attention_args", L.Kv8Attention),
             ("mz_score_args", L.ScoreArgs)]
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


def test_place_lays_the_tensors_apart():
    kv, n = place(max_tokens=100)
    assert kv.blocks == 4
    sizes = {"k": 2 * 4 * 4 * 2048, "v": 2 * 4 * 4 * 2048, "k_scale": 2 * 4 * 4 * 4, "v_scale": 2 * 4 * 4 * 4,
             "k_open": 2 * 4 * 4096, "v_open": 2 * 4 * 4096, "open": 2 * 4 * 4}
    spans = sorted((getattr(kv, f), getattr(kv, f) + s) for f, s in sizes.items())
    assert spans[0][0] == SOME and spans[-1][1] <= SOME + n
    assert all(a[1] <= b[0] and b[0] % 256 == 0 for a, b in zip(spans, spans[1:]))
    # past 32 bits
    kv, n = place(slots=64, heads=20, max_tokens=200000)
    assert n > 2 * 64 * 20 * 200000 * 64 and kv.v - kv.k == 64 * 20 * 6250 * 2048


@pytest.mark.parametrize("bad", [dict(fmt=2), dict(fmt=-1), dict(slots=0), dict(heads=0), dict(max_tokens=0),
                                 dict(max_tokens=-5), dict(base=SOME + 8), dict(slots=1 << 30, heads=1 << 30)])
def test_place_refuses(bad):
    with pytest.raises(L.MzError, match="mz_kv8_place"):
        place(**bad)


IO = dict(k=SOME, v=SOME, row_stride=64 * 4 * 3, token_stride=64 * 4, head_stride=64, rows=2, tokens=3, pos_stride=1)


def io_call(fn, kv_change=None, **change):
    kv, _ = place()
    for f, v in (kv_change or {}).items():
        setattr(kv, f, v)
    L.check(getattr(L.lib(), fn)(C.byref(NOBODY), C.byref(kv), C.byref(L.Kv8Io(**{**IO, **change}))))


BAD_CACHE = [dict(format=7), dict(slots=0), dict(heads=-1), dict(blocks=0), dict(blocks=1 << 25), dict(k=0),
             dict(v=SOME + 8), dict(k_open=SOME + 2), dict(v_open=0), dict(k_scale=SOME + 2), dict(v_scale=0),
             dict(open=0)]


@pytest.mark.parametrize("fn", ["mz_kv8_write", "mz_kv8_read"])
def test_write_and_read_refuse(fn):
    for bad in BAD_CACHE:
        with pytest.raises(L.MzError, match=fn):
            io_call(fn, bad)
    for bad in (dict(rows=-1), dict(tokens=-1), dict(pos_stride=-1), dict(k=SOME + 8), dict(v=SOME + 2),
                dict(slot=SOME + 1), dict(pos=SOME + 2), dict(count=SOME + 3), dict(row_stride=-64),
                dict(token_stride=68), dict(head_stride=1 << 60)):
        with pytest.raises(L.MzError, match=fn):
            io_call(fn, **bad)
    for args in ((None, 1, 1), (1, None, 1), (1, 1, None)):
        ctx, kv, a = (x and y for x, y in zip(args, (C.byref(NOBODY), C.byref(place()[0]), C.byref(L.Kv8Io(**IO)))))
        assert getattr(L.lib(), fn)(ctx, kv, a) == 2
    with pytest.raises(L.MzError, match="too large"):
        io_call(fn, dict(slots=1 << 24), rows=1 << 24)
    # nothing to do is no error
    io_call(fn, rows=0)
    io_call(fn, tokens=0)


def test_write_needs_both_and_read_refuses_overlap():
    with pytest.raises(L.MzError, match="null k or v"):
        io_call("mz_kv8_write", v=0)
    io_call("mz_kv8_read", k=0, v=0)  # nothing wanted
    for bad in (dict(head_stride=56), dict(token_stride=64), dict(row_stride=64 * 4), dict(row_stride=0)):
        with pytest.raises(L.MzError, match="overlap"):
            io_call("mz_kv8_read", **bad)


ATT = dict(q=SOME, out=SOME, q_row=8 * 64, q_token=8 * 64, q_head=64, out_row=8 * 64, out_token=8 * 64, out_head=64,
           rows=2, tokens=1, heads=8, scale=0.125, len_stride=1)


def att_call(kv_change=None, fn="mz_kv8_attention", **change):
    kv, _ = place()
    for f, v in (kv_change or {}).items():
        setattr(kv, f, v)
    a = L.Kv8Attention(**{**ATT, **change})
    if fn.endswith("bytes"):
        n = C.c_size_t(5)
        L.check(L.lib().mz_kv8_attention_bytes(C.byref(NOBODY), C.byref(kv), C.byref(a), C.byref(n)))
        assert n.value == 0
    else:
        L.check(L.lib().mz_kv8_attention(C.byref(NOBODY), C.byref(kv), C.byref(a)))


@pytest.mark.parametrize("fn", ["mz_kv8_attention", "mz_kv8_attention_bytes"])
def test_attention_refuses(fn):
    for bad in BAD_CACHE:
        with pytest.raises(L.MzError, match=fn):
            att_call(bad, fn)
    for bad in (dict(rows=-1), dict(tokens=-2), dict(heads=0), dict(heads=6), dict(heads=4 * 65), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(len_stride=-1), dict(q=0),
                dict(q=SOME + 8), dict(out=0), dict(out=SOME + 2), dict(len=SOME + 1), dict(first=SOME + 2),
                dict(slot=SOME + 1), dict(count=SOME + 1), dict(lse=SOME + 1), dict(q_head=60), dict(q_row=-8),
                dict(out_row=0), dict(out_head=32), dict(out_token=64, tokens=2, out_row=4096),
                dict(align=SOME), dict(align=SOME, head_slot=SOME, align_heads=0, align_cols=4),
                dict(align=SOME, head_slot=SOME, align_heads=2, align_cols=0), dict(align=SOME + 1),
                dict(out_row=1 << 47), dict(tokens=1 << 30, rows=1 << 30), dict(rows=1 << 21), dict(tokens=1 << 20)):
        with pytest.raises(L.MzError, match=fn):
            att_call(None, fn, **bad)
    att_call(None, fn, rows=0)
    att_call(None, fn, tokens=0)


SC = dict(dtype=L.DT_F32, rows=2, vocab=100, alts=3, logits=SOME, ld=100, tokens=SOME, token_stride=1, logp=SOME,
          out_stride=1)


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(rows=-1), dict(vocab=0), dict(ld=99), dict(alts=-1), dict(alts=17),
                                 dict(logits=0), dict(logits=SOME + 2), dict(dtype=L.DT_F16, logits=SOME + 1),
                                 dict(tokens=0), dict(tokens=SOME + 2), dict(out_stride=0), dict(token_stride=-1),
                                 dict(logp=SOME + 1), dict(entropy=SOME + 2), dict(alt_ids=SOME + 1), dict(at=SOME + 1),
                                 dict(rows=1 << 24), dict(alt_logp=SOME + 3), dict(ld=1 << 50), dict(vocab=(1 << 30) + 1, ld=1 << 31)])
def test_scores_refuse(bad):
    a = L.ScoreArgs(**{**SC, **bad})
    n = C.c_size_t()
    for call in (lambda: L.lib().mz_token_scores(C.byref(NOBODY), C.byref(a)),
                 lambda: L.lib().mz_token_scores_bytes(C.byref(NOBODY), C.byref(a), C.byref(n))):
        with pytest.raises(L.MzError, match="mz_token_scores"):
            L.check(call())


def test_scores_of_no_rows():
    a, n = L.ScoreArgs(**{**SC, "rows": 0}), C.c_size_t(3)
    assert L.lib().mz_token_scores(C.byref(NOBODY), C.byref(a)) == 0
    assert L.lib().mz_token_scores_bytes(C.byref(NOBODY), C.byref(a), C.byref(n)) == 0 and n.value == 0


def test_codes_are_the_types_that_they_say():
    """Every e4m3 number's byte and every rounding to one against torch's float8_e4m3fn, whole numbers against int8."""
    b = np.arange(256, dtype=np.uint8)
    t = torch.from_numpy(b.copy()).view(torch.float8_e4m3fn).double().numpy()
    ok = ~np.isnan(t)
    np.testing.assert_array_equal(R.code_bytes(t[ok], "e4m3"), b[ok])
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.uniform(-448, 448, 20000), rng.uniform(-1, 1, 20000) * 2.0 ** -6, t[ok],
                        (t[ok][:-1] + t[ok][1:]) / 2]).astype(np.float32)
    x = x[np.abs(x) <= 448]
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    np.testing.assert_array_equal(R.to_code(x.astype(np.float64), "e4m3"), want)
    np.testing.assert_array_equal(R.code_bytes(np.arange(-127.0, 128), "i8"), np.arange(-127, 128).astype(np.int8).view(np.uint8))


@pytest.mark.parametrize("fmt", ["i8", "e4m3"])
def test_quotients_are_decided_in_32_bits(fmt):
    """Rounding T x / top taken in 32 bits to a code gives the real quotient's code for every fp16 magnitude x <= top: no
    quotient lies nearer to halfway between two codes than the 32-bit rounding moves it, unless it is exactly there."""
    every = np.arange(1, 0x7c00, dtype=np.uint16).view(np.float16).astype(np.float64)
    rng = np.random.default_rng(1)
    for top in rng.choice(every, 60):
        x = every[every <= top]
        y = np.float32(R.TOP[fmt]) * x.astype(np.float32)
        np.testing.assert_array_equal(y.astype(np.float64), R.TOP[fmt] * x)  # exact in 32 bits
        q = (y / np.float32(top)).astype(np.float64)
        np.testing.assert_array_equal(R.to_code(q, fmt), R.to_code(R.TOP[fmt] * x / top, fmt))


def test_value_order_is_the_documented_place():
    x = np.arange(2048, dtype=np.float64).reshape(32, 64)
    y = R.value_order(x).reshape(-1)
    for t in range(32):
        for d in range(64):
            assert y[(d // 2 * 4 + t // 8) * 16 + d % 2 * 8 + t % 8] == x[t, d]
