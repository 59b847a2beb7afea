"""Attention over 8-bit caches where its definition is easily missed. Against oracle/decode8_ref.py (numpy, 64 bits); helpers and
the counting of roundings as in test_gpu_decode8.py."""
import numpy as np
import pytest
from test_gpu_decode8 import FMT, Both, H, U, ctx, dev, f16, run_attention  # noqa: F401

from oracle import decode8_ref as R

pytestmark = pytest.mark.gpu


def expected(b, q, causal, length, **kw):
    """Outputs and lse in 64 bits, and how far an output may be from them. Probabilities are carried with 16 bits or more (2^-16
    relative, of two roundings to 8 bits each) whatever their size, sums are of 32-bit numbers in any order (a score's error
    ds and n + 16 roundings u, relative to sum p |v|), the output is rounded once: h relative, or half its smallest step."""
    w, lse, prob, (av, aq) = R.attention(b.r, q, causal, length, **kw)
    rel = 2 * 80 * U * aq + ((prob > 0).sum(-1) + 16) * U + 2.0 ** -16
    return w, lse, rel[..., None] * av + H * np.abs(w) + 2.0 ** -25


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
