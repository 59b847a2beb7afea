"""The operators of decoding with caches held in 8 bits, and of scoring what was decoded, as cases that can be timed.

Three kinds of pass:

  write   keys and values of new positions into an 8-bit cache (mz_kv8_write: whole prompts or encoder outputs, or one
          position of each row), and what the cache then holds of the blocks they are in (mz_kv8_read)
  attend  attention of one or several query positions over such a cache (mz_kv8_attention): a decoder step over its
          self-attention cache or over the encoder's keys, beams that share a cache, prompts under a causal mask
  score   log probabilities of given tokens with the entropy and the best alternatives of each row of logits
          (mz_token_scores)

A cache holds blocks of 32 positions x 64 channels per (slot, head): 8-bit codes and one scale for the keys' block, one
for the values'. Values are kept by pairs of channels and groups of eight positions. Code c stands for c * scale;
scale = the block's largest magnitude / 127 (signed whole numbers, "i8") or / 448 (OCP e4m3). A block that is not full
yet is held as it was given, in fp16 and in the same order, until its last position arrives.
"""
import math

import torch

own = False

HD, BLK, TENC, MAX_T = 64, 32, 1500, 448
TOP = {"i8": 127.0, "e4m3": 448.0}
HEADS = (6, 8, 12, 16, 20)  # widths 384 to 1280
VOCABS = (51864, 51865, 51866)


def listed():
    return [
        # the encoder's keys and values of a group of eight clips, one layer of the widest model
        {"name": "write_cross_8", "kind": "write", "format": "i8", "rows": 8, "heads": 20, "tokens": TENC, "max_t": TENC,
         "layout": "tiles", "past": 0, "ragged": False},
        # a decoder step of a batch: one position of each row, each row at its own place
        {"name": "write_step_32", "kind": "write", "format": "e4m3", "rows": 32, "heads": 20, "tokens": 1,
         "max_t": MAX_T, "layout": "rows", "past": 223, "ragged": True},
        # the first steps of one request on the smallest model: latency
        {"name": "attend_self_1", "kind": "attend", "format": "i8", "rows": 1, "heads": 6, "group": 1, "tokens": 1,
         "past": 37, "max_t": MAX_T, "causal": True, "ragged": False, "slots": "own", "align": 0, "first": False},
        # a batch in the middle of its transcripts, the widest model
        {"name": "attend_self_32", "kind": "attend", "format": "e4m3", "rows": 32, "heads": 20, "group": 1, "tokens": 1,
         "past": 410, "max_t": MAX_T, "causal": True, "ragged": True, "slots": "mixed", "align": 0, "first": True},
        # one request over the encoder's positions, with alignment rows for the timestamps
        {"name": "attend_cross_1", "kind": "attend", "format": "i8", "rows": 1, "heads": 20, "group": 1, "tokens": 1,
         "past": TENC, "max_t": TENC, "causal": False, "ragged": False, "slots": "own", "align": 6, "first": False},
        # the benchmark's batch over the encoder's positions: what most of a decoder step's time goes to
        {"name": "attend_cross_32", "kind": "attend", "format": "i8", "rows": 32, "heads": 20, "group": 1, "tokens": 1,
         "past": TENC, "max_t": TENC, "causal": False, "ragged": False, "slots": "own", "align": 6, "first": False},
        # five beams of each of sixteen clips: the beams of a clip read the same cache
        {"name": "attend_beams_16x5", "kind": "attend", "format": "e4m3", "rows": 16, "heads": 16, "group": 1,
         "tokens": 5, "past": TENC, "max_t": TENC, "causal": False, "ragged": False, "slots": "mixed", "align": 0,
         "first": False},
        # prompts of previous text in one call, padded to the longest
        {"name": "attend_prompt_8x224", "kind": "attend", "format": "i8", "rows": 8, "heads": 20, "group": 1,
         "tokens": 224, "past": 150, "max_t": MAX_T, "causal": True, "ragged": True, "slots": "own", "align": 0,
         "first": False},
        # a few long sequences whose query heads share keys and values
        {"name": "attend_long_6", "kind": "attend", "format": "e4m3", "rows": 6, "heads": 16, "group": 2, "tokens": 1,
         "past": 16001, "max_t": 16384, "causal": True, "ragged": True, "slots": "own", "align": 0, "first": False},
        # the token that one decoder step chose, with five alternatives
        {"name": "score_1", "kind": "score", "dtype": "f32", "rows": 1, "vocab": 51865, "alts": 5, "mask": True},
        # the same for the benchmark's batch
        {"name": "score_32", "kind": "score", "dtype": "f32", "rows": 32, "vocab": 51866, "alts": 5, "mask": True},
        # every position of a batch of transcripts at once: their confidence
        {"name": "score_7040", "kind": "score", "dtype": "f32", "rows": 7040, "vocab": 51866, "alts": 1, "mask": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "attend", "attend", "score"])
    fmt = rng.choice(["i8", "e4m3"])
    if kind == "score":
        return {"kind": kind, "dtype": rng.choice(["f32", "f16"]), "rows": _log_int(rng, 1, 5000),
                "vocab": rng.choice(VOCABS + (_log_int(rng, 300, 51800),)), "alts": rng.randint(0, 8),
                "mask": rng.random() < 0.5}
    heads = rng.choice(HEADS)
    if kind == "write":
        tokens = 1 if rng.random() < 0.3 else _log_int(rng, 2, TENC)
        past = 0 if rng.random() < 0.3 else _log_int(rng, 1, MAX_T)
        return {"kind": kind, "format": fmt, "rows": _log_int(rng, 1, max(1, min(64, 150000 // (tokens * heads)))),
                "heads": heads, "tokens": tokens, "max_t": past + tokens + rng.randint(0, 40),
                "layout": rng.choice(["tiles", "rows"]), "past": past, "ragged": rng.random() < 0.6}
    what = rng.choice(["self", "cross", "beams", "prompt", "long"])
    c = {"kind": kind, "format": fmt, "rows": _log_int(rng, 1, 32), "heads": heads, "group": 1, "tokens": 1,
         "past": TENC, "max_t": TENC, "causal": False, "ragged": False, "slots": rng.choice(["own", "mixed"]),
         "align": 0, "first": False}
    if what == "self":
        c.update(past=_log_int(rng, 1, MAX_T - 1), max_t=MAX_T, causal=True, ragged=rng.random() < 0.7,
                 first=rng.random() < 0.5)
    elif what == "cross":
        c.update(align=rng.choice([0, rng.randint(1, heads)]))
    elif what == "beams":
        c.update(rows=_log_int(rng, 1, 16), tokens=rng.randint(2, 8))
    elif what == "prompt":
        t = _log_int(rng, 2, 224)
        c.update(rows=_log_int(rng, 1, 8), tokens=t, past=rng.randint(0, MAX_T - t), max_t=MAX_T, causal=True,
                 ragged=rng.random() < 0.7)
    else:
        g = rng.choice([1, 2, 4])
        past = _log_int(rng, 449, 16000)
        c.update(rows=_log_int(rng, 1, 6), heads=rng.choice([4, 8, 16]), group=g, tokens=rng.choice([1, 1, 3]),
                 past=past, max_t=past + rng.randint(3, 400), causal=True, ragged=rng.random() < 0.7)
    return c


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, std=1.0, dtype=torch.float16):
    return torch.randn(shape, generator=g, device="cuda").mul_(std).to(dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _spread(n, top, ragged, low):
    """A length for each of n rows, the first one the longest: requests are at different places."""
    return [max(low, int(top * (1.0 - 0.45 * ((5 * i) % 11) / 11.0))) if ragged else max(low, top) for i in range(n)]


def _divided(x, fmt):
    """(codes as the numbers they are, scales) of blocks x [..., 32, 64]."""
    x = x.float()
    top = x.abs().amax((-1, -2), keepdim=True)
    c = torch.where(top > 0, x * TOP[fmt] / top, torch.zeros_like(x))
    c = torch.round(c) if fmt == "i8" else c.to(torch.float8_e4m3fn).float()
    return c, (top / TOP[fmt])[..., 0, 0]


def _as_codes(c, fmt):
    return (c.to(torch.int8) if fmt == "i8" else c.to(torch.float8_e4m3fn)).view(torch.uint8)


def _as_numbers(codes, fmt):
    return (codes.view(torch.int8) if fmt == "i8" else codes.view(torch.float8_e4m3fn)).float()


def _value_order(c):
    """Blocks [..., 32 positions, 64 channels] in the order a cache keeps values: [..., 32 channel pairs][4 groups of
    positions][2 channels][8 positions]."""
    return c.unflatten(-2, (4, 8)).unflatten(-1, (32, 2)).movedim((-2, -4, -1, -3), (-4, -3, -2, -1)).contiguous()


def _from_value_order(c):
    return c.movedim((-4, -3, -2, -1), (-2, -4, -1, -3)).flatten(-2, -1).flatten(-3, -2)


def _natural(kv, name):
    """Codes and open blocks of the keys or the values, positions by channels."""
    if name == "k":
        return kv["k"], kv["k_open"]
    return _from_value_order(kv["v"]).contiguous(), _from_value_order(kv["v_open"]).contiguous()


def _cache(case, g, slots, heads, held):
    """A cache whose slots hold `held` positions each; what lies behind them was left by earlier sequences."""
    fmt, blocks = case["format"], -(-case["max_t"] // BLK)
    kv = {"format": fmt, "slots": slots, "heads": heads, "blocks": blocks}
    at = _ints([h // BLK if h % BLK else -1 for h in held])
    kv["open"] = (at + 1)[:, None].repeat(1, heads).contiguous()
    for name in ("k", "v"):
        x = _randn(g, (slots, heads, blocks, BLK, HD), 0.7)
        c, s = _divided(x, fmt)
        c = _as_codes(c, fmt).reshape(slots, heads, blocks, BLK, HD)
        kv[name] = c if name == "k" else _value_order(c)
        kv[name + "_scale"] = s.contiguous()
        x = _randn(g, (slots, heads, BLK, HD), 0.7)
        kv[name + "_open"] = x if name == "k" else _value_order(x)
    return kv


def _slots(case, n):
    """Where the rows' sequences are: in order, or wherever there was room in a cache of a few slots more."""
    if case.get("slots", "own") == "own":
        return n, list(range(n)), None
    r = torch.randperm(n + 2, generator=torch.Generator().manual_seed(7))[:n].tolist()
    return n + 2, r, _ints(r)


def _prepare_write(case, g, s):
    n, h, t = case["rows"], case["heads"], case["tokens"]
    past = _spread(n, case["past"], case["ragged"], 0)
    count = [t] * n if t == 1 else _spread(n, t, case["ragged"], 1)
    s["cache"] = _cache(case, g, n, h, past)
    shape = (n, h, t, HD) if case["layout"] == "tiles" else (n, t, h, HD)
    s["k"], s["v"] = (_randn(g, shape, 0.7) for _ in range(2))
    s["past"], s["count"] = _ints(past), _ints(count)
    # what is read back: every position of the blocks that the new ones are in, up to the last new one
    s["from"] = s["past"] // BLK * BLK
    s["held"] = s["past"] - s["from"] + s["count"]
    s["read"] = max(p % BLK + c for p, c in zip(past, count))
    s["out"] = {x: torch.zeros((n, h, s["read"], HD), device="cuda", dtype=torch.float16) for x in ("k", "v")}


def _prepare_attend(case, g, s):
    n, h, t = case["rows"], case["heads"], case["tokens"]
    past = _spread(n, case["past"], case["ragged"], 0)
    count = [t] * n if t == 1 or not case["causal"] else _spread(n, t, case["ragged"], 1)
    slots, where, s["slot"] = _slots(case, n)
    held = [0] * slots
    for w, p, c in zip(where, past, count):
        held[w] = p + c if case["causal"] else p
    s["cache"] = _cache(case, g, slots, h // case["group"], held)
    s["q"] = _randn(g, (n, t, h, HD), 1.5)
    s["past"], s["count"] = _ints(past), _ints(count)
    # left-padded rows: their first positions are no text
    s["first"] = _ints([(3 * i) % 7 if p > 16 else 0 for i, p in enumerate(past)]) if case["first"] else None
    s["out"] = {"out": torch.zeros((n, t, h, HD), device="cuda", dtype=torch.float16),
                "lse": torch.zeros((n, t, h), device="cuda")}
    if case["align"]:
        heads = [-1] * h
        for i in range(case["align"]):
            heads[(7 * i) % h] = i  # 7 and the counts of heads have no common factor
        s["head_slot"] = _ints(heads)
        s["out"]["align"] = torch.zeros((n, t, case["align"], TENC), device="cuda")


def _prepare_score(case, g, s):
    n, v = case["rows"], case["vocab"]
    dtype = torch.float32 if case["dtype"] == "f32" else torch.float16
    s["logits"] = torch.empty((n, v), device="cuda", dtype=dtype)
    s["tokens"] = torch.randint(0, v, (n,), generator=g, device="cuda", dtype=torch.int32)
    sure = torch.rand((n,), generator=g, device="cuda") * 16.0
    for i in range(0, n, 512):  # (in pieces: the whole in 32 bits twice over is not wanted)
        x = torch.randn((min(512, n - i), v), generator=g, device="cuda").mul_(2.5)
        x.scatter_add_(1, s["tokens"][i:i + 512].long()[:, None], sure[i:i + 512, None])
        s["logits"][i:i + 512] = x.to(dtype)
    if n > 8:  # padding behind shorter transcripts
        s["tokens"][torch.arange(n, device="cuda") % 37 == 36] = -1
    s["mask"] = (torch.rand((v,), generator=g, device="cuda") < 0.002).to(torch.uint8) if case["mask"] else None
    s["out"] = {"logp": torch.zeros((n,), device="cuda"), "entropy": torch.zeros((n,), device="cuda")}
    if case["alts"]:
        s["out"]["ids"] = torch.zeros((n, case["alts"]), device="cuda", dtype=torch.int32)
        s["out"]["best"] = torch.zeros((n, case["alts"]), device="cuda")


def prepare(case, seed):
    g, s = _gen(seed), {"case": case}
    {"write": _prepare_write, "attend": _prepare_attend, "score": _prepare_score}[case["kind"]](case, g, s)
    torch.cuda.synchronize()  # the library works on its own stream
    return s


# ---------------------------------------------------------------- the framework's calls


_ctx, _work = [], {}


def _context():
    if not _ctx:
        from mimizuku_amd import model
        _ctx.append(model.Context(0))
    return _ctx[0]


def _scratch(ctx, nbytes):
    """One workspace for every call of this program, which makes them one after the other on one stream."""
    if nbytes > _work.get("bytes", 0):
        _work.update(bytes=max(nbytes, 1 << 22), at=ctx.alloc(max(nbytes, 1 << 22)))
    return _work.get("at", 0), _work.get("bytes", 0)


def _at(t):
    return 0 if t is None else t.data_ptr()


def _calls(s):
    """The calls of a pass with their arguments filled in, as a program does once for the buffers it keeps."""
    from mimizuku_amd import _lib as L
    from mimizuku_amd import decode8
    ctx, case, lib = _context(), s["case"], L.lib()
    if case["kind"] == "score":
        v, n = case["vocab"], case["rows"]
        a = L.ScoreArgs(dtype=L.DT_F32 if case["dtype"] == "f32" else L.DT_F16, rows=n, vocab=v, alts=case["alts"],
                        logits=_at(s["logits"]), ld=v, mask=_at(s["mask"]), tokens=_at(s["tokens"]), token_stride=1,
                        logp=_at(s["out"]["logp"]), entropy=_at(s["out"]["entropy"]), out_stride=1,
                        alt_ids=_at(s["out"].get("ids")), alt_logp=_at(s["out"].get("best")))
        a.work, a.work_bytes = _scratch(ctx, decode8.scores_bytes(ctx, a))
        return [(lib.mz_token_scores, ctx.h, a)], [s["logits"]]
    kv = s["cache"]
    cache = L.Kv8(L.KV8_I8 if kv["format"] == "i8" else L.KV8_E4M3, kv["slots"], kv["heads"], kv["blocks"],
                  *[kv[x].data_ptr() for x in ("k", "v", "k_scale", "v_scale", "k_open", "v_open", "open")])
    if case["kind"] == "write":
        n, h, t, r = case["rows"], case["heads"], case["tokens"], s["read"]
        row, token, head = (h * t * HD, HD, t * HD) if case["layout"] == "tiles" else (t * h * HD, h * HD, HD)
        w = L.Kv8Io(k=_at(s["k"]), v=_at(s["v"]), row_stride=row, token_stride=token, head_stride=head, rows=n, tokens=t,
                    pos=_at(s["past"]), pos_stride=1, pos_add=0, count=_at(s["count"]))
        b = L.Kv8Io(k=_at(s["out"]["k"]), v=_at(s["out"]["v"]), row_stride=h * r * HD, token_stride=HD,
                    head_stride=r * HD, rows=n, tokens=r, pos=_at(s["from"]), pos_stride=1, pos_add=0,
                    count=_at(s["held"]))
        return [(lib.mz_kv8_write, ctx.h, cache, w), (lib.mz_kv8_read, ctx.h, cache, b)], []
    n, h, t = case["rows"], case["heads"], case["tokens"]
    a = L.Kv8Attention(q=_at(s["q"]), q_row=t * h * HD, q_token=h * HD, q_head=HD, out=_at(s["out"]["out"]),
                       out_row=t * h * HD, out_token=h * HD, out_head=HD, rows=n, tokens=t, heads=h,
                       causal=int(case["causal"]), scale=0.125, slot=_at(s["slot"]), count=_at(s["count"]),
                       len=_at(s["past"]), len_stride=1, len_add=int(case["causal"]), first=_at(s["first"]),
                       lse=_at(s["out"]["lse"]), head_slot=_at(s.get("head_slot")), align=_at(s["out"].get("align")),
                       align_heads=case["align"], align_cols=TENC if case["align"] else 0)
    a.work, a.work_bytes = _scratch(ctx, decode8.attention_bytes(ctx, cache, a))
    return [(lib.mz_kv8_attention, ctx.h, cache, a)], []


def _run_own(s):
    from mimizuku_amd._lib import check
    if "calls" not in s:
        s["calls"], s["kept"] = _calls(s)
    for fn, *args in s["calls"]:
        check(fn(*args))
    return s["out"]


# ---------------------------------------------------------------- the plain form


def _write(s):
    """The window of positions from the start of each row's first block: what the cache holds of that block, then the
    new positions; whole blocks of it go through codes and scales, an unfinished one stays."""
    case, kv = s["case"], s["cache"]
    fmt, n, h, t = case["format"], case["rows"], case["heads"], case["tokens"]
    blocks = -(-s["read"] // BLK)
    i = torch.arange(blocks * BLK, device="cuda")
    off = (s["past"] - s["from"]).long()
    b0 = (s["from"] // BLK).long().clamp(max=kv["blocks"] - 1)
    rows = torch.arange(n, device="cuda")
    out = {}
    for name in ("k", "v"):
        x = s[name] if case["layout"] == "tiles" else s[name].transpose(1, 2)
        src = (i[None] - off[:, None]).clamp(0, t - 1)
        new = torch.gather(x, 2, src[:, None, :, None].expand(n, h, blocks * BLK, HD))
        c, o = _natural(kv, name)
        old = (_as_numbers(c[rows, :, b0], fmt) * kv[name + "_scale"][rows, :, b0][..., None, None]).half()
        old = torch.where((kv["open"] == (b0 + 1)[:, None])[..., None, None], o, old)
        old = torch.nn.functional.pad(old, (0, 0, 0, (blocks - 1) * BLK))
        x = torch.where((i[None] < off[:, None])[:, None, :, None], old, new).unflatten(2, (blocks, BLK))
        c, sc = _divided(x, fmt)
        last = torch.arange(1, blocks + 1, device="cuda") * BLK
        full = (last[None] <= s["held"][:, None])[:, None, :, None, None]
        x = torch.where(full, (c * sc[..., None, None]).half(), x).flatten(2, 3)
        x = torch.where((i[None] < s["held"][:, None])[:, None, :, None], x, torch.zeros_like(x))
        out[name] = x[:, :, :s["read"]].contiguous()
    return out


def _held(kv, name):
    """Every position of a cache in 32 bits: [slots, heads, positions, 64]."""
    c, o = _natural(kv, name)
    x = _as_numbers(c, kv["format"]) * kv[name + "_scale"][..., None, None]
    b = torch.arange(1, kv["blocks"] + 1, device="cuda", dtype=torch.int32)
    x = torch.where((kv["open"][..., None] == b)[..., None, None], o.float()[:, :, None], x)
    return x.flatten(2, 3)


def _seen(s, n_pos):
    """[rows, tokens, positions]: which positions each query sees."""
    case = s["case"]
    i = torch.arange(case["tokens"], device="cuda")
    end = s["past"].long()[:, None] + (i[None] + 1 if case["causal"] else 0 * i[None])
    j = torch.arange(n_pos, device="cuda")
    m = j[None, None] < end[..., None]
    if s["first"] is not None:
        m = m & (j[None, None] >= s["first"].long()[:, None, None])
    return m


def _attend(s):
    case, kv = s["case"], s["cache"]
    n, h, t, grp = case["rows"], case["heads"], case["tokens"], case["group"]
    k, v = _held(kv, "k"), _held(kv, "v")
    if s["slot"] is not None:
        k, v = k[s["slot"].long()], v[s["slot"].long()]
    # the query heads of a group beside each other: [rows, cache heads, group * tokens, 64]
    q = s["q"].float().permute(0, 2, 1, 3).reshape(n, h // grp, grp * t, HD)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(n, h // grp, grp, t, -1) * 0.125
    x = x.masked_fill(~_seen(s, k.shape[2])[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    e = torch.exp(x - top)
    z = e.sum(-1, keepdim=True)
    p = e / torch.where(z > 0, z, torch.ones_like(z))
    o = torch.matmul(p.view(n, h // grp, grp * t, -1), v).view(n, h, t, HD).transpose(1, 2)
    there = torch.arange(t, device="cuda")[None] < s["count"][:, None]
    lse = (torch.log(z) + top).view(n, h, t).transpose(1, 2)
    out = {"out": torch.where(there[..., None, None], o, torch.zeros_like(o)).half(),
           "lse": torch.where(there[..., None], lse, torch.zeros_like(lse))}
    if case["align"]:
        of = torch.argsort(torch.where(s["head_slot"] < 0, h, s["head_slot"]))[:case["align"]]
        out["align"] = p.view(n, h, t, -1)[:, of, :, :TENC].transpose(1, 2).contiguous()
    return out


def _score(s):
    case = s["case"]
    x = s["logits"].float()
    if s["mask"] is not None:
        x = x.masked_fill(s["mask"].bool()[None], -math.inf)
    x = x - x.amax(-1, keepdim=True)
    e = torch.exp(x)
    z = e.sum(-1, dtype=torch.float64)
    lz = torch.log(z)
    hx = torch.where(e > 0, e * x, torch.zeros_like(x)).sum(-1, dtype=torch.float64)
    tok = s["tokens"].long()
    lp = torch.gather(x, 1, tok.clamp(min=0)[:, None])[:, 0].double() - lz
    out = {"logp": torch.where(tok < 0, torch.zeros_like(lp), lp).float(), "entropy": (lz - hx / z).float()}
    if case["alts"]:
        ids, best = [], []
        for _ in range(case["alts"]):  # the largest left, ties to the lowest id
            b, i = x.max(-1)
            best.append((b.double() - lz).float())
            ids.append(i.int())
            x.scatter_(1, i[:, None], -math.inf)
        out["ids"], out["best"] = torch.stack(ids, 1), torch.stack(best, 1)
    return out


def run(s):
    if own:
        return _run_own(s)
    return {"write": _write, "attend": _attend, "score": _score}[s["case"]["kind"]](s)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["kind"] == "score":
        n, v = case["rows"], case["vocab"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": n * v * size + (v if case["mask"] else 0) + n * (12 + 8 * case["alts"]), "flops": 6 * n * v}
    n, h, t = case["rows"], case["heads"], case["tokens"]
    past = _spread(n, case["past"], case["ragged"], 0)
    if case["kind"] == "write":
        count = [t] * n if t == 1 else _spread(n, t, case["ragged"], 1)
        vals = 0
        for p, c in zip(past, count):
            off, e = p % BLK, p % BLK + c
            vals += c * 2 + (off * 2 if e >= BLK else 0)  # the new positions, and the open block once it is full
            vals += e // BLK * BLK + (e - max(off, e // BLK * BLK)) * 2  # codes, and what stays as it was given
            vals += e * 2  # what is read back
        return {"bytes": 2.0 * h * HD * vals, "flops": 2.0 * 6 * n * h * t * HD}
    count = [t] * n if t == 1 or not case["causal"] else _spread(n, t, case["ragged"], 1)
    ends = [p + c if case["causal"] else p for p, c in zip(past, count)]
    keys = sum(e // BLK * BLK + 2 * (e % BLK) for e in ends) * (h // case["group"])
    pairs = sum(c * p + (c * (c + 1) // 2 if case["causal"] else 0) for p, c in zip(past, count)) * h
    return {"bytes": 2.0 * HD * keys + sum(count) * h * (4 * HD + 4) + 4.0 * n * t * case["align"] * TENC,
            "flops": 4.0 * HD * pairs}


# ---------------------------------------------------------------- the same in 64 bits, from the definitions


def _step_of(v, fmt):
    """v in 64 bits rounded to the numbers that codes stand for, halves to even."""
    if fmt == "i8":
        return torch.round(v)
    _, e = torch.frexp(v)
    unit = torch.ldexp(torch.ones_like(v), (e - 4).clamp(min=-9))
    return torch.round(v / unit) * unit


def _numbers64(codes, fmt):
    b = codes.to(torch.int64)
    if fmt == "i8":
        return torch.where(b > 127, b - 256, b).double()
    e, m = (b >> 3) & 15, (b & 7).double()
    x = torch.where(e > 0, torch.ldexp(1.0 + m / 8.0, e - 7), m / 512.0)
    return torch.where(b > 127, -x, x)


def _position64(kv, name, slot, p):
    """What one position of a slot stands for: [heads, 64] in 64 bits."""
    b, i = p // BLK, p % BLK
    c = kv[name][slot, :, b, i] if name == "k" else kv[name][slot, :, b, :, i // 8, :, i % 8].flatten(1)
    x = _numbers64(c, kv["format"]) * kv[name + "_scale"][slot, :, b].double()[:, None]
    still = kv["open"][slot] == b + 1
    o = kv["k_open"][slot, :, i] if name == "k" else kv["v_open"][slot, :, :, i // 8, :, i % 8].flatten(1)
    return torch.where(still[:, None], o.double(), x)


def _exact_write(case, s):
    fmt, out = case["format"], {}
    for name in ("k", "v"):
        x = s[name] if case["layout"] == "tiles" else s[name].transpose(1, 2)
        y = torch.zeros(s["out"][name].shape, device="cuda", dtype=torch.float64)
        for r in range(case["rows"]):
            p, c = int(s["past"][r]), int(s["count"][r])
            f = p // BLK * BLK
            w = [_position64(s["cache"], name, r, j).half().double() for j in range(f, p)]
            w = torch.cat([y[:, None] for y in w] + [x[r, :, :c].double()], 1)
            for j in range(0, w.shape[1] - BLK + 1, BLK):
                top = w[:, j:j + BLK].abs().amax((1, 2), keepdim=True)
                scale = (top / TOP[fmt]).float().double()  # held in 32 bits
                w[:, j:j + BLK] = _step_of(w[:, j:j + BLK] * TOP[fmt] / top, fmt) * scale
            y[r, :, :w.shape[1]] = w
        out[name] = y
    return out


def _exact_attend(case, s):
    kv, fmt = s["cache"], case["format"]
    n, h, t, grp = case["rows"], case["heads"], case["tokens"], case["group"]
    where = list(range(n)) if s["slot"] is None else s["slot"].tolist()
    o = torch.zeros((n, t, h, HD), device="cuda", dtype=torch.float64)
    lse = torch.zeros((n, t, h), device="cuda", dtype=torch.float64)
    align = torch.zeros((n, t, case["align"], TENC), device="cuda", dtype=torch.float64)
    for r in range(n):
        w, p, c = where[r], int(s["past"][r]), int(s["count"][r])
        k = _numbers64(kv["k"][w], fmt) * kv["k_scale"][w].double()[..., None, None]
        v = _numbers64(kv["v"][w], fmt).permute(0, 1, 3, 5, 2, 4).reshape(k.shape)
        v = v * kv["v_scale"][w].double()[..., None, None]
        b = int(kv["open"][w, 0]) - 1
        if b >= 0:
            k[:, b] = kv["k_open"][w].double()
            v[:, b] = kv["v_open"][w].double().permute(0, 2, 4, 1, 3).reshape(k[:, b].shape)
        k, v = k.flatten(1, 2), v.flatten(1, 2)
        lo = 0 if s["first"] is None else int(s["first"][r])
        for a in range(h):
            end = p + c if case["causal"] else p
            x = s["q"][r, :c, a].double() @ k[a // grp, lo:end].T.contiguous() * 0.125
            if case["causal"]:
                j = torch.arange(lo, end, device="cuda")
                i = torch.arange(c, device="cuda")
                x = x.masked_fill(j[None] > p + i[:, None], -math.inf)
            lse[r, :c, a] = torch.logsumexp(x, -1)
            y = torch.softmax(x, -1)
            o[r, :c, a] = y @ v[a // grp, lo:end]
            if case["align"] and int(s["head_slot"][a]) >= 0:
                align[r, :c, int(s["head_slot"][a]), lo:min(end, TENC)] = y[:, :TENC - lo]
    return {"out": o, "lse": lse, **({"align": align} if case["align"] else {})}


def _exact_score(case, s):
    n, out = case["rows"], {}
    for i in range(0, n, 256):
        x = s["logits"][i:i + 256].double()
        if s["mask"] is not None:
            x[:, s["mask"].bool()] = -math.inf
        lp = torch.log_softmax(x, -1)
        tok = s["tokens"][i:i + 256].long()
        part = {"logp": torch.where(tok < 0, 0.0, lp.gather(1, tok.clamp(min=0)[:, None])[:, 0]),
                "entropy": -torch.xlogy(lp.exp(), lp.exp()).sum(-1)}
        if case["alts"]:
            y, ids = torch.sort(x, dim=-1, descending=True, stable=True)
            ids = ids[:, :case["alts"]]
            part.update(ids=ids.int(), best=lp.gather(1, ids))
        for name, v in part.items():
            out.setdefault(name, []).append(v)
    return {name: torch.cat(v) for name, v in out.items()}


def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "attend": _exact_attend, "score": _exact_score}[case["kind"]](case, s)
