"""The operators of a decoder step of a caller's own, as cases that can be timed.

Three kinds of pass:

  w4      a product with 4-bit weights and a scale per group of columns (mz_w4_linear): projections of a decoder step, the
          logits, prompts
  cross   attention over the fp16 keys and values of an encoder's output of any length (mz_cross_attention): one token of
          each row, beams that share a clip, prompts
  sample  the next token with temperature, top-k, top-p and min-p from given random numbers (mz_sample)

Weights in 4 bits: of a group of 32, 64 or 128 columns of a row, with hi its maximum and lo its minimum, e = hi if hi > -lo else
lo, the scale is f16(e / -8) and code c, a whole number from -8 to 7, the nearest to w / scale, halves to even. c stands for
c * scale.

Sampling: with m a row's largest logit, weights are exp((x - m) / temperature). In the order of falling logits (of equal ones
the lower id first) those are kept that are among the first top_k, that are needed for top_p of the sum of weights of these
(the last one included), and whose weight is at least min_p; the first always is. The token is the lowest kept id up to
which the kept weights sum to more than u times their sum. Temperature 0: the first.
"""
import math

import torch

own = False

HD, TENC = 64, 1500
WIDTHS = (384, 512, 1024, 1280)
HEADS = (6, 8, 12, 16, 20)  # widths 384 to 1280
VOCABS = (51864, 51865, 51866)


def listed():
    return [
        # one request on the smallest model: its first feed-forward product, latency
        {"name": "w4_fc1_1", "kind": "w4", "m": 1, "n": 1536, "k": 384, "group": 32, "epilogue": "gelu", "bias": True},
        # a small batch on the widest model: its second feed-forward product, long rows
        {"name": "w4_fc2_8", "kind": "w4", "m": 8, "n": 1280, "k": 5120, "group": 64, "epilogue": "f16", "bias": True},
        # the logits of the benchmark's batch
        {"name": "w4_logits_32", "kind": "w4", "m": 32, "n": 51866, "k": 1280, "group": 32, "epilogue": "f32",
         "bias": False},
        # prompts of previous text, all of their positions at once
        {"name": "w4_prompt_1792", "kind": "w4", "m": 1792, "n": 5120, "k": 1280, "group": 128, "epilogue": "gelu",
         "bias": True},
        # one request with five seconds of audio on the smallest model: latency
        {"name": "cross_1", "kind": "cross", "rows": 1, "tokens": 1, "heads": 6, "group": 1, "positions": TENC, "len": 250,
         "layout": "tiles", "ragged": False, "slots": "own", "align": 0, "first": False},
        # the benchmark's batch with clips of many lengths and alignment rows for the timestamps, the widest model
        {"name": "cross_32", "kind": "cross", "rows": 32, "tokens": 1, "heads": 20, "group": 1, "positions": TENC,
         "len": TENC, "layout": "tiles", "ragged": True, "slots": "own", "align": 6, "first": False},
        # five beams of each of sixteen clips
        {"name": "cross_beams_16x5", "kind": "cross", "rows": 16, "tokens": 5, "heads": 16, "group": 1,
         "positions": TENC, "len": TENC, "layout": "rows", "ragged": False, "slots": "mixed", "align": 0,
         "first": False},
        # prompts of previous text over whole clips
        {"name": "cross_prompt_8x224", "kind": "cross", "rows": 8, "tokens": 224, "heads": 20, "group": 1,
         "positions": TENC, "len": TENC, "layout": "rows", "ragged": False, "slots": "own", "align": 0, "first": False},
        # one request's next token, with every limit
        {"name": "sample_1", "kind": "sample", "dtype": "f32", "rows": 1, "vocab": 51865, "temperature": 0.8,
         "top_k": 50, "top_p": 0.95, "min_p": 0.02, "mask": True},
        # the benchmark's batch, the most probable tokens up to nine tenths
        {"name": "sample_32", "kind": "sample", "dtype": "f32", "rows": 32, "vocab": 51866, "temperature": 0.6,
         "top_k": 0, "top_p": 0.9, "min_p": 0.0, "mask": True},
        # five candidates of each row by temperature alone, as where a transcript fails its checks
        {"name": "sample_160", "kind": "sample", "dtype": "f32", "rows": 160, "vocab": 51866, "temperature": 1.0,
         "top_k": 0, "top_p": 1.0, "min_p": 0.0, "mask": False},
        # a large batch of requests with settings of their own, some of them greedy
        {"name": "sample_1024", "kind": "sample", "dtype": "f16", "rows": 1024, "vocab": 51866, "temperature": "mixed",
         "top_k": "mixed", "top_p": "mixed", "min_p": "mixed", "mask": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["w4", "cross", "sample"])
    if kind == "w4":
        d = rng.choice(WIDTHS)
        n, k = rng.choice([(d, d), (4 * d, d), (d, 4 * d), (rng.choice(VOCABS), d), (_log_int(rng, 5, 3000), d)])
        m = _log_int(rng, 1, max(1, min(1792, 11_000_000_000 // (n * k))))
        return {"kind": kind, "m": m, "n": n, "k": k, "group": rng.choice([32, 64, 128]),
                "epilogue": rng.choice(["f16", "gelu", "f32"]), "bias": rng.random() < 0.6}
    if kind == "sample":
        return {"kind": kind, "dtype": rng.choice(["f32", "f16"]), "rows": _log_int(rng, 1, 500),
                "vocab": rng.choice(VOCABS + (_log_int(rng, 300, 51800),)),
                "temperature": rng.choice(["mixed", round(rng.uniform(0.1, 1.5), 3)]),
                "top_k": rng.choice(["mixed", 0, _log_int(rng, 1, 2000)]),
                "top_p": rng.choice(["mixed", 1.0, round(rng.uniform(0.05, 0.999), 3)]),
                "min_p": rng.choice(["mixed", 0.0, round(rng.uniform(0.001, 0.3), 4)]), "mask": rng.random() < 0.5}
    what = rng.choice(["step", "beams", "prompt", "long"])
    c = {"kind": kind, "rows": _log_int(rng, 1, 32), "tokens": 1, "heads": rng.choice(HEADS), "group": 1,
         "positions": TENC, "len": _log_int(rng, 1, TENC), "layout": rng.choice(["tiles", "rows"]),
         "ragged": rng.random() < 0.7, "slots": rng.choice(["own", "mixed"]), "align": 0, "first": rng.random() < 0.3}
    if what == "step":
        c.update(align=rng.choice([0, rng.randint(1, min(8, c["heads"]))]))
    elif what == "beams":
        c.update(rows=_log_int(rng, 1, 16), tokens=rng.randint(2, 8))
    elif what == "prompt":
        c.update(rows=_log_int(rng, 1, 8), tokens=_log_int(rng, 2, 224), len=rng.randint(300, TENC))
    else:  # several windows of audio at once, heads that share keys and values
        pos = _log_int(rng, TENC, 16000)
        c.update(rows=_log_int(rng, 1, 2), heads=rng.choice([4, 8, 16]), group=rng.choice([1, 2, 4]),
                 tokens=rng.choice([1, 1, 3]), positions=pos, len=pos - rng.randint(0, 300))
    return c


# ---------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, std=1.0, dtype=torch.float16):
    return torch.randn(shape, generator=g, device="cuda").mul_(std).to(dtype)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _floats(v):
    return torch.tensor(v, dtype=torch.float32, device="cuda")


def _coded(w, group):
    """(codes [n, k] i8, scales [n, k / group] f16) of weights in fp16."""
    x = w.unflatten(1, (-1, group)).float()
    hi, lo = x.amax(-1), x.amin(-1)
    s = (torch.where(hi > -lo, hi, lo) / -8.0).half()
    d = s.float()[..., None]
    c = torch.where(d != 0, torch.round(x / torch.where(d != 0, d, torch.ones_like(d))), torch.zeros_like(x))
    return c.clamp_(-8, 7).to(torch.int8).flatten(1), s


def _prepare_w4(case, g, s):
    m, n, k = case["m"], case["n"], case["k"]
    w = _randn(g, (n, k), k ** -0.5)
    s["x"] = _randn(g, (m, k))
    s["bias"] = _randn(g, (n,), 0.1) if case["bias"] else None
    s["out"] = torch.zeros((m, n), device="cuda", dtype=torch.float32 if case["epilogue"] == "f32" else torch.float16)
    if own:
        from mimizuku_amd import steps
        s["held"] = torch.zeros((steps.w4_bytes(n, k, case["group"]),), device="cuda", dtype=torch.uint8)
        torch.cuda.synchronize()
        s["weights"] = steps.W4(_context(), n, k, case["group"], at=s["held"].data_ptr())
        s["weights"].pack(w.data_ptr())
        _context().sync()
    else:
        s["codes"], s["scales"] = _coded(w, case["group"])


def _lens(case):
    """First and end of what each row sees; the first row is the longest."""
    n = case["rows"]
    end = [max(1, int(case["len"] * (1.0 - 0.8 * ((5 * i) % 11) / 11.0))) if case["ragged"] else case["len"]
           for i in range(n)]
    first = [min((3 * i) % 40, e - 1) if case["first"] else 0 for i, e in enumerate(end)]
    return first, end


def _prepare_cross(case, g, s):
    n, h, t, kvh, pos = case["rows"], case["heads"], case["tokens"], case["heads"] // case["group"], case["positions"]
    slots, where = n, list(range(n))
    s["slot"] = None
    if case["slots"] == "mixed":  # wherever there was room among a few slots more
        slots = n + 2
        where = torch.randperm(slots, generator=torch.Generator().manual_seed(7))[:n].tolist()
        s["slot"] = _ints(where)
    s["slots"] = slots
    if case["layout"] == "tiles":  # a tile per head, padded, keys and values of a slot beside each other
        pad = -(-pos // 64) * 64
        s["kv"] = _randn(g, (slots, 2, kvh, pad, HD))
        s["kv"][:, 1, :, pos:] = 0
        s["k"], s["v"] = (s["kv"][:, i].transpose(1, 2)[:, :pos] for i in (0, 1))
    else:  # a projection's rows: every head's keys, then every head's values
        s["kv"] = _randn(g, (slots, pos, 2, kvh, HD))
        s["k"], s["v"] = (s["kv"][:, :, i] for i in (0, 1))
    s["q"] = _randn(g, (n, t, h, HD), 1.5)
    first, end = _lens(case)
    s["first"], s["len"] = (_ints(first) if case["first"] else None), _ints(end)
    s["out"] = {"out": torch.zeros((n, t, h, HD), device="cuda", dtype=torch.float16),
                "lse": torch.zeros((n, t, h), device="cuda")}
    if case["align"]:
        heads = [-1] * h
        for i in range(case["align"]):
            heads[(7 * i) % h] = i  # 7 and the counts of heads have no common factor
        s["head_slot"] = _ints(heads)
        s["out"]["align"] = torch.zeros((n, t, case["align"], pos), device="cuda")


# what requests ask for, one after the other, where a case says "mixed"
MIXED = {"temperature": (0.0, 0.2, 0.4, 0.6, 0.8, 1.0, 1.3), "top_k": (0, 1, 40, 0, 400), "top_p": (1.0, 0.9, 0.5),
         "min_p": (0.0, 0.0, 0.05, 0.0)}


def _prepare_sample(case, g, s):
    n, v = case["rows"], case["vocab"]
    dtype = torch.float32 if case["dtype"] == "f32" else torch.float16
    s["logits"] = torch.empty((n, v), device="cuda", dtype=dtype)
    for i in range(0, n, 256):  # a bulk of improbable tokens and a few that the audio speaks for
        r = min(256, n - i)
        x = torch.randn((r, v), generator=g, device="cuda").mul_(2.5)
        likely = torch.randint(0, v, (r, 12), generator=g, device="cuda")
        x.scatter_add_(1, likely, torch.rand((r, 12), generator=g, device="cuda") * 16.0)
        s["logits"][i:i + r] = x.to(dtype)
    s["mask"] = (torch.rand((v,), generator=g, device="cuda") < 0.002).to(torch.uint8) if case["mask"] else None
    s["u"] = torch.rand((n,), generator=g, device="cuda").clamp_(min=2.0 ** -24)
    for name, values in MIXED.items():
        x = [values[i % len(values)] if case[name] == "mixed" else case[name] for i in range(n)]
        s[name] = _ints(x) if name == "top_k" else _floats(x)
    s["out"] = {"tokens": torch.zeros((n,), device="cuda", dtype=torch.int32), "logp": torch.zeros((n,), device="cuda"),
                "kept": torch.zeros((n,), device="cuda", dtype=torch.int32)}


def prepare(case, seed):
    g, s = _gen(seed), {"case": case}
    {"w4": _prepare_w4, "cross": _prepare_cross, "sample": _prepare_sample}[case["kind"]](case, g, s)
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
    """The call of a pass with its arguments filled in, as a program does once for the buffers it keeps."""
    from mimizuku_amd import _lib as L
    from mimizuku_amd import steps
    ctx, case, lib = _context(), s["case"], L.lib()
    if case["kind"] == "w4":
        epi = {"f16": L.EPI_F16, "gelu": L.EPI_GELU_F16, "f32": L.EPI_F32}[case["epilogue"]]
        a = L.W4LinearArgs(epilogue=epi, x=_at(s["x"]), ldx=case["k"], m=case["m"], bias=_at(s["bias"]), out=_at(s["out"]),
                           ldo=case["n"])
        return lib.mz_w4_linear, ctx.h, s["weights"].w, a
    if case["kind"] == "sample":
        v, n = case["vocab"], case["rows"]
        a = L.SampleArgs(dtype=L.DT_F32 if case["dtype"] == "f32" else L.DT_F16, rows=n, vocab=v, logits=_at(s["logits"]),
                         ld=v, mask=_at(s["mask"]), temperatures=_at(s["temperature"]), top_ks=_at(s["top_k"]),
                         top_ps=_at(s["top_p"]), min_ps=_at(s["min_p"]), u=_at(s["u"]), tokens=_at(s["out"]["tokens"]),
                         logp=_at(s["out"]["logp"]), kept=_at(s["out"]["kept"]), stride=1)
        a.work, a.work_bytes = _scratch(ctx, steps.sample_bytes(ctx, a))
        return lib.mz_sample, ctx.h, a
    n, h, t, grp = case["rows"], case["heads"], case["tokens"], case["group"]
    (ks, kp, kh, _), (vs, vp, vh, _) = s["k"].stride(), s["v"].stride()
    a = L.CrossArgs(q=_at(s["q"]), out=_at(s["out"]["out"]), q_row=t * h * HD, q_token=h * HD, q_head=HD,
                    out_row=t * h * HD, out_token=h * HD, out_head=HD, k=_at(s["k"]), v=_at(s["v"]), k_slot=ks, k_pos=kp,
                    k_head=kh, v_slot=vs, v_pos=vp, v_head=vh, rows=n, tokens=t, heads=h, kv_heads=h // grp,
                    slots=s["slots"], positions=case["positions"], scale=0.125, slot=_at(s["slot"]),
                    first=_at(s["first"]), len=_at(s["len"]), lse=_at(s["out"]["lse"]), head_slot=_at(s.get("head_slot")),
                    align=_at(s["out"].get("align")), align_heads=case["align"],
                    align_cols=case["positions"] if case["align"] else 0)
    a.work, a.work_bytes = _scratch(ctx, steps.cross_bytes(ctx, a))
    return lib.mz_cross_attention, ctx.h, a


def _run_own(s):
    from mimizuku_amd._lib import check
    if "call" not in s:
        s["call"] = _calls(s)
    fn, *args = s["call"]
    check(fn(*args))
    return s["out"]


# ---------------------------------------------------------------- the plain form


def _w4(s):
    case = s["case"]
    w = s["codes"].float().unflatten(1, (-1, case["group"])) * s["scales"].float()[..., None]
    y = s["x"].float() @ w.flatten(1).T
    if case["bias"]:
        y = y + s["bias"].float()
    if case["epilogue"] == "gelu":
        y = 0.5 * y * torch.erfc(-y * 0.5 ** 0.5)
    return y.to(s["out"].dtype)


def _cross(s):
    case = s["case"]
    n, h, t, grp, pos = case["rows"], case["heads"], case["tokens"], case["group"], case["positions"]
    k, v = s["k"], s["v"]
    if s["slot"] is not None:
        k, v = k[s["slot"].long()], v[s["slot"].long()]
    k, v = (x.float().transpose(1, 2).contiguous() for x in (k, v))  # [rows, cache heads, positions, 64]
    # the query heads of a group beside each other
    q = s["q"].float().permute(0, 2, 1, 3).reshape(n, h // grp, grp * t, HD)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(n, h, t, pos) * 0.125
    j = torch.arange(pos, device="cuda")
    seen = j[None] < s["len"][:, None]
    if s["first"] is not None:
        seen = seen & (j[None] >= s["first"][:, None])
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    z = e.sum(-1, keepdim=True)
    p = e / z
    o = torch.matmul(p.view(n, h // grp, grp * t, pos), v).view(n, h, t, HD).transpose(1, 2)
    out = {"out": o.half().contiguous(), "lse": (torch.log(z) + top).view(n, h, t).transpose(1, 2).contiguous()}
    if case["align"]:
        of = torch.argsort(torch.where(s["head_slot"] < 0, h, s["head_slot"]))[:case["align"]]
        out["align"] = p[:, of].transpose(1, 2).contiguous()
    return out


def _sample(s):
    # (in 64 bits: which token is drawn hangs on sums of up to 50,000 weights next to a border)
    case = s["case"]
    x = s["logits"].double()
    if s["mask"] is not None:
        x = x.masked_fill(s["mask"].bool()[None], -math.inf)
    y, ids = torch.sort(x, dim=-1, descending=True, stable=True)
    t = s["temperature"].double()[:, None]
    w = torch.exp((y - y[:, :1]) / torch.where(t > 0, t, torch.ones_like(t)))
    i = torch.arange(case["vocab"], device="cuda")[None]
    k = torch.where(s["top_k"] > 0, s["top_k"], case["vocab"])[:, None]
    k = torch.where(t > 0, k, torch.ones_like(k))
    among = (i < k) & torch.isfinite(y)
    w = torch.where(among, w, torch.zeros_like(w))
    before = torch.cumsum(w, -1) - w
    p = s["top_p"].double()[:, None]
    keep = among & ((before < p * w.sum(-1, keepdim=True)) | (p >= 1)) & (w >= s["min_p"].double()[:, None])
    keep[:, 0] = True
    w = torch.where(keep, w, torch.zeros_like(w))
    by_id = torch.zeros_like(w).scatter_(1, ids, w)
    run = torch.cumsum(by_id, -1)
    tok = ((run <= s["u"].double()[:, None] * run[:, -1:]).sum(-1)).clamp(max=case["vocab"] - 1)
    lp = torch.log(by_id.gather(1, tok[:, None])[:, 0]) - torch.log(run[:, -1])
    return {"tokens": tok.int(), "logp": lp.float(), "kept": keep.sum(-1).int()}


def run(s):
    if own:
        return _run_own(s)
    return {"w4": _w4, "cross": _cross, "sample": _sample}[s["case"]["kind"]](s)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["kind"] == "w4":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * k / 2 + 2 * n * k / case["group"] + 2 * m * k + (2 * n if case["bias"] else 0) +
                m * n * (4 if case["epilogue"] == "f32" else 2), "flops": 2.0 * m * n * k}
    if case["kind"] == "sample":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * v * (4 if case["dtype"] == "f32" else 2) + (v if case["mask"] else 0) + 32 * n,
                "flops": 4.0 * n * v}
    n, h, t = case["rows"], case["heads"], case["tokens"]
    seen = sum(e - f for f, e in zip(*_lens(case)))
    return {"bytes": 4.0 * HD * seen * (h // case["group"]) + n * t * h * (4 * HD + 4) +
            4.0 * n * t * case["align"] * case["positions"], "flops": 4.0 * HD * seen * h * t}


# ---------------------------------------------------------------- the same in 64 bits, from the definitions


def _exact_w4(case, seed):
    m, n, k, grp = case["m"], case["n"], case["k"], case["group"]
    g = _gen(seed)
    w = _randn(g, (n, k), k ** -0.5)  # the draws of prepare, in its order
    x = _randn(g, (m, k)).double()
    bias = _randn(g, (n,), 0.1).double() if case["bias"] else torch.zeros((n,), device="cuda", dtype=torch.float64)
    out = torch.empty((m, n), device="cuda", dtype=torch.float64)
    for i in range(0, n, 2048):
        a = w[i:i + 2048].double().reshape(-1, k // grp, grp)
        at = a.abs().argmax(-1, keepdim=True)
        far = a.gather(2, at)
        far = torch.where(a.amin(-1, keepdim=True) == -far, -far.abs(), far)  # of two alike in size the negative one
        scale = (far / -8.0).half().double()
        q = a / torch.where(scale == 0, 1.0, scale)
        whole = torch.floor(q)
        up = (q - whole > 0.5) | ((q - whole == 0.5) & (whole % 2 != 0))
        c = torch.where(scale == 0, 0.0, torch.clamp(whole + up, -8.0, 7.0))
        out[:, i:i + 2048] = x @ (c * scale).reshape(-1, k).T.contiguous() + bias[i:i + 2048]
    if case["epilogue"] == "gelu":
        out = out * torch.special.ndtr(out)
    return out


def _exact_cross(case, seed):
    s = prepare(case, seed)
    n, h, t, grp, pos = case["rows"], case["heads"], case["tokens"], case["group"], case["positions"]
    o = torch.zeros((n, t, h, HD), device="cuda", dtype=torch.float64)
    lse = torch.zeros((n, t, h), device="cuda", dtype=torch.float64)
    align = torch.zeros((n, t, case["align"], pos), device="cuda", dtype=torch.float64)
    index = s["head_slot"].tolist() if case["align"] else [-1] * h
    for r, (f, e) in enumerate(zip(*_lens(case))):
        at = r if s["slot"] is None else int(s["slot"][r])
        for a in range(h):
            k, v = s["k"][at, f:e, a // grp].double(), s["v"][at, f:e, a // grp].double()
            x = (s["q"][r, :, a].double() * 0.125) @ k.T.contiguous()
            lse[r, :, a] = torch.logsumexp(x, -1)
            y = torch.softmax(x, -1)
            o[r, :, a] = y @ v.contiguous()
            if index[a] >= 0:
                align[r, :, index[a], f:e] = y
    return {"out": o, "lse": lse, **({"align": align} if case["align"] else {})}


def _exact_sample(case, seed):
    s = prepare(case, seed)
    off = s["mask"].bool().cpu() if case["mask"] else torch.zeros((case["vocab"],), dtype=torch.bool)
    tokens, logp, kept = [], [], []
    rows = zip(s["logits"].cpu(), s["u"].tolist(), s["temperature"].tolist(), s["top_k"].tolist(), s["top_p"].tolist(),
               s["min_p"].tolist())
    for x, u, t, k, p, low in rows:
        ids = torch.nonzero(~off)[:, 0]
        x = x[ids].double()
        if t == 0:
            tokens.append(int(ids[int((x == x.max()).nonzero()[0, 0])]))
            logp.append(0.0)
            kept.append(1)
            continue
        if 0 < k < len(x):  # above the k-th largest, and of those equal to it the first ones
            edge = torch.kthvalue(x, len(x) - k + 1).values
            above, equal = x > edge, torch.nonzero(x == edge)[:, 0]
            above[equal[:k - int(above.sum())]] = True
            ids, x = ids[above], x[above]
        share = torch.softmax(x / t, 0)
        if p < 1:
            order = torch.argsort(-x, stable=True)
            need = int(torch.searchsorted(torch.cumsum(share[order], 0), p)) + 1
            order = torch.sort(order[:need]).values
            ids, x = ids[order], x[order]
        stay = torch.exp((x - x.max()) / t) >= low
        ids, x = ids[stay], x[stay]
        share = torch.softmax(x / t, 0)
        run = torch.cumsum(share, 0)
        i = min(int(torch.searchsorted(run, u * float(run[-1]), right=True)), len(x) - 1)
        tokens.append(int(ids[i]))
        logp.append(float(torch.log_softmax(x / t, 0)[i]))
        kept.append(len(x))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32, device="cuda"),
            "logp": torch.tensor(logp, dtype=torch.float64, device="cuda"),
            "kept": torch.tensor(kept, dtype=torch.int32, device="cuda")}


def exact(case, seed):
    return {"w4": _exact_w4, "cross": _exact_cross, "sample": _exact_sample}[case["kind"]](case, seed)
