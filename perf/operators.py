"""Timed cases of the operators between a token's projections.

* ``norm``    the residual's addition, the root-mean-square norm and the power-of-two int8 quantizer whose
              QuantAct the projections take;
* ``append``  rotary positions of q and k, and k and v into the paged 4-bit cache (read back as the values
              that the codes stand for);
* ``attn``    attention over that cache: single tokens and chunks of tokens, causal, with an optional window
              and first tokens that stay visible;
* ``sample``  temperature, top-k, top-p and min-p over the head's logits, from given random numbers.

The plain forms are elementary torch operations in 32 bits; ``own`` calls the framework's entry points.
A cache block is 32 channels: d is the f16 number of 8 significant bits nearest to -m / 8 (m the element of
largest magnitude, the positive one of two), an element's code is 8 more than the whole number nearest to its f32 quotient by d (at least 0, at most
15), and the value of code c is (c - 8) d.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
BASE = 1e6
SCALING = ("none", "linear", "ntk", "bands")
LOW, HIGH, ORIGINAL = 1.0, 32.0, 32768  # bands: turns over the original context


def listed():
    return [
        # one decode token of the 0.5B-class width, and a prefill of the 1.5B-class width
        {"name": "norm 1x896", "op": "norm", "n_tok": 1, "n": 896, "residual": True},
        {"name": "norm 512x1536", "op": "norm", "n_tok": 512, "n": 1536, "residual": True},
        # an odd width near the FFN's, with a last block in part
        {"name": "norm 2039x8957", "op": "norm", "n_tok": 2039, "n": 8957, "residual": True},
        # a decode batch of 8 tokens, each of its own sequence; 12 query and 2 KV heads of 128
        {"name": "append 8 tokens", "op": "append", "n_tok": 8, "seqs": 8, "heads": 12, "kv": 2, "dim": 128, "rot": 128,
         "layout": "half", "scaling": "none", "page": 64, "ctx": 4096},
        # a prefill chunk with half of the head rotated, interleaved, for a context stretched eightfold
        {"name": "append 4093 tokens", "op": "append", "n_tok": 4093, "seqs": 1, "heads": 12, "kv": 2, "dim": 128, "rot": 64,
         "layout": "interleaved", "scaling": "bands", "page": 128, "ctx": 40000},
        # one sequence at a long prompt's end: the call whose latency a chat user feels
        {"name": "attn decode 1x4001", "op": "attn", "seqs": 1, "q": 1, "ctx": 4001, "ragged": False, "heads": 12, "kv": 2, "dim": 128,
         "page": 64, "window": 0, "sinks": 0},
        # a serving batch of uneven contexts
        {"name": "attn decode 64x16384", "op": "attn", "seqs": 64, "q": 1, "ctx": 16384, "ragged": True, "heads": 12, "kv": 2, "dim": 128,
         "page": 64, "window": 0, "sinks": 0},
        # heads of 64, a window with four first tokens, contexts far longer than the window
        {"name": "attn window 16x32768", "op": "attn", "seqs": 16, "q": 1, "ctx": 32768, "ragged": True, "heads": 14, "kv": 2, "dim": 64,
         "page": 32, "window": 4096, "sinks": 4},
        # uneven chunks of prompts over cached prefixes
        {"name": "attn chunks 5x301", "op": "attn", "seqs": 5, "q": 301, "ctx": 6007, "ragged": True, "heads": 14, "kv": 2, "dim": 64,
         "page": 64, "window": 0, "sinks": 0},
        # a whole long prompt
        {"name": "attn prefill 8192", "op": "attn", "seqs": 1, "q": 8192, "ctx": 8192, "ragged": False, "heads": 12, "kv": 2, "dim": 128,
         "page": 64, "window": 0, "sinks": 0},
        # one chat user's token, and a serving batch whose requests differ in their parameters
        {"name": "sample 1x151936", "op": "sample", "rows": 1, "vocab": 151936, "mixed": False},
        {"name": "sample 192x151936", "op": "sample", "rows": 192, "vocab": 151936, "mixed": True},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "append", "attn", "attn", "attn", "sample"])
    if op == "norm":
        return {"op": op, "n_tok": _spread(rng, 1, 2039), "n": _spread(rng, 64, 8957), "residual": rng.random() < 0.75}
    kv, dim, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256]), rng.choice([32, 64, 128])
    heads = kv * rng.randint(1, 8)
    if op == "append":
        n_tok = _spread(rng, 1, 4093 * 16 // max(16, heads + 2 * kv))
        return {"op": op, "n_tok": n_tok, "seqs": rng.choice([1, n_tok]), "heads": heads, "kv": kv, "dim": dim,
                "rot": rng.choice([dim, dim // 2, dim // 4]), "layout": rng.choice(["half", "interleaved"]), "scaling": rng.choice(SCALING),
                "page": page, "ctx": n_tok + _spread(rng, 1, 32768)}
    if op == "sample":
        return {"op": op, "rows": _spread(rng, 1, 128), "vocab": _spread(rng, 1000, 151936), "mixed": rng.random() < 0.75}
    window = rng.choice([0, 0, _spread(rng, 16, 8192)])
    case = {"op": op, "heads": heads, "kv": kv, "dim": dim, "page": page, "window": window, "sinks": rng.choice([0, 1, 4, 37]) if window else 0}
    if rng.random() < 0.5:  # single tokens, or a few of each sequence
        case |= {"q": rng.choice([1, 1, 2, 5]), "ragged": rng.random() < 0.7, "ctx": _spread(rng, 8, 32768)}
        case["seqs"] = _spread(rng, 1, max(1, min(64, (1 << 27) // (case["ctx"] * kv * dim))))
    else:
        q = _spread(rng, 17, 2048)
        case |= {"q": q, "ragged": rng.random() < 0.5, "ctx": q + rng.choice([0, _spread(rng, 1, 4096)])}
        case["seqs"] = max(1, min(5, (1 << 27) // (heads * q * case["ctx"])))
    return case


# ---- inputs --------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _ints(g, low, high, *shape):
    return torch.randint(low, high, shape, generator=g, device="cuda", dtype=torch.int32)


def _heads(g, n, heads, dim, spread=1.0):
    """f32 head rows as a projection leaves them: a few channels of each head stand out."""
    x = torch.randn(n, heads, dim, generator=g, device="cuda") * spread
    x *= torch.exp(0.5 * torch.randn(heads, dim, generator=g, device="cuda"))
    return x


def _lengths(case, g):
    """Queries and context of every sequence."""
    n, q, ctx = case["seqs"], case["q"], case["ctx"]
    if not case["ragged"]:
        return torch.full((n,), q, dtype=torch.int32, device="cuda"), torch.full((n,), ctx, dtype=torch.int32, device="cuda")
    qs = torch.tensor([q - i * q // (2 * n) for i in range(n)], dtype=torch.int32, device="cuda")  # from all to half of q
    ctxs = qs + (_ints(g, 0, max(1, ctx - q + 1), n) if ctx > q else 0)
    ctxs[0] = ctx
    return qs, ctxs


def _raw(case, seed):
    """The inputs alone, the same for the plain form, the framework and the exact values."""
    g, op = _gen(seed), case["op"]
    if op == "norm":
        t, n = case["n_tok"], case["n"]
        x = torch.randn(t, n, generator=g, device="cuda")
        r = torch.randn(t, n, generator=g, device="cuda") * 3 if case["residual"] else None
        if r is not None:
            r[:, :: max(1, n // 5)] *= 20  # the few large channels of a residual stream
        return {"x": x, "r": r, "g": 1 + 0.2 * torch.randn(n, generator=g, device="cuda")}
    if op == "append":
        t, seqs, page = case["n_tok"], case["seqs"], case["page"]
        per = -(-case["ctx"] // page)
        if seqs == 1:
            seq = torch.zeros(t, dtype=torch.int32, device="cuda")
            pos = torch.arange(case["ctx"] - t, case["ctx"], dtype=torch.int32, device="cuda")
        else:
            seq = torch.arange(t, dtype=torch.int32, device="cuda")
            pos = _ints(g, 0, case["ctx"], t)
        # only the pages that the tokens fall in are the sequence's own; a long context's others share one page
        used = torch.zeros(seqs, per, dtype=torch.bool, device="cuda")
        used[seq.long(), (pos // page).long()] = True
        table = torch.zeros(seqs, per, dtype=torch.int32, device="cuda")
        n = int(used.sum())
        table[used] = 1 + torch.randperm(n, generator=g, device="cuda").int()
        return {"q": _heads(g, t, case["heads"], case["dim"]), "k": _heads(g, t, case["kv"], case["dim"], 2.0),
                "v": _heads(g, t, case["kv"], case["dim"]), "seq": seq, "pos": pos, "table": table, "pages": n + 1}
    if op == "attn":
        qs, ctxs = _lengths(case, g)
        page = case["page"]
        need = (ctxs + page - 1) // page
        per = int(need.max())
        live = torch.arange(per, device="cuda")[None] < need[:, None]
        n = int(need.sum())
        table = torch.zeros(case["seqs"], per, dtype=torch.int32, device="cuda")
        table[live] = torch.randperm(n, generator=g, device="cuda").int()
        start = torch.zeros(case["seqs"] + 1, dtype=torch.int32, device="cuda")
        start[1:] = torch.cumsum(qs, 0)
        q = _heads(g, int(start[-1]), case["heads"], case["dim"])
        k = torch.randn(n * page, case["kv"], case["dim"], generator=g, device="cuda")
        k *= torch.exp(0.5 * torch.randn(case["kv"], case["dim"], generator=g, device="cuda"))
        v = torch.randn(n * page, case["kv"], case["dim"], generator=g, device="cuda")
        return {"qs": qs, "ctx": ctxs, "start": start, "table": table, "pages": n, "q": q, "k": k, "v": v}
    n, V = case["rows"], case["vocab"]
    x = torch.randn(n, V, generator=g, device="cuda") * 2.5
    x += 4 * torch.randn(n, V, generator=g, device="cuda").clamp_(min=3).sub_(3)  # a few likely tokens
    s = {"x": x, "u": torch.rand(n, generator=g, device="cuda")}
    ones = torch.ones(n, device="cuda")
    s |= {"t": 0.7 * ones, "k": (40 * ones).int(), "p": 0.95 * ones, "m": 0.0 * ones}
    if case["mixed"]:
        def pick(values):
            return torch.tensor(values, device="cuda")[_ints(g, 0, len(values), n).long()]
        s |= {"t": pick([0.0, 0.3, 0.7, 1.0, 1.3]), "k": pick([0, 1, 20, 50, 1000]).int(), "p": pick([1.0, 0.95, 0.9, 0.5]),
              "m": pick([0.0, 0.0, 0.02, 0.1])}
        x[_ints(g, 0, 4, n) == 0, : V // 3] = -math.inf  # a grammar's mask
    return s


def _frequencies(case):
    """Radians a position of each rotated pair, and the amplitude (f64)."""
    rot, kind, f = case["rot"], case["scaling"], 8.0
    base = BASE * f ** (rot / (rot - 2)) if kind == "ntk" else BASE
    theta = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if kind == "linear":
        return [t / f for t in theta], 1.0
    if kind == "bands":
        keep = [min(1.0, max(0.0, (ORIGINAL * t / (2 * math.pi) - LOW) / (HIGH - LOW))) for t in theta]
        return [t * ((1 - k) / f + k) for t, k in zip(theta, keep)], 0.1 * math.log(f) + 1
    return theta, 1.0


# ---- the plain forms -----------------------------------------------------------------------------


def _codes(x):
    """4-bit codes (as bytes) and f16 scales of 32-channel blocks of the last axis."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    high, low = b.amax(-1, keepdim=True), b.amin(-1, keepdim=True)
    d = _eight_bits(-torch.where(high >= -low, high, low) / 8)
    c = torch.where(d != 0, torch.round(b / torch.where(d != 0, d, 1.0)), 0.0).clamp(-8, 7) + 8
    return c.to(torch.uint8).reshape(x.shape), d[..., 0].half()


def _power(e):
    """2^e in f32 for whole e (its bits: a library's pow may be a last bit off)."""
    return ((e + 127) << 23).view(torch.float32)


def _eight_bits(d):
    """The nearest f16 of 8 significant bits (ties to even), as f32."""
    step = _power(torch.clamp(torch.frexp(d)[1] - 8, min=-24))
    return (torch.round(d / step) * step).clamp(-8160.0, 8160.0)


def _values(c, d):
    return ((c.float() - 8).reshape(*c.shape[:-1], -1, 32) * d.float()[..., None]).reshape(c.shape)


def _rotate(x, cos, sin, layout):
    rot = 2 * cos.shape[-1]
    y = x.clone()
    if layout == "half":
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        y[..., : rot // 2], y[..., rot // 2: rot] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    return y


def _plain_norm(s):
    v = s["x"] if s["r"] is None else s["x"] + s["r"]
    y = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * s["g"]
    t, n = y.shape
    b = torch.nn.functional.pad(y, (0, -n % 32)).reshape(t, -1, 32)
    m, e = torch.frexp(b.abs().amax(-1, keepdim=True))
    S = _power(torch.clamp(e - 7 + (m > 127 / 128).int(), min=-32))
    c = torch.sign(b) * torch.floor(b.abs() / S + 0.5)
    return [v, (c * S).reshape(t, -1)[:, :n].to(torch.bfloat16)]


def _plain_append(s):
    angle = s["pos"].double()[:, None] * s["theta"]
    cos, sin = (s["amplitude"] * angle.cos()).float()[:, None], (s["amplitude"] * angle.sin()).float()[:, None]
    q, k = _rotate(s["q"], cos, sin, s["case"]["layout"]), _rotate(s["k"], cos, sin, s["case"]["layout"])
    out, page = [q], s["case"]["page"]
    at = s["table"][s["seq"].long(), (s["pos"] // page).long()].long(), (s["pos"] % page).long()
    for x, c, d in ((k, s["kc"], s["kd"]), (s["v"], s["vc"], s["vd"])):
        c[at], d[at] = _codes(x)
        out.append(_values(c[at], d[at]).half())
    return out


def _visible(pos, key, window, sinks):
    see = key <= pos
    return see & ((key > pos - window) | (key < sinks)) if window else see


def _plain_attn(s):
    case, kv, dim = s["case"], s["case"]["kv"], s["case"]["dim"]
    G, S, Q = case["heads"] // kv, case["seqs"], int(case["q"])
    K, V = (_values(c[s["table"].long()], d[s["table"].long()]).reshape(S, -1, kv, dim).permute(0, 2, 1, 3).contiguous()
            for c, d in ((s["kc"], s["kd"]), (s["vc"], s["vd"])))
    q = torch.zeros(S, Q, kv, G, dim, device="cuda")
    q[s["tok_seq"], s["tok_i"]] = s["q"].reshape(-1, kv, G, dim)
    q = q.permute(0, 2, 1, 3, 4).reshape(S, kv, Q * G, dim)
    w = torch.matmul(q * dim ** -0.5, K.transpose(2, 3).contiguous())  # [S, kv, Q * G, L]
    pos = (s["ctx"] - s["qs"])[:, None] + torch.arange(Q, device="cuda")
    see = _visible(pos[..., None], torch.arange(w.shape[-1], device="cuda"), case["window"], case["sinks"])
    w = w.reshape(S, kv, Q, G, -1).masked_fill_(~see[:, None, :, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w = w.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    o = torch.matmul(w.reshape(S, kv, Q * G, -1), V) / w.sum(-1).reshape(S, kv, Q * G, 1)
    o = torch.nan_to_num(o).reshape(S, kv, Q, G, dim).permute(0, 2, 1, 3, 4)
    return [o[s["tok_seq"], s["tok_i"]].reshape(-1, kv * G, dim)]


def _plain_sample(s):
    x = s["x"]
    n, V = x.shape
    l, order = torch.sort(x, dim=-1, descending=True, stable=True)
    greedy = (s["t"] == 0)[:, None]
    z = (l - l[:, :1]) * (1.0 / torch.where(greedy, 1.0, s["t"][:, None]))
    w = torch.round(torch.exp(z) * 4294967296.0).long()
    rank = torch.arange(V, device="cuda")
    k = torch.where(greedy[:, 0], 1, torch.where(s["k"] <= 0, V, s["k"]))[:, None]
    w *= rank < k
    before = torch.cumsum(w, -1) - w
    total = before[:, -1:] + w[:, -1:]
    w *= (before.double() < s["p"].double()[:, None] * total.double()) | (s["p"] >= 1)[:, None]
    w *= w.double() >= s["m"].double()[:, None] * 4294967296.0
    kept = torch.zeros_like(w).scatter_(1, order, w)  # in the order of the vocabulary
    run_ = torch.cumsum(kept, -1)
    at = torch.floor(s["u"].double()[:, None] * run_[:, -1:].double()).long()
    token = (run_ <= at).sum(-1)
    return [token.int(), (kept.gather(1, token[:, None])[:, 0].double() / run_[:, -1].double()).float()]


# ---- the passes ----------------------------------------------------------------------------------


def _empty(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


def _tokens(seq, pos, table):
    return {"seq_ptr": seq.data_ptr(), "pos_ptr": pos.data_ptr(), "n_tok": seq.numel(), "table_ptr": table.data_ptr(),
            "n_seq": table.shape[0], "table_stride": table.shape[1]}


def _fill(s, cache):
    """Puts k and v of every slot of the cache's pages into it."""
    n, page = s["pages"], s["case"]["page"]
    slot = torch.arange(n * page, dtype=torch.int32, device="cuda")
    table = torch.arange(n, dtype=torch.int32, device="cuda")[None].contiguous()
    cache.append_dev(None, k_ptr=s["k"].data_ptr(), v_ptr=s["v"].data_ptr(), stream=_stream(), **_tokens(torch.zeros_like(slot), slot, table))
    torch.cuda.synchronize()


def prepare(case, seed):
    s = _raw(case, seed) | {"case": case}
    op = case["op"]
    if own:
        from apeiron_amd import chart

        dev = s["dev"] = chart.device()
        if op == "norm":
            s["out"] = [_empty(*s["x"].shape), _empty(*s["x"].shape, dtype=torch.bfloat16)]
            s["act"] = _empty(*s["x"].shape, dtype=torch.int8), _empty(s["x"].shape[0], -(-case["n"] // 32), dtype=torch.int64)
        elif op == "append":
            scaling = {"none": None, "linear": ("linear", 8.0), "ntk": ("ntk", 8.0), "bands": ("bands", 8.0, LOW, HIGH, ORIGINAL)}[case["scaling"]]
            s["rope"] = chart.Rope(dev, case["dim"], case["rot"], layout=case["layout"], base=BASE, scaling=scaling)
            s["cache"] = chart.KvCache4(dev, s["pages"], case["page"], case["kv"], case["dim"])
            s["out"] = [torch.zeros_like(s["q"]), torch.zeros_like(s["k"], dtype=torch.float16), torch.zeros_like(s["v"], dtype=torch.float16)]
        elif op == "attn":
            s["cache"] = chart.KvCache4(dev, s["pages"], case["page"], case["kv"], case["dim"])
            _fill(s, s["cache"])
            s["out"] = [torch.zeros_like(s["q"])]
        else:
            s["out"] = [_empty(case["rows"], dtype=torch.int32), _empty(case["rows"])]
    elif op == "append":
        theta, s["amplitude"] = _frequencies(case)
        s["theta"] = torch.tensor(theta, dtype=torch.float64, device="cuda")
        n, page, kv, dim = s["pages"], case["page"], case["kv"], case["dim"]
        for name in ("k", "v"):
            s[name + "c"], s[name + "d"] = _empty(n, page, kv, dim, dtype=torch.uint8), _empty(n, page, kv, dim // 32, dtype=torch.float16)
    elif op == "attn":
        n, page, kv, dim = s["pages"], case["page"], case["kv"], case["dim"]
        for name in ("k", "v"):
            c, d = _codes(s[name])
            s[name + "c"], s[name + "d"] = c.reshape(n, page, kv, dim), d.reshape(n, page, kv, dim // 32)
        s["tok_seq"] = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), s["qs"].long())
        s["tok_i"] = torch.arange(s["tok_seq"].numel(), device="cuda") - s["start"].long()[s["tok_seq"]]
    if op == "attn":
        del s["k"], s["v"]
    return s


def _stream():
    return torch.cuda.current_stream().cuda_stream


def run(s):
    case, op = s["case"], s["case"]["op"]
    if not own:
        return {"norm": _plain_norm, "append": _plain_append, "attn": _plain_attn, "sample": _plain_sample}[op](s)
    from apeiron_amd import chart

    out, dev, stream = s["out"], s["dev"], _stream()
    if op == "norm":
        chart.norm_quant_dev(dev, s["x"].data_ptr(), s["g"].data_ptr(), EPS, case["n_tok"], case["n"],
                             residual_ptr=None if s["r"] is None else s["r"].data_ptr(), sum_ptr=out[0].data_ptr(),
                             codes_ptr=s["act"][0].data_ptr(), scales_ptr=s["act"][1].data_ptr(), values_ptr=out[1].data_ptr(), stream=stream)
    elif op == "append":
        tokens = _tokens(s["seq"], s["pos"], s["table"])
        s["cache"].append_dev(s["rope"], q_ptr=s["q"].data_ptr(), n_heads=case["heads"], q_out_ptr=out[0].data_ptr(),
                              k_ptr=s["k"].data_ptr(), v_ptr=s["v"].data_ptr(), stream=stream, **tokens)
        s["cache"].read_dev(k_ptr=out[1].data_ptr(), v_ptr=out[2].data_ptr(), stream=stream, **tokens)
    elif op == "attn":
        s["cache"].attn_dev(s["q"].data_ptr(), out[0].data_ptr(), n_heads=case["heads"], n_tok=s["q"].shape[0], n_seq=case["seqs"],
                            q_start_ptr=s["start"].data_ptr(), ctx_ptr=s["ctx"].data_ptr(), table_ptr=s["table"].data_ptr(),
                            table_stride=s["table"].shape[1], max_q=case["q"], max_ctx=case["ctx"], scale=case["dim"] ** -0.5,
                            window=case["window"], sinks=case["sinks"], stream=stream)
    else:
        chart.sample_dev(dev, s["x"].data_ptr(), case["rows"], case["vocab"], s["u"].data_ptr(), out[0].data_ptr(), probs_ptr=out[1].data_ptr(),
                         temperature_ptr=s["t"].data_ptr(), top_k_ptr=s["k"].data_ptr(), top_p_ptr=s["p"].data_ptr(), min_p_ptr=s["m"].data_ptr(),
                         stream=stream)
    return out


def _pairs(q, ctx, window, sinks):
    """Visible (query, key) pairs of one sequence."""
    n = 0
    for pos in (ctx - q, ctx - 1) if q > 64 else range(ctx - q, ctx):
        n += pos + 1 if not window else min(pos + 1, window) + min(max(pos + 1 - window, 0), sinks)
    return n * q // 2 if q > 64 else n


def work(case):
    op = case["op"]
    if op == "norm":
        t, n = case["n_tok"], case["n"]
        return {"bytes": t * n * (4 + 4 * case["residual"] + 4 + 1 + 2) + 8 * t * -(-n // 32) + 4 * n, "flops": 8 * t * n}
    if op == "append":
        q, kv = case["n_tok"] * case["heads"] * case["dim"], 2 * case["n_tok"] * case["kv"] * case["dim"]
        return {"bytes": 8 * q + 4 * kv + kv * 9 // 16 + 2 * kv, "flops": 3 * q + 6 * kv}
    if op == "sample":
        return {"bytes": 4 * case["rows"] * case["vocab"] + 28 * case["rows"], "flops": 4 * case["rows"] * case["vocab"]}
    # uneven lengths: three quarters of the largest chunk and half of the largest prefix, as they are drawn
    S, q, ctx = case["seqs"], case["q"], case["ctx"]
    if case["ragged"]:
        sizes = [(q, ctx)] + [(max(1, q * 3 // 4), max(1, q * 3 // 4) + (ctx - q) // 2)] * (S - 1)
    else:
        sizes = [(q, ctx)] * S
    keys = sum(min(c, case["window"] + n + case["sinks"]) if case["window"] else c for n, c in sizes)
    size = keys * case["kv"] * case["dim"] * 9 // 8 + 8 * sum(n for n, _ in sizes) * case["heads"] * case["dim"]
    return {"bytes": size, "flops": 4 * case["heads"] * case["dim"] * sum(_pairs(n, c, case["window"], case["sinks"]) for n, c in sizes)}


# ---- 64 bits -------------------------------------------------------------------------------------


def _exact_power(e, low):
    return ((torch.clamp(e, min=low).long() + 1023) << 52).view(torch.float64)


def _exact_cache(x):
    """f64 values of the cache for f32 rows, from the format's definition."""
    b = x.double().unflatten(-1, (-1, 32))
    top, bottom = b.max(-1, keepdim=True).values, b.min(-1, keepdim=True).values
    d = torch.where(top + bottom >= 0, top, bottom) / -8
    unit = _exact_power(torch.floor(torch.log2(d.abs().clamp(min=1e-300))) - 7, -24)
    d = (torch.round(d / unit) * unit).clamp(-8160, 8160)
    # the code is the nearest to the quotient's f32 value (this rounding of the f64 quotient gives it exactly)
    q = torch.round((b / torch.where(d == 0, 1.0, d)).float().double()).clamp(-8, 7)
    return (q * d).flatten(-2)


def _exact_attn(case, s):
    kv, dim, page = case["kv"], case["dim"], case["page"]
    G = case["heads"] // kv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i in range(case["seqs"]):
        n, ctx, at = int(s["qs"][i]), int(s["ctx"][i]), int(s["start"][i])
        slots = (s["table"][i, : -(-ctx // page)].long()[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[:ctx]
        key = torch.arange(ctx, device="cuda")
        for h in range(kv):
            K, V = _exact_cache(s["k"][slots, h]), _exact_cache(s["v"][slots, h])
            step = max(1, (1 << 27) // (ctx * G))
            for j in range(0, n, step):
                m = min(step, n - j)
                q = s["q"][at + j: at + j + m, h * G: (h + 1) * G].double()
                w = (q.reshape(m * G, dim) @ K.T).reshape(m, G, ctx) / math.sqrt(dim)
                pos = ctx - n + j + torch.arange(m, device="cuda")[:, None]
                see = key <= pos
                if case["window"]:
                    see = see & ((pos - key < case["window"]) | (key < case["sinks"]))
                w = torch.softmax(torch.where(see[:, None], w, -math.inf), -1)
                out[at + j: at + j + m, h * G: (h + 1) * G] = (w.reshape(m * G, ctx) @ V).reshape(m, G, dim)
    return [out]


def exact(case, seed):
    s, op = _raw(case, seed), case["op"]
    if op == "norm":
        v = s["x"].double()
        if s["r"] is not None:
            v = v + s["r"].double()
        y = v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS) * s["g"].double()
        t, n = y.shape
        b = torch.cat([y, torch.zeros(t, -n % 32, dtype=y.dtype, device="cuda")], 1).reshape(t, -1, 32)
        S = _exact_power(torch.ceil(torch.log2((b.abs().amax(-1, keepdim=True) / 127).clamp(min=1e-300))), -32)
        c = torch.copysign(torch.floor(b.abs() / S + 0.5), b)
        return [v, (c * S).reshape(t, -1)[:, :n]]
    if op == "append":
        theta, amplitude = _frequencies(case)
        z = torch.polar(torch.full((case["n_tok"], len(theta)), amplitude, dtype=torch.float64, device="cuda"),
                        s["pos"].double()[:, None] * torch.tensor(theta, dtype=torch.float64, device="cuda"))[:, None]

        def turned(x):
            x, rot = x.double(), case["rot"]
            if case["layout"] == "half":
                pair = torch.complex(x[..., : rot // 2], x[..., rot // 2: rot]) * z
                head = torch.cat([pair.real, pair.imag], -1)
            else:
                head = torch.view_as_real(torch.view_as_complex(x[..., :rot].reshape(*x.shape[:-1], -1, 2).contiguous()) * z).flatten(-2)
            return torch.cat([head, x[..., rot:]], -1)

        return [turned(s["q"]), _exact_cache(turned(s["k"])), _exact_cache(s["v"])]
    if op == "attn":
        return _exact_attn(case, s)
    token, prob = [], []
    for i in range(case["rows"]):
        x, T, k, p, m = s["x"][i].double(), float(s["t"][i]), int(s["k"][i]), float(s["p"][i]), float(s["m"][i])
        order = torch.sort(x, descending=True, stable=True).indices
        keep = order[: 1 if T == 0 else k if k > 0 else None]
        w = torch.round(torch.exp((x[keep] - x[order[0]]) / (T or 1.0)) * 2.0 ** 32)
        before = torch.cumsum(w, 0) - w
        w = w * ((before < p * w.sum()) | torch.tensor(p >= 1, device="cuda")) * (w >= m * 2.0 ** 32)
        run_ = torch.zeros_like(x).index_put_((keep,), w)
        total = torch.cumsum(run_, 0)
        token.append((total <= torch.floor(float(s["u"][i]) * total[-1])).sum().int())
        prob.append(run_[token[-1]] / total[-1])
    return [torch.stack(token), torch.stack(prob)]
