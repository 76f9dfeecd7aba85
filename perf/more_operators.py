"""Timed cases of the operators whose cost does not follow the whole context.

* ``conv``    the short causal convolution of a recurrent layer's channels over a sequence, with the inputs before
              the call from the sequence's state, and SiLU;
* ``delta``   the gated delta rule over a sequence, from and to the sequence's state: with every head's S (keys by
              values), decay g = -exp(A) softplus(a + dt), rate b = sigmoid(.) and q and k of length one,
              S = e^g S, then S += k (b (v - S^T k))^T, and o = scale S^T q;
* ``shared``  attention over the paged 4-bit cache for sequences that begin with the same positions;
* ``blocks``  attention over that cache's blocks of positions: the means of the blocks' keys (those that the call's
              tokens complete first), the blocks whose means a query's heads of a KV head score highest together,
              the first ones, the last ones and the query's own.

The plain forms are elementary torch operations in 32 bits (block scores and the decays' sums in 64); ``own`` calls
the framework's entry points.  The cache's format: 32-channel blocks, d the f16 number of 8 significant bits nearest
to -m / 8 (m the element of largest magnitude, the positive one of two), an element's code 8 more than the whole
number nearest to its f32 quotient by d (at least 0, at most 15), and the value of code c (c - 8) d.
"""
from __future__ import annotations

import math

import torch

own = False

NORM_EPS = 1e-6


def listed():
    return [
        # a decode batch's recurrent layer: 16 heads of 128 for q, k and v
        {"name": "conv 64 tokens", "op": "conv", "seqs": 64, "q": 1, "ragged": False, "channels": 6144, "width": 4},
        # uneven prompts, an odd number of channels
        {"name": "conv 5 x 1021", "op": "conv", "seqs": 5, "q": 1021, "ragged": True, "channels": 4099, "width": 4},
        # one chat user's token, and a decode batch
        {"name": "delta 1 token", "op": "delta", "seqs": 1, "q": 1, "ragged": False, "kheads": 16, "heads": 16, "kdim": 128, "vdim": 128},
        {"name": "delta 64 tokens", "op": "delta", "seqs": 64, "q": 1, "ragged": False, "kheads": 16, "heads": 16, "kdim": 128, "vdim": 128},
        # uneven chunks of prompts, value heads that share key heads
        {"name": "delta 5 x 301", "op": "delta", "seqs": 5, "q": 301, "ragged": True, "kheads": 8, "heads": 16, "kdim": 128, "vdim": 128},
        # a whole long prompt
        {"name": "delta 8192", "op": "delta", "seqs": 1, "q": 8192, "ragged": False, "kheads": 16, "heads": 16, "kdim": 128, "vdim": 128},
        # eight samples of one prompt
        {"name": "shared 8 x 2048", "op": "shared", "seqs": 8, "q": 1, "prefix": 2048, "ctx": 2176, "ragged": False, "heads": 14, "kv": 2,
         "dim": 64, "page": 64},
        # a serving batch behind one long document
        {"name": "shared 64 x 16384", "op": "shared", "seqs": 64, "q": 1, "prefix": 16384, "ctx": 17408, "ragged": True, "heads": 12, "kv": 2,
         "dim": 128, "page": 64},
        # questions of up to 49 tokens over a document that ends inside a page
        {"name": "shared 16 x 49 of 8003", "op": "shared", "seqs": 16, "q": 49, "prefix": 8003, "ctx": 8052, "ragged": True, "heads": 12, "kv": 2,
         "dim": 128, "page": 64},
        # one user's token at the end of a long context, and a serving batch of uneven ones
        {"name": "blocks 1 x 32768", "op": "blocks", "seqs": 1, "q": 1, "ctx": 32768, "ragged": False, "heads": 12, "kv": 2, "dim": 128,
         "page": 64, "block": 64, "top": 16, "first": 1, "last": 1},
        {"name": "blocks 64 x 32768", "op": "blocks", "seqs": 64, "q": 1, "ctx": 32768, "ragged": True, "heads": 12, "kv": 2, "dim": 128,
         "page": 64, "block": 64, "top": 16, "first": 1, "last": 1},
        # a chunk of a long prompt
        {"name": "blocks 2039 of 16001", "op": "blocks", "seqs": 1, "q": 2039, "ctx": 16001, "ragged": False, "heads": 14, "kv": 2, "dim": 64,
         "page": 128, "block": 64, "top": 16, "first": 1, "last": 1},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["conv", "delta", "delta", "shared", "shared", "blocks", "blocks"])
    if op == "conv":
        channels, q = _spread(rng, 64, 8192), rng.choice([1, 1, _spread(rng, 2, 2048)])
        return {"op": op, "seqs": _spread(rng, 1, max(1, min(128, (1 << 24) // (channels * q)))), "q": q, "ragged": rng.random() < 0.5,
                "channels": channels, "width": rng.choice([2, 3, 4, 4])}
    if op == "delta":
        kheads, q = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, _spread(rng, 2, 64), _spread(rng, 65, 4096)])
        heads = kheads * rng.choice([1, 1, 2])
        return {"op": op, "seqs": _spread(rng, 1, max(1, min(64, (1 << 17) // (heads * q)))), "q": q, "ragged": rng.random() < 0.5,
                "kheads": kheads, "heads": heads, "kdim": rng.choice([64, 128]), "vdim": rng.choice([64, 128])}
    kv, dim, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 256]), rng.choice([32, 64, 128])
    case = {"op": op, "heads": kv * rng.randint(1, 8), "kv": kv, "dim": dim, "page": page, "ragged": rng.random() < 0.7}
    if op == "shared":
        prefix, q = _spread(rng, 33, 16384), rng.choice([1, 1, 1, _spread(rng, 2, 64)])
        seqs = _spread(rng, 1, max(1, min(64, (1 << 25) // (case["heads"] * q * (prefix + 1024)))))
        return case | {"seqs": seqs, "q": q, "prefix": prefix, "ctx": prefix + q + rng.choice([0, _spread(rng, 1, 1024)])}
    block, top = rng.choice([b for b in (32, 64, 128) if b <= page]), rng.choice([4, 8, 16, 24])
    case |= {"block": block, "top": top, "first": rng.choice([0, 1, 2]), "last": rng.choice([0, 1, 3])}
    if rng.random() < 0.6:
        ctx = _spread(rng, 8, 32768)
        return case | {"q": 1, "ctx": ctx, "seqs": _spread(rng, 1, max(1, min(64, (1 << 28) // (ctx * kv * dim))))}
    q = _spread(rng, 2, max(2, min(2039, (1 << 29) // (kv * dim * block * (top + 4)))))
    return case | {"q": q, "ctx": q + rng.choice([0, _spread(rng, 1, 14000)]), "seqs": 1 if q > 200 else rng.randint(1, 5)}


# ---- inputs --------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _heads(g, n, heads, dim):
    """f32 head rows as a projection leaves them: a few channels of each head stand out."""
    return _randn(g, n, heads, dim) * torch.exp(0.5 * _randn(g, heads, dim))


def _queries(case):
    """Tokens of every sequence (from all to half of q) and where they start."""
    n, q = case["seqs"], case["q"]
    qs = torch.tensor([q - (i * q // (2 * n) if case["ragged"] else 0) for i in range(n)], dtype=torch.int32, device="cuda")
    start = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    start[1:] = torch.cumsum(qs, 0)
    return qs, start


def _places(s):
    """Sequence of every token and its place among the sequence's tokens."""
    s["tok_seq"] = torch.repeat_interleave(torch.arange(s["qs"].numel(), device="cuda"), s["qs"].long())
    s["tok_i"] = torch.arange(s["tok_seq"].numel(), device="cuda") - s["start"].long()[s["tok_seq"]]


def _recurrent(case, g):
    qs, start = _queries(case)
    n = case["seqs"]
    slots = torch.randperm(2 * n, generator=g, device="cuda").int()
    s = {"qs": qs, "start": start, "from": slots[:n].clone(), "to": slots[n:].clone()}
    if n > 1:
        s["from"][n // 2] = -1  # a sequence that begins
    return s


def _raw(case, seed):
    """The inputs alone, the same for the plain form, the framework and the exact values."""
    g, op = _gen(seed), case["op"]
    if op == "conv":
        s, C, W = _recurrent(case, g), case["channels"], case["width"]
        return s | {"x": _randn(g, int(s["start"][-1]), C), "w": _randn(g, C, W) * W ** -0.5, "bias": 0.1 * _randn(g, C),
                    "tail": _randn(g, 2 * case["seqs"], W - 1, C)}
    if op == "delta":
        s, H, K = _recurrent(case, g), case["heads"], case["kheads"]
        n = int(s["start"][-1])
        silu = torch.nn.functional.silu
        s |= {"q": silu(_heads(g, n, K, case["kdim"])), "k": silu(_heads(g, n, K, case["kdim"])), "v": silu(_heads(g, n, H, case["vdim"]))}
        s |= {"a": _randn(g, n, H), "b": _randn(g, n, H), "A": torch.log(1 + 15 * torch.rand(H, generator=g, device="cuda"))}
        dt = torch.exp(torch.rand(H, generator=g, device="cuda") * math.log(100.0) + math.log(1e-3))
        return s | {"dt": dt + torch.log(-torch.expm1(-dt)), "state": 0.3 * _randn(g, 2 * case["seqs"], H, case["kdim"], case["vdim"])}
    qs, start = _queries(case)
    n, page, ctx, shared = case["seqs"], case["page"], case["ctx"], case.get("prefix", 0)
    more = ctx - shared - case["q"]  # before a sequence's own tokens; uneven: from all of it to nearly nothing, half on average
    ctxs = qs + shared + torch.tensor([int(more * (1 - 0.618034 * i % 1)) if case["ragged"] else more for i in range(n)], dtype=torch.int32, device="cuda")
    need, per = (ctxs + page - 1) // page, -(-ctx // page)
    live = (torch.arange(per, device="cuda")[None] < need[:, None]) & (torch.arange(per, device="cuda")[None] >= shared // page)
    common = -(-shared // page)
    own_pages = int(live.sum())
    order = torch.randperm(own_pages + common, generator=g, device="cuda").int()
    table = torch.zeros(n, per, dtype=torch.int32, device="cuda")
    table[live] = order[common:]
    table[:, : shared // page] = order[: shared // page]
    s = {"qs": qs, "start": start, "ctx": ctxs, "table": table, "pages": own_pages + common, "q": _heads(g, int(start[-1]), case["heads"], case["dim"])}
    if shared:
        s["prefix"] = order[:common].clone()
    k = _randn(g, s["pages"] * page, case["kv"], case["dim"])
    if op == "blocks":  # neighbouring positions are alike: what makes blocks differ
        k += 0.7 * _randn(g, s["pages"] * page // case["block"], 1, case["kv"], case["dim"]).expand(-1, case["block"], -1, -1).reshape(k.shape)
    return s | {"k": k * torch.exp(0.5 * _randn(g, case["kv"], case["dim"])), "v": _randn(g, s["pages"] * page, case["kv"], case["dim"])}


# ---- the plain forms -----------------------------------------------------------------------------


def _power(e):
    """2^e in f32 for whole e (its bits: a library's pow may be a last bit off)."""
    return ((e + 127) << 23).view(torch.float32)


def _codes(x):
    """4-bit codes (as bytes) and f16 scales of 32-channel blocks of the last axis."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    high, low = b.amax(-1, keepdim=True), b.amin(-1, keepdim=True)
    d = -torch.where(high >= -low, high, low) / 8
    step = _power(torch.clamp(torch.frexp(d)[1] - 8, min=-24))
    d = (torch.round(d / step) * step).clamp(-8160.0, 8160.0)
    c = torch.where(d != 0, torch.round(b / torch.where(d != 0, d, 1.0)), 0.0).clamp(-8, 7) + 8
    return c.to(torch.uint8).reshape(x.shape), d[..., 0].half()


def _values(c, d):
    return ((c.float() - 8).reshape(*d.shape, 32) * d.float()[..., None]).reshape(c.shape)


def _padded(s, x):
    """Rows of tokens as [sequence][place]."""
    y = torch.zeros(s["case"]["seqs"], s["case"]["q"], *x.shape[1:], dtype=x.dtype, device="cuda")
    y[s["tok_seq"], s["tok_i"]] = x
    return y


def _begin(s, pool):
    """The sequences' states before the call."""
    at = s["from"].long()
    return pool[at.clamp(min=0)] * (at >= 0).reshape(-1, *[1] * (pool.dim() - 1))


def _plain_conv(s):
    W, qs = s["case"]["width"], s["qs"].long()
    rows = torch.cat([_begin(s, s["tail"]), _padded(s, s["x"])], 1)  # [sequence][W - 1 + q][channel]
    y = (rows.unfold(1, W, 1) * s["w"]).sum(-1) + s["bias"]
    last = qs[:, None] + torch.arange(W - 1, device="cuda")
    s["tail"][s["to"].long()] = rows.gather(1, last[..., None].expand(-1, -1, rows.shape[-1]))
    y = y[s["tok_seq"], s["tok_i"]]
    return [y / (1 + torch.exp(-y)), s["tail"]]


def _plain_delta(s):
    case, C = s["case"], min(64, s["case"]["q"])
    S, H, N = case["seqs"], case["heads"], -(-case["q"] // C)

    def chunks(x):  # [sequence][chunk][head][token of the chunk][..]
        x = _padded(s, x)
        x = torch.nn.functional.pad(x, [0, 0] * (x.dim() - 2) + [0, N * C - x.shape[1]])
        return x.reshape(S, N, C, *x.shape[2:]).transpose(2, 3)

    def unit(x):
        x = x * torch.rsqrt((x * x).sum(-1, keepdim=True) + NORM_EPS)
        return chunks(x).repeat_interleave(H // case["kheads"], 2)

    q, k, v = unit(s["q"]) * case["kdim"] ** -0.5, unit(s["k"]), chunks(s["v"])
    decay = chunks(-torch.exp(s["A"]) * torch.logaddexp(s["a"] + s["dt"], torch.zeros_like(s["a"])))
    rate = chunks(1 / (1 + torch.exp(-s["b"])))[..., None]
    g = torch.cumsum(decay.double(), -1)
    lower = torch.ones(C, C, dtype=torch.bool, device="cuda").tril()
    D = torch.exp(torch.where(lower, g[..., :, None] - g[..., None, :], -math.inf).float())
    A = (torch.matmul(k * rate, k.transpose(-1, -2).contiguous()) * D).tril(-1)
    T = torch.eye(C, device="cuda") - A
    for i in range(2, C):  # the inverse of I + A, row by row
        T[..., i, :i] -= torch.matmul(A[..., i, None, 1:i], T[..., 1:i, :i] - torch.eye(C, device="cuda")[1:i, :i])[..., 0, :]
    eg = torch.exp(g.float())[..., None]
    U, W = torch.matmul(T, v * rate), torch.matmul(T, k * rate * eg)
    P = (torch.matmul(q, k.transpose(-1, -2).contiguous()) * D)
    q, k = q * eg, (k * torch.exp((g[..., -1:] - g).float())[..., None]).transpose(-1, -2).contiguous()
    state, out = _begin(s, s["state"]), []
    for n in range(N):
        u = U[:, n] - torch.matmul(W[:, n], state)
        out.append(torch.matmul(q[:, n], state) + torch.matmul(P[:, n], u))
        state = state * eg[:, n, :, -1:] + torch.matmul(k[:, n], u)
    s["state"][s["to"].long()] = state
    o = torch.stack(out, 1).transpose(2, 3).reshape(S, N * C, H, -1)
    return [o[s["tok_seq"], s["tok_i"]], s["state"]]


def _rows(s, pages):
    """k and v of the positions of pages [..][page], as [..][kv][position][dim]."""
    both = []
    for c, d in ((s["kc"], s["kd"]), (s["vc"], s["vd"])):
        x = _values(c[pages.long()], d[pages.long()])
        both.append(x.reshape(*pages.shape[:-1], -1, *x.shape[-2:]).transpose(-2, -3).contiguous())
    return both


def _plain_shared(s):
    case, kv, dim, P = s["case"], s["case"]["kv"], s["case"]["dim"], s["case"]["prefix"]
    G, S, Q, skip = case["heads"] // kv, case["seqs"], case["q"], P // case["page"]
    q = (_padded(s, s["q"]).reshape(S, Q, kv, G, dim) * dim ** -0.5).permute(0, 2, 1, 3, 4).reshape(S, kv, Q * G, dim)
    K, V = _rows(s, s["prefix"])
    K, V = K[:, :P].contiguous(), V[:, :P].contiguous()
    k, v = _rows(s, s["table"][:, skip:])
    together = q.transpose(0, 1).reshape(kv, S * Q * G, dim)
    w = torch.matmul(together, K.transpose(1, 2).contiguous())  # the prefix, once for all
    x = torch.matmul(q, k.transpose(2, 3).contiguous())
    pos = (s["ctx"] - s["qs"])[:, None] + torch.arange(Q, device="cuda")
    key = skip * case["page"] + torch.arange(x.shape[-1], device="cuda")
    see = (key <= pos[..., None]) & (key >= P)
    x = x.reshape(S, kv, Q, G, -1).masked_fill_(~see[:, None, :, None], -math.inf).reshape(S, kv, Q * G, -1)
    w = w.reshape(kv, S, Q * G, P).transpose(0, 1)
    top = torch.maximum(w.amax(-1, keepdim=True), x.amax(-1, keepdim=True))
    w, x = torch.exp(w - top), torch.exp(x - top)
    o = torch.matmul(w.transpose(0, 1).reshape(kv, S * Q * G, P), V).reshape(kv, S, Q * G, dim).transpose(0, 1) + torch.matmul(x, v)
    o = (o / (w.sum(-1) + x.sum(-1))[..., None]).reshape(S, kv, Q, G, dim).transpose(1, 2)
    return [o[s["tok_seq"], s["tok_i"]].reshape(-1, kv * G, dim)]


def _mean(values):
    """Means over the positions of blocks of f16 values [..][position][kv][dim]: the exact sum rounded to f32, then f16."""
    return values.double().mean(-3).float().half()


def _plain_blocks(s):
    case, kv, dim, B = s["case"], s["case"]["kv"], s["case"]["dim"], s["case"]["block"]
    G, S, Q, page = case["heads"] // kv, case["seqs"], case["q"], case["page"]
    per = page // B
    done = s["pos"] % B == B - 1
    at = s["table"][s["seq"].long(), (s["pos"] // page).long()][done].long(), (s["pos"] % page // B)[done].long()
    kc, kd = (x.reshape(-1, per, B, kv, x.shape[-1]) for x in (s["kc"], s["kd"]))
    vc, vd = (x.reshape(-1, per, B, kv, x.shape[-1]) for x in (s["vc"], s["vd"]))
    s["means"][at] = _mean(_values(kc[at], kd[at]))
    # scores of every block, and the highest of those that are not read anyway
    q = _padded(s, s["q"]).reshape(S, Q, kv, G, dim).transpose(1, 2)
    M = s["means"][s["table"].long()].reshape(S, -1, kv, dim).permute(0, 2, 3, 1).double().contiguous()
    score = torch.matmul(q.double().sum(3) * dim ** -0.5, M)  # [S, kv, Q, block]
    n, pos = score.shape[-1], (s["ctx"] - s["qs"])[:, None] + torch.arange(Q, device="cuda")
    block, mine = torch.arange(n, device="cuda"), (pos // B)[:, None, :, None]
    fixed = ((block < case["first"]) | (block >= mine - case["last"])) & (block <= mine)
    score = torch.where(fixed | (block > mine), -math.inf, score)
    best, order = torch.sort(score, dim=-1, descending=True, stable=True)
    top = min(case["top"], n)
    chosen = torch.where(best[..., :top] > -math.inf, order[..., :top], n).sort(-1).values
    chosen = torch.nn.functional.pad(chosen, (0, case["top"] - top), value=n)
    read = torch.zeros(S, kv, Q, n + 1, dtype=torch.bool, device="cuda").scatter_(-1, chosen, True)[..., :n] | fixed
    width = min(n, top + case["first"] + case["last"] + 1)
    taken, which = torch.sort((~read).int(), dim=-1, stable=True)
    taken, which = taken[..., :width] == 0, which[..., :width]  # [S, kv, Q, width]
    # their keys and values
    where = s["table"].long().repeat_interleave(per, 1)[torch.arange(S, device="cuda")[:, None, None, None], which]
    place = where, which % per, slice(None), torch.arange(kv, device="cuda")[:, None, None]
    K, V = (_values(c[place], d[place]).reshape(S, kv, Q, width * B, dim) for c, d in ((kc, kd), (vc, vd)))
    w = torch.matmul(q * dim ** -0.5, K.transpose(-1, -2).contiguous())
    key = which[..., None] * B + torch.arange(B, device="cuda")
    see = (taken[..., None] & (key <= pos[:, None, :, None, None])).reshape(S, kv, Q, 1, -1)
    w = w.masked_fill_(~see, -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    o = torch.nan_to_num(torch.matmul(w, V) / w.sum(-1, keepdim=True)).transpose(1, 2)
    chosen = torch.where(chosen < n, chosen, -1).int().transpose(1, 2)
    return [o[s["tok_seq"], s["tok_i"]].reshape(-1, kv * G, dim), chosen[s["tok_seq"], s["tok_i"]], s["means"]]


# ---- the passes ----------------------------------------------------------------------------------


def _tokens(seq, pos, table):
    return {"seq_ptr": seq.data_ptr(), "pos_ptr": pos.data_ptr(), "n_tok": seq.numel(), "table_ptr": table.data_ptr(),
            "n_seq": table.shape[0], "table_stride": table.shape[1]}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def prepare(case, seed):
    s = _raw(case, seed) | {"case": case}
    op = case["op"]
    _places(s)
    if op in ("conv", "delta"):
        if own:
            from apeiron_amd import chart

            s["dev"], s["out"] = chart.device(), torch.zeros_like(s["x"] if op == "conv" else s["v"])
        return s
    n, page, kv, dim = s["pages"], case["page"], case["kv"], case["dim"]
    # every slot of the cache's pages
    every = {"seq": torch.zeros(n * page, dtype=torch.int32, device="cuda"), "pos": torch.arange(n * page, dtype=torch.int32, device="cuda"),
             "table": torch.arange(n, dtype=torch.int32, device="cuda")[None].contiguous()}
    s["seq"], s["pos"] = s["tok_seq"].int(), ((s["ctx"] - s["qs"])[s["tok_seq"]] + s["tok_i"]).int()
    if op == "blocks":
        s["means"] = torch.zeros(n, page // case["block"], kv, dim, dtype=torch.float16, device="cuda")
    if own:
        from apeiron_amd import chart

        cache = s["cache"] = chart.KvCache4(chart.device(), n, page, kv, dim)
        cache.append_dev(None, k_ptr=s["k"].data_ptr(), v_ptr=s["v"].data_ptr(), stream=_stream(), **_tokens(**every))
        if op == "blocks":
            cache.block_means_dev(s["means"].data_ptr(), block_len=case["block"], stream=_stream(), **_tokens(**every))
            s["chosen"] = torch.zeros(s["q"].shape[0], kv, case["top"], dtype=torch.int32, device="cuda")
        s["out"] = torch.zeros_like(s["q"])
        torch.cuda.synchronize()
    else:
        for name in ("k", "v"):
            c, d = _codes(s[name])
            s[name + "c"], s[name + "d"] = c.reshape(n, page, kv, dim), d.reshape(n, page, kv, dim // 32)
        if op == "blocks":
            s["means"] = _mean(_values(s["kc"], s["kd"]).reshape(n, page // case["block"], case["block"], kv, dim))
    del s["k"], s["v"]
    return s


def run(s):
    case, op = s["case"], s["case"]["op"]
    if not own:
        return {"conv": _plain_conv, "delta": _plain_delta, "shared": _plain_shared, "blocks": _plain_blocks}[op](s)
    from apeiron_amd import chart

    stream, out = _stream(), s["out"]
    if op in ("conv", "delta"):
        seqs = {"n_tok": out.shape[0], "n_seq": case["seqs"], "max_q": case["q"], "q_start_ptr": s["start"].data_ptr(), "from_ptr": s["from"].data_ptr(),
                "to_ptr": s["to"].data_ptr(), "n_slots": 2 * case["seqs"], "stream": stream}
    else:
        seqs = {"n_heads": case["heads"], "n_tok": out.shape[0], "n_seq": case["seqs"], "q_start_ptr": s["start"].data_ptr(), "ctx_ptr": s["ctx"].data_ptr(),
                "table_ptr": s["table"].data_ptr(), "table_stride": s["table"].shape[1], "max_q": case["q"], "max_ctx": case["ctx"],
                "scale": case["dim"] ** -0.5, "stream": stream}
    if op == "conv":
        chart.conv_dev(s["dev"], s["x"].data_ptr(), out.data_ptr(), n_channels=case["channels"], width=case["width"], weight_ptr=s["w"].data_ptr(),
                       bias_ptr=s["bias"].data_ptr(), silu=True, state_ptr=s["tail"].data_ptr(), **seqs)
        return [out, s["tail"]]
    if op == "delta":
        chart.delta_rule_dev(s["dev"], s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["a"].data_ptr(), s["b"].data_ptr(), out.data_ptr(),
                             n_heads=case["heads"], n_k_heads=case["kheads"], k_dim=case["kdim"], v_dim=case["vdim"], a_log_ptr=s["A"].data_ptr(),
                             dt_bias_ptr=s["dt"].data_ptr(), scale=case["kdim"] ** -0.5, norm_eps=NORM_EPS, state_ptr=s["state"].data_ptr(), **seqs)
        return [out, s["state"]]
    if op == "shared":
        s["cache"].attn_shared_dev(s["q"].data_ptr(), out.data_ptr(), prefix_len=case["prefix"], prefix_table_ptr=s["prefix"].data_ptr(), **seqs)
        return [out]
    s["cache"].block_means_dev(s["means"].data_ptr(), block_len=case["block"], stream=stream, **_tokens(s["seq"], s["pos"], s["table"]))
    s["cache"].attn_blocks_dev(s["q"].data_ptr(), out.data_ptr(), means_ptr=s["means"].data_ptr(), block_len=case["block"], n_top=case["top"],
                               n_first=case["first"], n_last=case["last"], chosen_ptr=s["chosen"].data_ptr(), **seqs)
    return [out, s["chosen"], s["means"]]


def work(case):
    op, S = case["op"], case["seqs"]
    tokens = sum(case["q"] - (i * case["q"] // (2 * S) if case["ragged"] else 0) for i in range(S))
    if op == "conv":
        C, W = case["channels"], case["width"]
        return {"bytes": 8 * tokens * C + 8 * S * (W - 1) * C + 4 * C * (W + 1), "flops": tokens * C * (2 * W + 5)}
    if op == "delta":
        H, dk, dv = case["heads"], case["kdim"], case["vdim"]
        return {"bytes": 4 * tokens * (2 * case["kheads"] * dk + 2 * H * dv + 2 * H) + 8 * S * H * dk * dv, "flops": 7 * tokens * H * dk * dv}
    kv, D, H = case["kv"], case["dim"], case["heads"]
    # uneven contexts: half of what may stand before a sequence's tokens, as they are drawn
    own_keys = sum((case["ctx"] - case.get("prefix", 0) - case["q"]) // (2 if case["ragged"] and i else 1) + case["q"] for i in range(S))
    ends = 8 * tokens * H * D
    if op == "shared":
        keys = case["prefix"] + own_keys
        return {"bytes": keys * kv * D * 9 // 8 + ends, "flops": 4 * H * D * (tokens * case["prefix"] + tokens * own_keys // S)}
    B = case["block"]
    seen = min(own_keys // S, (case["top"] + case["first"] + case["last"]) * B + B // 2)
    keys = min(own_keys, tokens * seen)  # what the tokens read together, or all of it once
    means = own_keys // B * kv * D * 2
    return {"bytes": keys * kv * D * 9 // 8 + means + ends + 4 * tokens * kv * case["top"],
            "flops": 4 * H * D * tokens * seen + 2 * kv * D * tokens * own_keys // S // B}


# ---- 64 bits -------------------------------------------------------------------------------------


def _exact_cache(x):
    """f64 values of the cache for f32 rows, from the format's definition."""
    b = x.double().unflatten(-1, (-1, 32))
    top, bottom = b.max(-1, keepdim=True).values, b.min(-1, keepdim=True).values
    d = torch.where(top + bottom >= 0, top, bottom) / -8
    unit = ((torch.floor(torch.log2(d.abs().clamp(min=1e-300))) - 7).clamp(min=-24).long() + 1023 << 52).view(torch.float64)
    d = (torch.round(d / unit) * unit).clamp(-8160, 8160)
    # the code is the nearest to the quotient's f32 value (this rounding of the f64 quotient gives it exactly)
    q = torch.round((b / torch.where(d == 0, 1.0, d)).float().double()).clamp(-8, 7)
    return (q * d).flatten(-2)


def _exact_conv(case, s):
    W = case["width"]
    tail, out = s["tail"].double(), torch.zeros_like(s["x"], dtype=torch.float64)
    for i in range(case["seqs"]):
        a, b, src = int(s["start"][i]), int(s["start"][i + 1]), int(s["from"][i])
        before = s["tail"][src].double() if src >= 0 else torch.zeros_like(tail[0])
        x = torch.cat([before, s["x"][a:b].double()])
        y = s["bias"].double() + sum(x[j: j + b - a] * s["w"][:, j].double() for j in range(W))
        out[a:b] = y * torch.sigmoid(y)
        tail[int(s["to"][i])] = x[b - a:]
    return [out, tail]


def _exact_delta(case, s):
    r = case["heads"] // case["kheads"]
    q, k = (torch.repeat_interleave(x.double() / torch.sqrt(x.double().square().sum(-1, keepdim=True) + NORM_EPS), r, 1) for x in (s["q"], s["k"]))
    v, rate = s["v"].double(), torch.sigmoid(s["b"].double())
    x = s["a"].double() + s["dt"].double()
    keep = torch.exp(-torch.exp(s["A"].double()) * (x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))))
    src = s["from"].long()
    S = torch.where((src >= 0)[:, None, None, None], s["state"].double()[src.clamp(min=0)], 0.0)
    out, first = torch.zeros_like(v), s["start"].long()
    for t in range(case["q"]):
        on = (s["qs"] > t).nonzero()[:, 0]  # the sequences that have a token here
        i = first[on] + t
        R = S[on] * keep[i][..., None, None]
        u = rate[i][..., None] * (v[i] - (k[i][..., None, :] @ R)[..., 0, :])
        R = R + k[i][..., None] * u[..., None, :]
        S[on] = R
        out[i] = (q[i][..., None, :] @ R)[..., 0, :] / math.sqrt(case["kdim"])
    state = s["state"].double()
    state[s["to"].long()] = S
    return [out, state]


def _exact_attention(q, K, V, see):
    """f64 attention of rows q [token][head of the group][dim] over K, V [position][dim] where see [token][position]."""
    w = (q @ K.T) / math.sqrt(q.shape[-1])
    return torch.softmax(torch.where(see[:, None], w, -math.inf), -1) @ V


def exact(case, seed):
    s, op = _raw(case, seed), case["op"]
    if op == "conv":
        return _exact_conv(case, s)
    if op == "delta":
        return _exact_delta(case, s)
    kv, page, shared = case["kv"], case["page"], case.get("prefix", 0)
    G, B = case["heads"] // kv, case.get("block", 0)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    chosen = torch.full((s["q"].shape[0], kv, case.get("top", 0)), -1, dtype=torch.int32, device="cuda")
    for i in range(case["seqs"]):
        n, ctx, at = int(s["qs"][i]), int(s["ctx"][i]), int(s["start"][i])
        key = torch.arange(ctx, device="cuda")
        slots = s["table"][i].long()[key // page] * page + key % page
        if shared:
            slots = torch.where(key < shared, s["prefix"].long()[(key // page).clamp(max=s["prefix"].numel() - 1)] * page + key % page, slots)
        for h in range(kv):
            K, V = _exact_cache(s["k"][slots, h]), _exact_cache(s["v"][slots, h])
            step = max(1, (1 << 27) // (ctx * G))
            for j in range(0, n, step):
                m = min(step, n - j)
                rows = slice(at + j, at + j + m)
                q = s["q"][rows, h * G: (h + 1) * G].double()
                pos = ctx - n + j + torch.arange(m, device="cuda")[:, None]
                see = key <= pos
                if op == "blocks":
                    whole = ctx // B
                    means = K[: whole * B].reshape(whole, B, -1).mean(1).float().half().double()
                    block, mine = torch.arange(-(-ctx // B), device="cuda"), pos // B
                    always = (block < case["first"]) | ((mine - block >= 0) & (mine - block <= case["last"]))
                    rank = torch.full((m, block.numel()), -math.inf, dtype=torch.float64, device="cuda")
                    rank[:, :whole] = q.sum(1) @ means.T
                    rank[always | (block > mine)] = -math.inf
                    order = torch.argsort(rank, dim=-1, descending=True, stable=True)[:, : case["top"]]
                    good = torch.gather(rank, 1, order) > -math.inf
                    pick = torch.zeros(m, block.numel() + 1, dtype=torch.bool, device="cuda")
                    pick.scatter_(1, torch.where(good, order, block.numel()), True)
                    see = see & (pick[:, :-1] | always)[:, key // B]
                    found = torch.where(good, order, 1 << 30).sort(-1).values.int()
                    chosen[rows, h, : found.shape[1]] = torch.where(found < 1 << 30, found, -1)
                out[rows, h * G: (h + 1) * G] = _exact_attention(q, K, V, see)
    if op == "shared":
        return [out]
    means = torch.cat([_exact_cache(x).reshape(-1, B, kv, case["dim"]).mean(1) for x in s["k"].split(1 << 18)])
    return [out, chosen, means.reshape(s["pages"], page // B, kv, case["dim"])]
