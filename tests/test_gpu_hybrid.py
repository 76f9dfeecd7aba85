"""The operators whose cost does not follow the whole context, together, as a server of a hybrid model runs them: a
common prompt once, a batch of prompts from where it ended, then a token a step for all of them, captured as a graph.

Three layers: norm, projection, short convolution, gated delta rule; attention behind the batch's common prefix; attention
over blocks. Everything is compared with 64-bit layers over each sequence's whole text. Those take the cache's values as
they were stored (an f32 rounding can move a 4-bit code, which is a step of an eighth and no error of these operators),
having found each within a code of their own, and the blocks as they were chosen, having found none left out that
scores more than the rounding above one taken.

Tolerance, root mean square: projections of n products leave about sqrt(n) 2^-24, 1e-6, attention as much, the norm,
convolution and delta rule less. A layer has four of these one after the other, an error of a score comes out of the softmax
as large as it is (scores are a few units), and the residual stream adds the layers: 3 * 4 * 1e-6 times about 4, under 1e-4.
A wrong state, page or block changes outputs by tenths.
"""
import numpy as np
import pytest

from apeiron_amd import chart
from test_gpu_token_ops import OK, cuda, dev, ptr, stream  # noqa: F401

torch = pytest.importorskip("torch")

N, K, H, DK, DV, HEADS, KV, D, PAGE, BLOCK, TOP = 256, 2, 4, 64, 64, 4, 2, 64, 32, 32, 3
C = 2 * K * DK + H * DV
PREFIX, STEPS = 192, 6


class Model:
    def __init__(self, d, prompts):
        g = torch.Generator().manual_seed(len(prompts))
        r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
        self.d, self.prompts, self.n = d, prompts, len(prompts)
        self.gain = [1 + 0.1 * r(N) for _ in range(3)]
        self.w = {k: r(N, m) / N ** 0.5 for k, m in (("conv", C), ("ab", 2 * H), ("shared", (HEADS + 2 * KV) * D), ("blocks", (HEADS + 2 * KV) * D))}
        self.o = [r(m, N) / m ** 0.5 for m in (H * DV, HEADS * D, HEADS * D)]
        self.taps, self.A, self.dt = 0.5 * r(C, 4), torch.rand(H, generator=g).cuda() * 2, r(H) - 3
        self.length = [PREFIX + p + STEPS for p in prompts]
        common = r(PREFIX, N)
        self.x = [torch.cat([common, r(n - PREFIX, N)]) for n in self.length]
        # a slot for the prefix and one for each sequence; pages of the prefix and of each sequence after it
        self.tail, self.state = torch.full((self.n + 1, 3, C), 9.0, device="cuda"), torch.full((self.n + 1, H, DK, DV), 9.0, device="cuda")
        self.per = -(-max(self.length) // PAGE)
        own = self.per - PREFIX // PAGE
        page = torch.randperm(PREFIX // PAGE + self.n * own, generator=g).int()
        self.prefix = page[: PREFIX // PAGE].cuda()
        self.table = torch.cat([self.prefix.expand(self.n, -1), page[PREFIX // PAGE:].reshape(self.n, own).cuda()], 1).contiguous()
        self.cache = [chart.KvCache4(d, page.numel(), PAGE, KV, D) for _ in range(2)]
        self.means = torch.zeros(page.numel(), PAGE // BLOCK, KV, D, dtype=torch.float16, device="cuda")

    def arrays(self, qs, ctx, src, dst):
        i32 = lambda v: cuda(np.asarray(v, np.int32))  # noqa: E731
        return dict(start=i32(np.concatenate([[0], np.cumsum(qs)])), ctx=i32(ctx), src=i32(src), dst=i32(dst), seq=i32(np.repeat(np.arange(len(qs)), qs)),
                    pos=i32(np.concatenate([c - q + np.arange(q) for q, c in zip(qs, ctx)])), n_seq=len(qs), n_tok=sum(qs), max_q=max(qs))

    def run(self, x, t, shared):
        """The layers over the rows x of the sequences t."""
        d, n, st = self.d, t["n_tok"], stream()
        y, z, c, out = (torch.empty(n, m, device="cuda") for m in (N, C, C, H * DV))
        chosen = torch.full((n, KV, TOP), -7, dtype=torch.int32, device="cuda")

        def norm(x, i):
            chart.norm_quant_dev(d, ptr(x), ptr(self.gain[i]), 1e-6, n, N, y_ptr=ptr(y), stream=st)
            return y

        # the recurrent layer
        torch.mm(norm(x, 0), self.w["conv"], out=z)
        ab = torch.mm(y, self.w["ab"])
        seqs = dict(n_seq=t["n_seq"], n_tok=n, max_q=t["max_q"], n_slots=self.n + 1, q_start_ptr=ptr(t["start"]), from_ptr=ptr(t["src"]), to_ptr=ptr(t["dst"]), stream=st)
        chart.conv_dev(d, ptr(z), ptr(c), n_channels=C, width=4, weight_ptr=ptr(self.taps), silu=True, state_ptr=ptr(self.tail), **seqs)
        chart.delta_rule_dev(d, ptr(c), ptr(c) + 4 * K * DK, ptr(c) + 8 * K * DK, ptr(ab), ptr(ab) + 4 * H, ptr(out), n_heads=H, n_k_heads=K, k_dim=DK, v_dim=DV,
                             a_log_ptr=ptr(self.A), dt_bias_ptr=ptr(self.dt), scale=DK ** -0.5, norm_eps=1e-6, state_ptr=ptr(self.state), q_stride=C, k_stride=C,
                             v_stride=C, a_stride=2 * H, b_stride=2 * H, **seqs)
        x = x + torch.mm(out, self.o[0])
        # the attention layers
        for i, name in ((1, "shared"), (2, "blocks")):
            qkv, cache = torch.mm(norm(x, i), self.w[name]), self.cache[i - 1]
            width = qkv.shape[1]
            tokens = dict(seq_ptr=ptr(t["seq"]), pos_ptr=ptr(t["pos"]), n_tok=n, table_ptr=ptr(self.table), n_seq=t["n_seq"], table_stride=self.per, stream=st)
            cache.append_dev(None, k_ptr=ptr(qkv) + 4 * HEADS * D, k_stride=width, v_ptr=ptr(qkv) + 4 * (HEADS + KV) * D, v_stride=width, **tokens)
            a = dict(n_heads=HEADS, n_tok=n, n_seq=t["n_seq"], q_start_ptr=ptr(t["start"]), ctx_ptr=ptr(t["ctx"]), table_ptr=ptr(self.table), table_stride=self.per,
                     max_q=t["max_q"], max_ctx=self.per * PAGE, scale=D ** -0.5, q_stride=width, stream=st)
            o = torch.empty(n, HEADS * D, device="cuda")
            if name == "blocks":
                cache.block_means_dev(ptr(self.means), block_len=BLOCK, **tokens)
                cache.attn_blocks_dev(ptr(qkv), ptr(o), means_ptr=ptr(self.means), block_len=BLOCK, n_top=TOP, n_first=1, n_last=1, chosen_ptr=ptr(chosen), **a)
            else:
                cache.attn_shared_dev(ptr(qkv), ptr(o), prefix_len=shared, prefix_table_ptr=ptr(self.prefix), **a)
            x = x + torch.mm(o, self.o[i])
        return x, chosen

    def reference(self, s, chosen):
        """64-bit layers over all of sequence s: outputs, and the delta rule's last state."""
        T, f = self.length[s], lambda t: t.double()  # noqa: E731
        x = f(self.x[s])
        norm = lambda x, i: x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * f(self.gain[i])  # noqa: E731
        y = norm(x, 0)
        z = torch.cat([torch.zeros(3, C, device="cuda").double(), y @ f(self.w["conv"])])
        c = torch.nn.functional.silu(sum(z[i:i + T] * f(self.taps)[:, i] for i in range(4)))
        ab = y @ f(self.w["ab"])
        q, k, v = c[:, : K * DK].reshape(T, K, DK), c[:, K * DK: 2 * K * DK].reshape(T, K, DK), c[:, 2 * K * DK:].reshape(T, H, DV)
        q, k = ((t / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-6)).repeat_interleave(H // K, 1) for t in (q, k))
        keep, rate = torch.exp(-torch.exp(f(self.A)) * torch.nn.functional.softplus(ab[:, :H] + f(self.dt))), torch.sigmoid(ab[:, H:])
        S, out = torch.zeros(H, DK, DV, device="cuda").double(), torch.zeros(T, H, DV, device="cuda").double()
        for t in range(T):
            S = S * keep[t, :, None, None]
            u = rate[t, :, None] * (v[t] - (S * k[t, :, :, None]).sum(1))
            S = S + k[t, :, :, None] * u[:, None, :]
            out[t] = (S * q[t, :, :, None]).sum(1) * DK ** -0.5
        x = x + out.reshape(T, -1) @ f(self.o[0])
        pos = torch.arange(T, device="cuda")
        for i, name in ((1, "shared"), (2, "blocks")):
            qkv = norm(x, i) @ f(self.w[name])
            q, kv = qkv[:, : HEADS * D].reshape(T, HEADS, D), qkv[:, HEADS * D:].reshape(T, 2, KV, D)
            held = torch.empty(2, T, KV, D, dtype=torch.float16, device="cuda")
            where = cuda(np.full(T, s, np.int32)), cuda(np.arange(T, dtype=np.int32))
            self.cache[i - 1].read_dev(k_ptr=ptr(held[0]), v_ptr=ptr(held[1]), seq_ptr=ptr(where[0]), pos_ptr=ptr(where[1]), n_tok=T, table_ptr=ptr(self.table),
                                       n_seq=self.n, table_stride=self.per, stream=stream())
            step = kv.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True) / 8  # of a code; its largest positive one is 7, so up to a whole step there
            assert ((held.double().transpose(0, 1) - kv).unflatten(-1, (-1, 32)).abs() <= 1.02 * step).all()
            k, v = f(held)
            see = (pos[None] <= pos[:, None]).expand(KV, T, T)
            if name == "blocks":
                blocks = T // BLOCK
                mean = k[: blocks * BLOCK].reshape(blocks, BLOCK, KV, D).mean(1).float().half().double()
                score = torch.bmm(q.reshape(T, KV, HEADS // KV, D).sum(2).transpose(0, 1).contiguous(), mean.permute(1, 2, 0).contiguous()) * D ** -0.5
                own, b = pos // BLOCK, torch.arange(blocks, device="cuda")
                middle = ((b[None] >= 1) & (b[None] < own[:, None] - 1)).expand(KV, T, blocks)
                pick = chosen[s].transpose(0, 1).long()  # [KV][T][TOP]
                taken = torch.zeros(KV, T, blocks + 1, dtype=torch.bool, device="cuda").scatter_(2, torch.where(pick < 0, blocks, pick), True)[:, :, :blocks]
                assert (taken.sum(-1) == middle.sum(-1).clamp(max=TOP)).all() and (middle | ~taken).all()
                least = torch.where(taken, score, torch.inf).amin(-1)
                assert (torch.where(middle & ~taken, score, -torch.inf).amax(-1) <= least + 1e-4).all()
                key = pos // BLOCK
                read = torch.cat([taken, torch.zeros(KV, T, 1, dtype=torch.bool, device="cuda")], 2)[:, :, key.clamp(max=blocks)]
                see = see & (read | (key == 0)[None, None] | (key[None] >= own[:, None] - 1)[None])
            kk, vv = (t.repeat_interleave(HEADS // KV, 1).transpose(0, 1) for t in (k, v))
            p = torch.softmax(torch.where(see.repeat_interleave(HEADS // KV, 0), torch.bmm(q.transpose(0, 1).contiguous(), kk.transpose(1, 2).contiguous()) * D ** -0.5, -torch.inf), -1)
            x = x + torch.bmm(p, vv.contiguous()).transpose(0, 1).reshape(T, -1) @ f(self.o[i])
        return x, S


@pytest.mark.gpu
@pytest.mark.parametrize("prompts", [[3, 40, 1, 17, 90], [33], [1] * 12, [300, 2, 150]])
def test_a_hybrid_model_serves_a_batch_behind_a_common_prompt(dev, prompts):  # noqa: F811
    d = chart.Device(0)
    M = Model(d, prompts)
    n = M.n
    out, chosen = [[] for _ in prompts], [[] for _ in prompts]

    def keep(x, pick, qs):
        at = 0
        for s, q in enumerate(qs):
            out[s].append(x[at:at + q].clone())
            chosen[s].append(pick[at:at + q].clone())
            at += q

    # the prefix by itself, into slot 0 (its pages are in every row of the table), then the prompts from there
    x, pick = M.run(M.x[0][:PREFIX].contiguous(), M.arrays([PREFIX], [PREFIX], [-1], [0]), 0)
    for s in range(n):
        out[s].append(x)
        chosen[s].append(pick)
    t = M.arrays(prompts, [PREFIX + p for p in prompts], [0] * n, [s + 1 for s in range(n)])
    kept = M.state[0].clone(), M.tail[0].clone()
    keep(*M.run(torch.cat([M.x[s][PREFIX:PREFIX + p] for s, p in enumerate(prompts)]), t, PREFIX), prompts)
    assert torch.equal(M.state[0], kept[0]) and torch.equal(M.tail[0], kept[1])
    assert d.sync_status(stream()) == OK

    # steps: one eager, the others replays of a graph of the same arrays, with eager work of the context between
    t = M.arrays([1] * n, [PREFIX + p + 1 for p in prompts], [s + 1 for s in range(n)], [s + 1 for s in range(n)])
    row = torch.stack([M.x[s][PREFIX + p] for s, p in enumerate(prompts)])

    def step():
        x, pick = M.run(row, t, PREFIX)
        t["ctx"].add_(1)
        t["pos"].add_(1)
        return x, pick

    torch.cuda.synchronize()
    keep(*step(), [1] * n)
    graph, other = torch.cuda.CUDAGraph(), Model(d, [700, 5])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        x, pick = step()
    for i in range(1, STEPS):
        row.copy_(torch.stack([M.x[s][PREFIX + p + i] for s, p in enumerate(prompts)]))
        graph.replay()
        torch.cuda.synchronize()
        keep(x, pick, [1] * n)
        other.run(other.x[0], other.arrays([PREFIX + 700 + STEPS], [PREFIX + 700 + STEPS], [-1], [1]), 0)
        torch.cuda.synchronize()
    assert d.sync_status(stream()) == OK

    for s in range(n):
        want, S = M.reference(s, [torch.cat(c) for c in chosen])
        got = torch.cat(out[s]).double()
        assert got.shape == want.shape
        error = (got - want).square().mean(-1).sqrt() / want.square().mean(-1).sqrt()
        assert (error <= 1e-4).all(), (s, error.max(), error.argmax())
        assert (M.state[s + 1] - S).square().mean().sqrt() <= 1e-4 * S.square().mean().sqrt()
    for model in (M, other):
        for c in model.cache:
            c.free()
    d.close()


def prompt_pass(M, prompts):
    """What a pass over prompts behind the prefix needs, and the pass: from slot 0 and the prefix's pages, so that it may be repeated."""
    M.run(M.x[0][:PREFIX].contiguous(), M.arrays([PREFIX], [PREFIX], [-1], [0]), 0)
    t = M.arrays(prompts, [PREFIX + p for p in prompts], [0] * M.n, [s + 1 for s in range(M.n)])
    x = torch.cat([M.x[s][PREFIX:PREFIX + p] for s, p in enumerate(prompts)])
    torch.cuda.synchronize()
    return lambda: M.run(x, t, PREFIX)


@pytest.mark.gpu
def test_two_contexts_at_once_on_two_streams(dev):  # noqa: F811
    """Contexts have scratch of their own: passes that run at the same time leave what each leaves alone."""
    devices, streams, kinds = [chart.Device(0), chart.Device(0)], [torch.cuda.Stream(), torch.cuda.Stream()], ([300, 2, 150], [64, 64, 64, 64, 64])
    models = [Model(d, p) for d, p in zip(devices, kinds)]
    passes = [prompt_pass(M, p) for M, p in zip(models, kinds)]
    want = []
    for M, go in zip(models, passes):
        x, pick = go()
        torch.cuda.synchronize()
        want.append((x.clone(), pick.clone(), M.state.clone(), M.tail.clone()))
    for _ in range(5):
        got = []
        for st, go in zip(streams, passes):
            with torch.cuda.stream(st):
                got.append(go())
        torch.cuda.synchronize()
        for M, (x, pick), (x0, pick0, state, tail) in zip(models, got, want):
            assert torch.equal(x, x0) and torch.equal(pick, pick0) and torch.equal(M.state, state) and torch.equal(M.tail, tail)
    for d, M, st in zip(devices, models, streams):
        assert d.sync_status(st.cuda_stream) == OK
        for c in M.cache:
            c.free()
        d.close()


@pytest.mark.gpu
def test_two_graphs_share_a_contexts_scratch(dev):  # noqa: F811
    """Captured one after the other, the second growing the scratch; replayed in turn, with eager passes between."""
    d, kinds = chart.Device(0), ([3, 40, 1], [500, 300, 64])
    models = [Model(d, p) for p in kinds]
    passes = [prompt_pass(M, p) for M, p in zip(models, kinds)]
    want, graphs, outs = [], [], []
    for M, go in zip(models, passes):
        x, pick = go()
        torch.cuda.synchronize()
        want.append((x.clone(), pick.clone(), M.state.clone()))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(go())
        graphs.append(graph)
    for turn in range(4):
        for M, graph, out, (x, pick, state), go in zip(models, graphs, outs, want, passes):
            out[0].zero_(), out[1].zero_(), M.state[1:].zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], x) and torch.equal(out[1], pick) and torch.equal(M.state, state), turn
            if turn == 2:
                go()
    assert d.sync_status(stream()) == OK
    for M in models:
        for c in M.cache:
            c.free()
    d.close()
