"""The generation example as a whole: every operator in its place, against a token-by-token model in 64 bits over
the CPU oracle's projections.

Tolerance: the device's f32 steps differ from the reference's 64 bits by about 1e-6, which moves an int8 code across
a rounding boundary (one step is at most 1/64 of its block's largest value, 1/64 / sqrt(hidden) ~ 1e-3 of an
output) in about one of 1e4 elements, and a 4-bit code as rarely (a quarter of its block's largest value in one of
a key's channels).  A few such moves stay under 2e-2 of the logits' size; a token at a wrong position, head, page
or mask is of their size.
"""
import importlib.util
import os
import sys

import numpy as np
import pytest

import oracle

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def gen():
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    spec = importlib.util.spec_from_file_location("generate", os.path.join(ROOT, "examples", "generate.py"))
    m = importlib.util.module_from_spec(spec)
    sys.modules["generate"] = m
    spec.loader.exec_module(m)
    return m


def quantize4(x):
    b = x.reshape(*x.shape[:-1], -1, 32).astype(np.float32)
    hi, lo = b.max(-1, keepdims=True), b.min(-1, keepdims=True)
    d = (np.where(hi >= -lo, hi, lo) * np.float32(-0.125)).astype(np.float32)
    e = np.maximum(np.frexp(d)[1] - 8, -24)
    d = np.ldexp(np.rint(np.ldexp(d, -e)), e)
    c = np.clip(np.rint((b / np.where(d == 0, np.float32(1), d)).astype(np.float32)), -8, 7) * (d != 0)
    return (c * d).astype(np.float64).reshape(x.shape)


class Reference:
    """One sequence, token by token."""

    def __init__(self, model):
        self.m, self.c = model, model.cfg
        self.k, self.v = [[] for _ in range(self.c.layers)], [[] for _ in range(self.c.layers)]
        self.gains = [[g.cpu().numpy().astype(np.float64) for g in gs] for gs in (model.norm1, model.norm2, [model.norm])]
        self.embedding = model.embedding.cpu().numpy()

    def product(self, raw, n_out, x):
        st, codes, scales = oracle.quant_act_f32(x.astype(np.float32))
        assert st == 0
        st, y = oracle.matvec_q8act(self.c.ggml_type, raw, n_out, len(x), codes, scales)
        assert st == 0
        return y.astype(np.float64) * 2.0 ** -32

    def norm(self, x, g):
        return x / np.sqrt((x * x).mean() + self.c.eps) * g

    def rotate(self, x, pos):
        d = self.c.head_dim
        a = pos * self.c.base ** (-np.arange(0, d, 2) / d)
        p, q = x[:, : d // 2], x[:, d // 2:]
        return np.concatenate([p * np.cos(a) - q * np.sin(a), q * np.cos(a) + p * np.sin(a)], 1)

    def __call__(self, token, pos):
        c, x = self.c, self.embedding[token].astype(np.float64)
        kv, G = c.kv_heads * c.head_dim, c.heads // c.kv_heads
        for i, raw in enumerate(self.m.raw):
            h = self.norm(x, self.gains[0][i])
            q = self.rotate(self.product(raw["q"], c.heads * c.head_dim, h).reshape(-1, c.head_dim), pos)
            self.k[i].append(quantize4(self.rotate(self.product(raw["k"], kv, h).reshape(-1, c.head_dim), pos)))
            self.v[i].append(quantize4(self.product(raw["v"], kv, h).reshape(-1, c.head_dim)))
            K, V, att = np.array(self.k[i]), np.array(self.v[i]), []
            see = np.arange(pos + 1) <= pos
            if c.window:
                see &= (np.arange(pos + 1) > pos - c.window) | (np.arange(pos + 1) < c.sinks)
            for n in range(c.heads):
                s = np.where(see, K[:, n // G] @ q[n] / np.sqrt(c.head_dim), -np.inf)
                p = np.exp(s - s.max())
                att.append(p @ V[:, n // G] / p.sum())
            x = x + self.product(raw["o"], c.hidden, np.concatenate(att))
            h = self.norm(x, self.gains[1][i])
            gate, up = self.product(raw["gate"], c.ffn, h), self.product(raw["up"], c.ffn, h)
            x = x + self.product(raw["down"], c.hidden, gate / (1 + np.exp(-gate)) * up)
        return self.product(self.m.raw_head, c.vocab, self.norm(x, self.gains[2][0]))


@pytest.mark.parametrize("heads,kv,dim,window,sinks,lens", [(4, 2, 64, 0, 0, [37, 5]), (3, 1, 128, 20, 3, [41]), (2, 1, 256, 0, 0, [9, 30, 2])])
def test_generation_matches_the_reference(gen, heads, kv, dim, window, sinks, lens):
    cfg = gen.Config(hidden=heads * dim, heads=heads, kv_heads=kv, head_dim=dim, ffn=320, layers=2, vocab=600, page=32, window=window, sinks=sinks)
    model = gen.Model(cfg, len(lens), 64, seed=dim)
    rng = np.random.default_rng(dim)
    prompts = [rng.integers(0, cfg.vocab, size=n).tolist() for n in lens]
    first = gen.prefill(model, prompts, rng.random(len(lens)), top_k=5)
    refs = [Reference(model) for _ in lens]
    for s, p in enumerate(prompts):
        for i, t in enumerate(p):
            want = refs[s](t, i)
        got = first.logits[s].cpu().numpy()
        assert np.linalg.norm(got - want) <= 2e-2 * np.linalg.norm(want), (s, np.linalg.norm(got - want) / np.linalg.norm(want))
    decode = gen.Decoder(model, first, graph=True, top_k=5)
    tokens = first.drawn.tolist()
    for step in range(4):  # eager, then captured, then replayed
        drawn = decode(rng.random(len(lens))).tolist()
        logits = decode.step.logits.cpu().numpy()
        for s, n in enumerate(lens):
            want = refs[s](tokens[s], n + step)
            assert np.linalg.norm(logits[s] - want) <= 2e-2 * np.linalg.norm(want), (step, s)
            order = np.argsort(-logits[s])[:5]
            assert drawn[s] in order
        tokens = drawn
    assert model.dev.sync_status(torch.cuda.current_stream().cuda_stream) == 0
    model.close()


def test_replays_equal_the_eager_steps(gen):
    """The same prompts and random numbers, eager and captured: the same tokens and logits, bit for bit, over many
    replays with eager work and synchronizations between them."""
    cfg = gen.Config(layers=2, vocab=5000)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, cfg.vocab, size=n).tolist() for n in (150, 33, 7)]
    us = rng.random((13, 3))
    runs = []
    model = gen.Model(cfg, 3, 256, seed=3)
    for graph in (False, True):
        first = gen.prefill(model, prompts, us[0])
        decode = gen.Decoder(model, first, graph=graph)
        got = [first.drawn.tolist()]
        for i in range(12):
            got.append((decode(us[i + 1]).tolist(), decode.step.logits.cpu()))
            x = torch.randn(512, 512, device="cuda")
            (x @ x).sum().item()
        runs.append(got)
    assert runs[0][0] == runs[1][0]
    for a, b in zip(runs[0][1:], runs[1][1:]):
        assert a[0] == b[0] and torch.equal(a[1], b[1])
    model.close()
