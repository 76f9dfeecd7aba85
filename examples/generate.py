"""Token generation with everything between the embedding and the drawn token on the device: a random-weight
decoder of the Qwen2.5 architecture (no biases), prompts of uneven lengths prefilled in one batch, then one
token a step for every sequence, the step replayed as one HIP graph.

A layer is
    norm_quant (residual + RMS norm + QuantAct) -> q/k/v -> KvCache4.append (rotary positions, k and v into the
    4-bit cache) -> KvCache4.attn -> o -> norm_quant -> the fused FFN
and a step ends with norm_quant -> the head -> sample.  Run it as

    python examples/generate.py [--layers 4] [--prompts 3] [--tokens 32]
"""
from __future__ import annotations

import argparse
import os
import sys
import time
from dataclasses import dataclass

import numpy as np
import torch

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from apeiron_amd import chart, synth


@dataclass
class Config:
    """The 0.5B-class widths; vocabulary and layers smaller by default."""
    hidden: int = 896
    heads: int = 14
    kv_heads: int = 2
    head_dim: int = 64
    ffn: int = 4864
    layers: int = 4
    vocab: int = 32000
    eps: float = 1e-6
    base: float = 1e6
    page: int = 64
    window: int = 0
    sinks: int = 0
    ggml_type: int = synth.Q8_0


class Model:
    def __init__(self, cfg: Config, max_seqs: int, max_len: int, seed: int = 0, device: int = 0):
        self.cfg, self.dev = cfg, chart.Device(device)
        rng = np.random.default_rng(seed)
        c, kv = cfg, cfg.kv_heads * cfg.head_dim
        shapes = {"q": (c.heads * c.head_dim, c.hidden), "k": (kv, c.hidden), "v": (kv, c.hidden), "o": (c.hidden, c.heads * c.head_dim),
                  "gate": (c.ffn, c.hidden), "up": (c.ffn, c.hidden), "down": (c.hidden, c.ffn)}
        self.raw = [{n: synth.payload(c.ggml_type, rng, *s) for n, s in shapes.items()} for _ in range(c.layers)]
        self.raw_head = synth.payload(c.ggml_type, rng, c.vocab, c.hidden)
        self.w = [{n: self.dev.upload(c.ggml_type, raw[n], *shapes[n]) for n in shapes} for raw in self.raw]
        self.head = self.dev.upload(c.ggml_type, self.raw_head, c.vocab, c.hidden)

        def gain():
            return torch.from_numpy((1 + 0.1 * rng.standard_normal(c.hidden)).astype(np.float32)).cuda()
        self.norm1, self.norm2, self.norm = [gain() for _ in range(c.layers)], [gain() for _ in range(c.layers)], gain()
        self.embedding = torch.from_numpy(rng.standard_normal((c.vocab, c.hidden)).astype(np.float32)).cuda()
        self.rope = chart.Rope(self.dev, c.head_dim, base=c.base)
        per = -(-max_len // c.page)
        self.max_len = per * c.page
        self.caches = [chart.KvCache4(self.dev, max_seqs * per, c.page, c.kv_heads, c.head_dim) for _ in range(c.layers)]
        # every sequence owns its pages here; a server would hand them out as sequences grow
        self.table = torch.from_numpy(rng.permutation(max_seqs * per).reshape(max_seqs, per).astype(np.int32)).cuda()

    def close(self) -> None:
        """Frees what the model holds on the device."""
        for t in [t for layer in self.w for t in layer.values()] + [self.head, self.rope, *self.caches]:
            t.free()
        self.dev.close()


class Step:
    """One forward pass of n_tok tokens of n_seq sequences over buffers of its own (so that it can be captured).
    Inputs to fill before a run: tokens, seq, pos, q_start, ctx and u; output: drawn (and logits, probs)."""

    def __init__(self, model: Model, n_tok: int, n_seq: int, max_q: int, max_ctx: int, temperature: float = 0.8, top_k: int = 40,
                 top_p: float = 0.95):
        self.m, self.n_tok, self.n_seq, self.max_q, self.max_ctx = model, n_tok, n_seq, max_q, max_ctx
        c = model.cfg

        def f32(*shape):
            return torch.zeros(*shape, device="cuda")

        def i32(*shape):
            return torch.zeros(*shape, dtype=torch.int32, device="cuda")
        self.tokens, self.seq, self.pos, self.q_start, self.ctx = i32(n_tok), i32(n_tok), i32(n_tok), i32(n_seq + 1), i32(n_seq)
        self.u, self.drawn, self.probs, self.logits = f32(n_seq), i32(n_seq), f32(n_seq), f32(n_seq, c.vocab)
        self.x, self.res = f32(n_tok, c.hidden), f32(n_tok, c.hidden)
        self.q, self.att = f32(n_tok, c.heads * c.head_dim), f32(n_tok, c.heads * c.head_dim)
        self.k, self.v = f32(n_tok, c.kv_heads * c.head_dim), f32(n_tok, c.kv_heads * c.head_dim)
        self.act = torch.zeros(n_tok, c.hidden, dtype=torch.int8, device="cuda"), torch.zeros(n_tok, -(-c.hidden // 32), dtype=torch.int64, device="cuda")
        self.hid = torch.zeros(n_tok, c.ffn, dtype=torch.int8, device="cuda"), torch.zeros(n_tok, -(-c.ffn // 32), dtype=torch.int64, device="cuda")
        self.last_act = self.act if n_tok == n_seq else (torch.zeros(n_seq, c.hidden, dtype=torch.int8, device="cuda"),
                                                         torch.zeros(n_seq, -(-c.hidden // 32), dtype=torch.int64, device="cuda"))
        self.t, self.top_k, self.top_p = f32(n_seq) + temperature, i32(n_seq) + top_k, f32(n_seq) + top_p

    def _project(self, ws, act, ys, n, stream):
        if n == 1:
            for w, y in zip(ws, ys):
                w.gemv_q8_dev(act[0].data_ptr(), act[1].data_ptr(), y.data_ptr(), stream)
        else:
            chart.gemm_group_q8_dev(self.m.dev, ws, act[0].data_ptr(), act[1].data_ptr(), n, [y.data_ptr() for y in ys], stream)

    def run(self) -> None:
        m, c, n, dev = self.m, self.m.cfg, self.n_tok, self.m.dev
        stream = torch.cuda.current_stream().cuda_stream
        where = dict(seq_ptr=self.seq.data_ptr(), pos_ptr=self.pos.data_ptr(), n_tok=n, table_ptr=m.table.data_ptr(), n_seq=self.n_seq,
                     table_stride=m.table.shape[1], stream=stream)
        act = dict(codes_ptr=self.act[0].data_ptr(), scales_ptr=self.act[1].data_ptr(), stream=stream)
        torch.index_select(m.embedding, 0, self.tokens, out=self.res)
        x = None  # what the residual takes next
        for w, g1, g2, cache in zip(m.w, m.norm1, m.norm2, m.caches):
            self._norm(x, g1, act)
            self._project([w["q"], w["k"], w["v"]], self.act, [self.q, self.k, self.v], n, stream)
            cache.append_dev(m.rope, q_ptr=self.q.data_ptr(), n_heads=c.heads, q_out_ptr=self.q.data_ptr(), k_ptr=self.k.data_ptr(),
                             v_ptr=self.v.data_ptr(), **where)
            cache.attn_dev(self.q.data_ptr(), self.att.data_ptr(), n_heads=c.heads, n_tok=n, n_seq=self.n_seq, q_start_ptr=self.q_start.data_ptr(),
                           ctx_ptr=self.ctx.data_ptr(), table_ptr=m.table.data_ptr(), table_stride=m.table.shape[1], max_q=self.max_q,
                           max_ctx=self.max_ctx, scale=c.head_dim ** -0.5, window=c.window, sinks=c.sinks, stream=stream)
            if n == 1:
                w["o"].gemv_f32_dev(self.att.data_ptr(), self.x.data_ptr(), stream)
            else:
                w["o"].gemm_f32_dev(self.att.data_ptr(), n, self.x.data_ptr(), stream)
            self._norm(self.x, g2, act)
            x = self.x
            ffn = (dev, w["gate"], w["up"], w["down"], self.act[0].data_ptr(), self.act[1].data_ptr())
            out = (self.x.data_ptr(), self.hid[0].data_ptr(), self.hid[1].data_ptr(), stream)
            chart.ffn_q8_dev(*ffn, *out) if n == 1 else chart.ffn_prefill_q8_dev(*ffn, n, *out)
        self._norm(x, m.norm, act)
        if self.last_act is not self.act:  # only each sequence's last token goes to the head
            last = self.q_start[1:] - 1
            for a, b in zip(self.act, self.last_act):
                torch.index_select(a, 0, last, out=b)
        self._project([m.head], self.last_act, [self.logits], self.n_seq, stream)
        chart.sample_dev(dev, self.logits.data_ptr(), self.n_seq, c.vocab, self.u.data_ptr(), self.drawn.data_ptr(), probs_ptr=self.probs.data_ptr(),
                         temperature_ptr=self.t.data_ptr(), top_k_ptr=self.top_k.data_ptr(), top_p_ptr=self.top_p.data_ptr(), stream=stream)

    def _norm(self, x, gain, act):
        """res += x (the first time only the embedding is there), and the norm's QuantAct."""
        first = x is None
        chart.norm_quant_dev(self.m.dev, self.res.data_ptr() if first else x.data_ptr(), gain.data_ptr(), self.m.cfg.eps, self.n_tok,
                             self.m.cfg.hidden, residual_ptr=None if first else self.res.data_ptr(),
                             sum_ptr=None if first else self.res.data_ptr(), **act)


def prefill(model: Model, prompts: list[list[int]], u, **sampling) -> Step:
    """Runs the prompts as one ragged batch; the step holds each sequence's first drawn token."""
    lens = [len(p) for p in prompts]
    step = Step(model, sum(lens), len(prompts), max(lens), max(lens), **sampling)
    step.tokens.copy_(torch.tensor([t for p in prompts for t in p], dtype=torch.int32))
    step.seq.copy_(torch.repeat_interleave(torch.arange(len(prompts), dtype=torch.int32), torch.tensor(lens)))
    step.pos.copy_(torch.tensor([i for n in lens for i in range(n)], dtype=torch.int32))
    step.q_start.copy_(torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32))
    step.ctx.copy_(torch.tensor(lens, dtype=torch.int32))
    step.u.copy_(torch.as_tensor(u, dtype=torch.float32))
    step.run()
    return step


class Decoder:
    """One token a sequence and call, from the prefill's drawn tokens on; with graph=True the step is captured once
    (after an eager one, which grows the scratch) and replayed."""

    def __init__(self, model: Model, first: Step, graph: bool = True, **sampling):
        n = first.n_seq
        self.step = s = Step(model, n, n, 1, model.max_len, **sampling)
        s.seq.copy_(torch.arange(n, dtype=torch.int32))
        s.q_start.copy_(torch.arange(n + 1, dtype=torch.int32))
        s.pos.copy_(first.ctx)
        s.ctx.copy_(first.ctx + 1)
        s.drawn.copy_(first.drawn)
        self.model, self.use_graph, self.graph, self.calls = model, graph, None, 0

    def _body(self):
        s = self.step
        s.tokens.copy_(s.drawn)
        s.run()
        s.pos.add_(1)
        s.ctx.add_(1)

    def __call__(self, u) -> torch.Tensor:
        self.step.u.copy_(torch.as_tensor(u, dtype=torch.float32))
        if self.use_graph and self.calls == 1:
            torch.cuda.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph, stream=torch.cuda.Stream()):
                self._body()
        if self.graph is not None:
            self.graph.replay()
        else:
            self._body()
        self.calls += 1
        return self.step.drawn


def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--prompts", type=int, default=3)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    rng = np.random.default_rng(a.seed)
    prompts = [rng.integers(0, Config.vocab, size=rng.integers(5, 200)).tolist() for _ in range(a.prompts)]
    model = Model(Config(layers=a.layers), a.prompts, 256 + a.tokens, seed=a.seed)
    first = prefill(model, prompts, rng.random(a.prompts))
    out = [first.drawn.tolist()]
    decode = Decoder(model, first)
    for i in range(a.tokens - 1):
        if i == 2:
            torch.cuda.synchronize()
            t0 = time.perf_counter()
        out.append(decode(rng.random(a.prompts)).tolist())
    torch.cuda.synchronize()
    if a.tokens > 3:
        print(f"{(time.perf_counter() - t0) / (a.tokens - 3) * 1e6:.0f} us a step of {a.prompts} sequences, {a.layers} layers")
    status = model.dev.sync_status(torch.cuda.current_stream().cuda_stream)
    assert status == 0, f"device status {status}"
    for p, toks in zip(prompts, zip(*out)):
        print(f"prompt of {len(p)}: {' '.join(map(str, toks[:12]))} ..")
    model.close()


if __name__ == "__main__":
    main()
