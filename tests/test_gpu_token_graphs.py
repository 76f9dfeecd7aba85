"""Graphs of captured calls replayed after calls of the same context that need more scratch than they did."""
import ctypes

import numpy as np
import pytest

from apeiron_amd import chart, synth
from test_gpu_token_ops import OK, cuda, filled, ptr, stream

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def scratch(d):
    n = ctypes.c_size_t(0)
    assert d.lib.ah_ctx_scratch_bytes(d.h, ctypes.byref(n)) == OK
    return n.value


class Work:
    """Attention in pieces, sampling, a GEMM and an FFN of one size, over buffers of their own."""

    def __init__(self, d, qs, ctx, rows, V, n_tok):
        rng = np.random.default_rng(len(qs) + rows)
        f32 = lambda *s: cuda(rng.standard_normal(s).astype(np.float32))  # noqa: E731
        self.d, self.qs, self.max_ctx, self.rows, self.V, self.n_tok = d, qs, max(ctx), rows, V, n_tok
        self.P, _, _ = filled(d, ctx, 64, 2, 64, seed=rows)
        self.q = f32(sum(qs), 14 * 64)
        self.start, self.ctx = cuda(np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)), cuda(np.asarray(ctx, np.int32))
        self.logits, self.u = f32(rows, V), cuda(rng.random(rows).astype(np.float32))
        self.p = cuda(np.full(rows, 0.9, np.float32))
        up = lambda o, i: d.upload(synth.Q8_0, synth.payload(synth.Q8_0, rng, o, i), o, i)  # noqa: E731
        self.w, self.gate, self.up, self.down = up(192, 512), up(640, 512), up(640, 512), up(512, 640)
        self.x = f32(n_tok, 512)
        self.codes = torch.zeros(n_tok, 512, dtype=torch.int8, device="cuda"), torch.zeros(n_tok, 16, dtype=torch.int64, device="cuda")
        chart.norm_quant_dev(d, ptr(self.x), ptr(f32(512)), 1e-6, n_tok, 512, codes_ptr=ptr(self.codes[0]), scales_ptr=ptr(self.codes[1]), stream=stream())
        self.hid = torch.zeros(n_tok, 640, dtype=torch.int8, device="cuda"), torch.zeros(n_tok, 20, dtype=torch.int64, device="cuda")
        self.out = [torch.zeros_like(self.q), torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(n_tok, 192, device="cuda"),
                    torch.zeros(n_tok, 512, device="cuda")]

    def run(self):
        st, P = stream(), self.P
        P.cache.attn_dev(ptr(self.q), ptr(self.out[0]), n_heads=14, n_tok=sum(self.qs), n_seq=len(self.qs), q_start_ptr=ptr(self.start), ctx_ptr=ptr(self.ctx),
                         table_ptr=ptr(P.table), table_stride=P.per, max_q=max(self.qs), max_ctx=self.max_ctx, scale=0.125, stream=st)
        chart.sample_dev(self.d, ptr(self.logits), self.rows, self.V, ptr(self.u), ptr(self.out[1]), top_p_ptr=ptr(self.p), stream=st)
        self.w.gemm_f32_dev(ptr(self.x), self.n_tok, ptr(self.out[2]), st)
        chart.ffn_prefill_q8_dev(self.d, self.gate, self.up, self.down, ptr(self.codes[0]), ptr(self.codes[1]), self.n_tok, ptr(self.out[3]), ptr(self.hid[0]),
                                 ptr(self.hid[1]), st)


def test_replays_after_larger_calls(dev_pair):
    plain, d = dev_pair
    sizes = dict(qs=[1] * 8, ctx=[4001, 3000, 65, 1, 900, 2000, 4001, 77], rows=8, V=7001, n_tok=48), dict(qs=[1500, 40], ctx=[2500, 3000], rows=300, V=20000, n_tok=700)
    for s in sizes:  # eager alone: what is outgrown is freed
        Work(plain, **s).run()
    torch.cuda.synchronize()
    alone = scratch(plain)
    small, large = (Work(d, **s) for s in sizes)
    small.run()
    torch.cuda.synchronize()
    first, want = scratch(d), [t.clone() for t in small.out]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        small.run()
    assert scratch(d) == first
    large.run()
    torch.cuda.synchronize()
    # the captured calls' scratch is still held beside the larger one, before anything is replayed
    assert scratch(d) == first + alone
    again = [t.clone() for t in large.out]
    others = [torch.full((first // 4,), float("nan"), device="cuda") for _ in range(4)]  # what would take freed memory's place
    for i in range(4):
        for t in small.out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(small.out, want)), i
        large.run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(large.out, again)), i
    assert all(torch.isnan(t).all() for t in others) and scratch(d) == first + alone
    assert d.sync_status(stream()) == OK


@pytest.fixture
def dev_pair():
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    a, b = chart.Device(0), chart.Device(0)
    yield a, b
    a.close()
    b.close()
