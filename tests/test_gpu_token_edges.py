"""Attention of chunks where the caller's arrays are out of range, for every kernel that serves chunks: even and uneven
sequences, pieces joined in the launch (heads of 64) and by another (128, 256), chunks beside single tokens."""
import numpy as np
import pytest

from test_gpu_token_ops import CACHE, INVALID, OK, cuda, dev, filled, ptr, stream  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


class Call:
    """A call over a filled cache whose arrays can be changed; the pieces follow from the host's arguments alone, so
    what a change leaves in range comes out bit for bit as before."""

    def __init__(self, dev, dim, G, qs, ctx, kv=2, page=64):  # noqa: F811
        self.dev, self.dim, self.heads, self.qs = dev, dim, kv * G, qs
        self.P, self.k, self.v = filled(dev, ctx, page, kv, dim, seed=dim + len(qs))
        self.start, self.ctx = np.concatenate([[0], np.cumsum(qs)]).astype(np.int32), np.asarray(ctx, np.int32)
        rng = np.random.default_rng(G)
        self.q = rng.standard_normal((sum(qs), self.heads * dim)).astype(np.float32)

    def __call__(self, start=None, ctx=None, table=None, q=None):
        dq, ds = cuda(self.q if q is None else q), cuda(np.asarray(self.start if start is None else start, np.int32))
        dc, table = cuda(np.asarray(self.ctx if ctx is None else ctx, np.int32)), self.P.table if table is None else table
        out = torch.full_like(dq, 7.0)
        self.P.cache.attn_dev(ptr(dq), ptr(out), n_heads=self.heads, n_tok=len(self.q), n_seq=len(self.qs), q_start_ptr=ptr(ds), ctx_ptr=ptr(dc),
                              table_ptr=ptr(table), table_stride=self.P.per, max_q=max(self.qs), max_ctx=int(self.ctx.max()), scale=self.dim ** -0.5,
                              stream=stream())
        return self.dev.sync_status(stream()), out.cpu().numpy()

    def rows(self, *seqs):
        """The tokens of these sequences, as a mask."""
        m = np.zeros(len(self.q), bool)
        for s in seqs:
            m[self.start[s]:self.start[s + 1]] = True
        return m


# (tokens and contexts of the sequences): even ones, uneven ones, more than a wave has lanes
EVEN, UNEVEN = ([200] * 4, [900, 200, 513, 700]), ([200, 90, 131, 260, 1], [900, 90, 1500, 700, 30])
MANY = ([70 + i % 3 for i in range(150)], [80 + 7 * (i % 40) for i in range(150)])


@pytest.mark.parametrize("dim,G", [(64, 7), (128, 4), (256, 2)])
@pytest.mark.parametrize("qs,ctx", [EVEN, UNEVEN, MANY], ids=["even", "uneven", "many"])
def test_a_start_out_of_range_leaves_the_other_sequences(dev, dim, G, qs, ctx):  # noqa: F811
    C = Call(dev, dim, G, qs, ctx)
    st, good = C()
    assert st == OK and not (good == 7).all(-1).any()
    n, n_tok = len(qs), len(C.q)
    for at in sorted({0, 1, 2, n // 2, n - 1, n}):  # an entry ends one sequence and starts the next
        for value in (-1, -2 ** 31, n_tok + 1, 2 ** 31 - 1):
            start = C.start.copy()
            start[at] = value
            st, o = C(start=start)
            kept = C.rows(*[s for s in range(n) if s != at and s + 1 != at])
            assert st == CACHE, (at, value)
            assert np.array_equal(o[kept], good[kept]) and (o[~kept] == 7).all(), (at, value)
    # several at once
    start = C.start.copy()
    start[[0, n - 2, n - 1]] = [-5, n_tok + 9, -1]
    st, o = C(start=start)
    kept = C.rows(*range(1, n - 3))
    assert st == CACHE and np.array_equal(o[kept], good[kept]) and (o[~kept] == 7).all()


def test_more_tokens_than_a_launch_holds_are_refused(dev):  # noqa: F811
    """A workgroup a token, fewer than 2^32 threads a launch: refused on the host, nothing is read."""
    from apeiron_amd import _lib, chart

    L, h, x = dev.lib, dev.h, torch.zeros(64, device="cuda")
    p = ptr(x)
    # (values of a token, its threads)
    for n, threads in ((32, 64), (1024, 128), (2048, 256), (4096, 512), (4097, 1024), (32768, 1024)):
        assert L.ah_norm_quant_dev(h, p, None, p, 1e-6, (1 << 32) // threads, n, None, p, None, None, None, None) == INVALID, n
    rope, cache = chart.Rope(dev, 128), chart.KvCache4(dev, 2, 32, 8, 128)
    assert L.ah_rope_dev(h, rope.h, p, 16 * 128, 16, p, 1 << 24, p, 16 * 128, None) == INVALID
    assert L.ah_rope_dev(h, rope.h, p, 128, 1, p, 1 << 26, p, 128, None) == INVALID
    t = _lib.Kv4Tokens(p, p, 1 << 24, p, 1, 1)
    assert L.ah_kv4_append_dev(h, cache.h, None, t, None, 0, 0, None, 0, p, 1024, p, 1024, None) == INVALID
    assert L.ah_kv4_append_dev(h, cache.h, rope.h, t, p, 2048, 16, p, 2048, p, 1024, p, 1024, None) == INVALID
    assert L.ah_kv4_read_dev(h, cache.h, t, p, p, None) == INVALID
    small = chart.KvCache4(dev, 2, 32, 1, 64)  # a wave a token
    t = _lib.Kv4Tokens(p, p, 1 << 26, p, 1, 1)
    assert L.ah_kv4_append_dev(h, small.h, None, t, None, 0, 0, None, 0, p, 64, p, 64, None) == INVALID
    assert dev.sync_status(stream()) == OK
