"""Attention of chunks where the caller's arrays are out of range, for every kernel that serves chunks: even and uneven
sequences, pieces joined in the launch (heads of 64) and by another (128, 256), chunks beside single tokens."""
import numpy as np
import pytest

from test_attention_accuracy import bound
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

    def exact(self, s, hidden=()):
        """f64 attention of sequence s, its pages `hidden` not seen, and its largest score in powers of two."""
        n, c, page, kv = self.qs[s], int(self.ctx[s]), self.P.cache.page_len, self.P.cache.n_kv_heads
        q = self.q[self.start[s]:self.start[s + 1]].reshape(n, self.heads, self.dim).astype(np.float64)
        key = np.arange(c)
        see = (key <= (c - n + np.arange(n))[:, None]) & ~np.isin(key // page, hidden)
        out, S = np.zeros(q.shape), 0.0
        for h in range(self.heads):
            g = h * kv // self.heads
            x = np.where(see, q[:, h] @ self.k[s][:c, g].astype(np.float64).T * self.dim ** -0.5, -np.inf)
            top = x.max(-1, keepdims=True)
            p = np.exp(x - np.where(np.isfinite(top), top, 0))
            S, den = max(S, np.abs(x[see]).max() * np.log2(np.e)), p.sum(-1, keepdims=True)
            out[:, h] = p @ self.v[s][:c, g].astype(np.float64) / np.where(den > 0, den, 1)
        return out.reshape(n, -1), S

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


MIXED = ([1] * 20 + [300, 0] + [1] * 20 + [150], [130 + 9 * i for i in range(20)] + [901, 40] + [77 + 9 * i for i in range(20)] + [150])
SIZES = pytest.mark.parametrize("qs,ctx", [EVEN, UNEVEN, MIXED], ids=["even", "uneven", "mixed"])


@pytest.mark.parametrize("dim,G", [(64, 7), (128, 4), (256, 2)])
@SIZES
def test_contexts_and_lengths_out_of_range(dev, dim, G, qs, ctx):  # noqa: F811
    C = Call(dev, dim, G, qs, ctx, page=32)
    st, good = C()
    assert st == OK
    longest = int(np.argmax(qs))
    for s in sorted({0, longest, len(qs) - 1}):
        for value in (-1, -2 ** 31, C.P.per * 32 + 1, 2 ** 31 - 1):
            c = C.ctx.copy()
            c[s] = value
            st, o = C(ctx=c)
            kept = ~C.rows(s)
            assert st == CACHE and np.array_equal(o[kept], good[kept]) and (o[~kept] == 7).all(), (s, value)
    # a sequence that is longer than max_q (its neighbour gives it a token)
    if longest + 1 < len(qs) and qs[longest + 1]:
        start = C.start.copy()
        start[longest + 1] += 1
        st, o = C(start=start)
        kept = ~C.rows(longest, longest + 1)
        assert st == CACHE and np.array_equal(o[kept], good[kept]) and (o[start[longest]:start[longest + 1]] == 7).all()
    # no keys: zeros, and nothing is refused
    c = C.ctx.copy()
    c[longest] = 0
    st, o = C(ctx=c)
    assert st == OK and (o[C.rows(longest)] == 0).all() and np.array_equal(o[~C.rows(longest)], good[~C.rows(longest)])


@pytest.mark.parametrize("dim,G", [(64, 7), (128, 4), (256, 2)])
@SIZES
def test_pages_out_of_range_are_not_seen(dev, dim, G, qs, ctx):  # noqa: F811
    """Pages of one tile: the first and the second of a pair of tiles, neighbours, the last one, and all of a row's."""
    C = Call(dev, dim, G, qs, ctx, page=32)
    st, good = C()
    assert st == OK
    n_pages = C.P.cache.n_pages
    for s in sorted({int(np.argmax(qs)), len(qs) - 1}):
        last = (ctx[s] - 1) // 32
        for hidden in sorted({(0,), (1,), (0, 1), (last,), (last - 1,), tuple(range(last // 2))}):
            hidden = [p for p in hidden if 0 <= p <= last]
            if not hidden or len(hidden) == last + 1:
                continue
            table = C.P.table.clone()
            for i, p in enumerate(hidden):
                table[s, p] = (-1, n_pages, 2 ** 31 - 1, -2 ** 31)[i % 4]
            st, o = C(table=table)
            kept = ~C.rows(s)
            ref, S = C.exact(s, hidden)
            err = np.linalg.norm(o[~kept] - ref) / np.linalg.norm(ref)
            assert st == CACHE and np.array_equal(o[kept], good[kept]), (s, hidden)
            assert err <= bound(S, ctx[s]) and (o[~kept][(ref == 0).all(-1)] == 0).all(), (s, hidden, err)


@pytest.mark.parametrize("dim,G", [(64, 7), (128, 4), (256, 2)])
@SIZES
def test_rows_that_are_not_finite_stay_alone(dev, dim, G, qs, ctx):  # noqa: F811
    C = Call(dev, dim, G, qs, ctx, page=64)
    st, good = C()
    at = [(int(C.start[int(np.argmax(qs))]) + 3, 1), (len(C.q) - 1, 0)]
    for bad in (np.nan, np.inf):
        q = C.q.copy()
        for tok, head in at:
            q[tok, head * dim + 5] = bad
        st, o = C(q=q)
        assert st == OK
        o, whole = o.reshape(len(q), -1, dim), good.reshape(len(q), -1, dim)
        touched = np.zeros(o.shape[:2], bool)
        for tok, head in at:
            touched[tok, head] = True
        assert np.isnan(o[touched]).all() and np.array_equal(o[~touched], whole[~touched])


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
