"""Attention that reads a part of the 4-bit cache, or reads it once for many: behind a batch's common prefix, and over the
blocks whose means a query scores highest.

Outputs are compared with 64-bit attention over the cache's values, with the tolerance of attention over the whole cache
(tests/test_gpu_token_ops.py: the halves of q, f32's scores, weights and sums).  Means are f64 sums that are exact, so
they have one value; the chosen blocks are compared exactly.
"""
import ctypes

import numpy as np
import pytest

from apeiron_amd import _lib, chart
from test_gpu_token_ops import CACHE, INVALID, OK, Paged, U, cuda, dev, filled, ptr, quantize4, stream  # noqa: F401

torch = pytest.importorskip("torch")


def compare(got, q, k, v, see, scale):
    """One sequence's rows got, q [n][heads][dim] against f64 attention over k, v [c][kv][dim] where see [n][kv][c]."""
    n, heads, dim = q.shape
    c, kv = k.shape[:2]
    for h in range(heads):
        K, V, m, x = k[:, h * kv // heads].astype(np.float64), v[:, h * kv // heads].astype(np.float64), see[:, h * kv // heads], q[:, h].astype(np.float64)
        sc = np.where(m, x @ K.T * scale, -np.inf)
        top = sc.max(-1, keepdims=True, initial=-np.inf)
        p = np.exp(sc - np.where(np.isfinite(top), top, 0))
        den = p.sum(-1, keepdims=True)
        safe = np.where(den > 0, den, 1)
        ref, mag = p @ V / safe, p @ np.abs(V) / safe
        size = abs(scale) * np.where(m, np.abs(x) @ np.abs(K).T, 0).max(-1, keepdims=True, initial=0)
        wide = abs(scale) * np.abs(x).max(-1, keepdims=True) * np.where(m, np.abs(K).sum(-1)[None], 0).max(-1, keepdims=True, initial=0)
        rel = 2 * (2.0 ** -21 * wide + (2 * dim + 4) * U * size) + 2.0 ** -18 + 2 * (c + 64) * U
        err = np.abs(got[:, h] - ref)
        assert (err <= rel * mag).all(), (h, err.max(), (err / np.maximum(rel * mag, 1e-30)).max())


class Batch:
    """Sequences in a cache, their queries and the arrays of a call."""

    def __init__(self, d, qs, ctx, kv, G, dim, page, prefix=0, seed=0, spread=1.0, pad=0):
        rng = np.random.default_rng(seed)
        self.d, self.qs, self.ctxs, self.kv, self.heads, self.dim, self.prefix = d, qs, ctx, kv, kv * G, dim, prefix
        self.P = Paged(d, len(ctx), max(max(ctx), 1), page, kv, dim, seed=seed)
        common = (rng.standard_normal((2, prefix, kv, dim)) * spread).astype(np.float32)
        self.k, self.v = [], []
        for s, c in enumerate(ctx):
            k, v = (rng.standard_normal((2, c, kv, dim)) * spread).astype(np.float32)
            k[:prefix], v[:prefix] = common[0][:c], common[1][:c]
            if c:
                self.P.append(np.full(c, s), np.arange(c), k, v)
            self.k.append(quantize4(k) if c else k)
            self.v.append(quantize4(v) if c else v)
        self.width = self.heads * dim + pad
        self.start = np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)
        self.q = rng.standard_normal((sum(qs), self.width)).astype(np.float32)
        self.scale = dim ** -0.5

    def arrays(self, **change):
        i32 = lambda x: cuda(np.asarray(x, np.int32))  # noqa: E731
        self.keep = i32(change.pop("start", self.start)), i32(change.pop("ctx", self.ctxs)), change.pop("table", self.P.table), cuda(change.pop("q", self.q))
        out = torch.full((len(self.q), self.width), 7.0, device="cuda")
        st = change.pop("stream", None) or stream()
        args = dict(n_heads=self.heads, n_tok=len(self.q), n_seq=len(self.qs), q_start_ptr=ptr(self.keep[0]), ctx_ptr=ptr(self.keep[1]), table_ptr=ptr(self.keep[2]),
                    table_stride=self.P.per, max_q=max(self.qs), max_ctx=max(self.ctxs), scale=self.scale, q_stride=self.width, out_stride=self.width, stream=st)
        return out, args | change

    def plain(self, **change):
        out, args = self.arrays(**change)
        self.P.cache.attn_dev(ptr(self.keep[3]), ptr(out), **args)
        return self.d.sync_status(args["stream"]), out.cpu().numpy()

    def rows(self, s, x):
        return x[self.start[s]:self.start[s + 1], : self.heads * self.dim].reshape(self.qs[s], self.heads, self.dim)

    def positions(self, s):
        return self.ctxs[s] - self.qs[s] + np.arange(self.qs[s])

    # behind the prefix
    def shared(self, prefix_table=None, prefix=None, **change):
        out, args = self.arrays(**change)
        prefix = self.prefix if prefix is None else prefix
        table = self.P.table[0, : -(-prefix // self.P.cache.page_len)].clone() if prefix_table is None else prefix_table
        self.P.cache.attn_shared_dev(ptr(self.keep[3]), ptr(out), prefix_len=prefix, prefix_table_ptr=ptr(table), **args)
        return self.d.sync_status(args["stream"]), out.cpu().numpy()

    # over blocks
    def means(self, block, seq=None, pos=None, out=None):
        c = self.P.cache
        if out is None:
            out = torch.full((c.n_pages, c.page_len // block, self.kv, self.dim), 3.0, dtype=torch.float16, device="cuda")
        seq = np.repeat(np.arange(len(self.ctxs)), self.ctxs) if seq is None else seq
        pos = np.concatenate([np.arange(n) for n in self.ctxs]) if pos is None else pos
        c.block_means_dev(ptr(out), block_len=block, stream=stream(), **self.P.where(seq, pos))
        return out

    def blocks(self, means, block, top, first, last, **change):
        out, args = self.arrays(**change)
        chosen = torch.full((len(self.q), self.kv, top), -7, dtype=torch.int32, device="cuda")
        self.P.cache.attn_blocks_dev(ptr(self.keep[3]), ptr(out), means_ptr=ptr(means), block_len=block, n_top=top, n_first=first, n_last=last,
                                     chosen_ptr=ptr(chosen), **args)
        return self.d.sync_status(args["stream"]), out.cpu().numpy(), chosen.cpu().numpy()

    def choose(self, s, block, top, first, last):
        """The blocks chosen by score [n][kv][top] (-1 behind them) and what the queries see [n][kv][ctx], by the definition."""
        n, c, pos = self.qs[s], self.ctxs[s], self.positions(s)
        chosen, see = np.full((n, self.kv, top), -1, np.int32), np.zeros((n, self.kv, c), bool)
        mean = self.k[s][: c // block * block].astype(np.float64).reshape(-1, block, self.kv, self.dim).mean(1).astype(np.float32).astype(np.float16).astype(np.float64)
        q = self.rows(s, self.q).astype(np.float64).reshape(n, self.kv, -1, self.dim).sum(2)
        for t in range(n):
            own = pos[t] // block
            middle = np.arange(first, max(first, own - last)) if pos[t] >= 0 else np.zeros(0, int)
            for h in range(self.kv):
                score = self.scale * (mean[middle, h] @ q[t, h])
                pick = np.sort(middle[np.argsort(-np.where(np.isnan(score), -np.inf, score), kind="stable")[:top]])
                chosen[t, h, : len(pick)] = pick
                read = set(pick) | set(range(min(first, own + 1))) | set(range(max(0, own - last), own + 1))
                see[t, h] = np.isin(np.arange(c) // block, list(read)) & (np.arange(c) <= pos[t])
        return chosen, see


# ---- behind a common prefix ---------------------------------------------------------------------------


SHARED = [  # (tokens, contexts, prefix, page)
    ([1, 1, 1], [70, 65, 100], 64, 32), ([1] * 9, [301 + 7 * i for i in range(9)], 300, 64), ([1], [40], 39, 64), ([1, 1], [2, 2], 1, 32),
    ([1] * 40, [1001 + i for i in range(40)], 1000, 128), ([5, 0, 33, 1, 17], [140, 129, 200, 130, 146], 129, 32),
    ([200, 1, 64], [700, 301, 364], 300, 64), ([300, 150], [4300, 4000], 1025, 64), ([20] * 12, [90] * 12, 70, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,G,pad", [(64, 2, 7, 0), (128, 2, 6, 4), (256, 1, 3, 0), (64, 1, 1, 1), (128, 1, 19, 0)])
@pytest.mark.parametrize("call", range(len(SHARED)))
def test_shared_prefix_matches_f64(dev, dim, kv, G, pad, call):  # noqa: F811
    qs, ctx, prefix, page = SHARED[call]
    B = Batch(dev, qs, ctx, kv, G, dim, page, prefix=prefix, seed=dim + call, pad=pad)
    table = B.P.table.clone()
    first = table[0, : -(-prefix // page)].clone()
    table[:, : prefix // page] = 1 << 30  # the sequences' own entries before the prefix's end are not read
    status, out = B.shared(prefix_table=first, table=table)
    assert status == OK and (out[:, B.heads * dim:] == 7).all()
    for s in range(len(qs)):
        if qs[s]:
            see = np.arange(ctx[s]) <= B.positions(s)[:, None, None]
            compare(B.rows(s, out), B.rows(s, B.q), B.k[s], B.v[s], np.broadcast_to(see, (qs[s], kv, ctx[s])), B.scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,G", [(64, 7), (128, 4), (256, 2)])
def test_shared_prefix_of_large_scores_and_longer_contexts_than_planned(dev, dim, G):  # noqa: F811
    ctx = [900, 1500, 701, 2600]
    B = Batch(dev, [1, 3, 1, 90], ctx, 2, G, dim, 64, prefix=640, seed=dim, spread=4.0)
    for change in ({}, {"max_ctx": 1}, {"max_ctx": 700}, {"max_ctx": 10 ** 9}):
        status, out = B.shared(**change)
        assert status == OK
        for s in range(4):
            see = np.arange(ctx[s]) <= B.positions(s)[:, None, None]
            compare(B.rows(s, out), B.rows(s, B.q), B.k[s], B.v[s], np.broadcast_to(see, (B.qs[s], 2, ctx[s])), B.scale)


MANY = [  # (head_dim, KV heads, queries of each, tokens, what follows the prefix of each sequence, prefix)
    (64, 1, 7, [50, 1, 0, 128, 64], [60, 1, 5, 128, 200], 133), (128, 1, 6, [90, 100, 70], [90, 100, 300], 640), (256, 2, 3, [300, 220], [333, 250], 31),
    (64, 4, 16, [32, 31, 1, 0, 20] * 5, [32, 31, 1, 3, 90] * 5, 100), (128, 4, 16, [32] * 24, [32 + i % 3 for i in range(24)], 65),
    (256, 8, 16, [16, 3, 16, 1] * 6, [16, 20, 70, 1] * 6, 64), (64, 64, 10, [16, 2, 13, 1, 16], [16, 2, 40, 1, 17], 40), (64, 32, 1, [1] * 110, [1 + i % 9 for i in range(110)], 33),
    (128, 2, 16, [17] * 9 + [1], [20] * 9 + [300], 2000), (128, 1, 6, [90, 1, 100, 60], [90, 1, 300, 64], 5700)]


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,G,qs,after,prefix", MANY)
def test_shared_prefix_of_many_rows(dev, dim, kv, G, qs, after, prefix):  # noqa: F811
    """More than 1536 rows of a KV head behind the prefix, and sequences of many rows."""
    ctx = [prefix + n for n in after]
    B = Batch(dev, qs, ctx, kv, G, dim, 32, prefix=prefix, seed=dim, pad=3)
    status, out = B.shared()
    assert status == OK and (out[:, B.heads * dim:] == 7).all()
    for s in range(len(qs)):
        if qs[s]:
            see = np.arange(ctx[s]) <= B.positions(s)[:, None, None]
            compare(B.rows(s, out), B.rows(s, B.q), B.k[s], B.v[s], np.broadcast_to(see, (qs[s], kv, ctx[s])), B.scale)
    good = out
    for value in (-1, prefix + qs[0] - 1, 10 ** 6):  # the first out of range: the others as before
        status, out = B.shared(ctx=[value] + ctx[1:])
        assert status == CACHE and (out[: qs[0]] == 7).all() and np.array_equal(out[qs[0]:], good[qs[0]:])
    start = B.start.copy()
    start[1] = sum(qs) + 1
    status, out = B.shared(start=start)
    assert status == CACHE and (out[: qs[0] + qs[1]] == 7).all() and np.array_equal(out[qs[0] + qs[1]:], good[qs[0] + qs[1]:])
    B.q = np.concatenate([B.q, np.full((40, B.width), np.nan, np.float32)])  # rows of no sequence
    status, out = B.shared()
    assert status == OK and (out[-40:] == 7).all() and np.isfinite(out).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,G,pad", [(64, 2, 7, 0), (128, 2, 6, 4), (64, 1, 1, 1), (128, 1, 19, 0), (128, 4, 2, 2)])
@pytest.mark.parametrize("qs,after,prefix", [([1, 1, 1], [6, 1, 36], 4097), ([1] * 9, [1 + 7 * i for i in range(9)], 4128), ([5, 0, 33, 1, 17], [11, 2, 71, 1, 17], 5000), ([1] * 40, [1 + i for i in range(40)], 4100)])
def test_a_long_shared_prefix(dev, dim, kv, G, pad, qs, after, prefix):  # noqa: F811
    """Past the lengths that a sequence reads for itself."""
    ctx = [prefix + n for n in after]
    B = Batch(dev, qs, ctx, kv, G, dim, 64, prefix=prefix, seed=dim, pad=pad)
    table = B.P.table.clone()
    first = table[0, : -(-prefix // 64)].clone()
    table[:, : prefix // 64] = 1 << 30  # the sequences' own entries before the prefix's end are not read
    status, out = B.shared(prefix_table=first, table=table)
    assert status == OK and (out[:, B.heads * dim:] == 7).all()
    for s in range(len(qs)):
        if qs[s]:
            see = np.arange(ctx[s]) <= B.positions(s)[:, None, None]
            compare(B.rows(s, out), B.rows(s, B.q), B.k[s], B.v[s], np.broadcast_to(see, (qs[s], kv, ctx[s])), B.scale)
    # a page of the prefix out of range: its positions are not seen; a context inside the prefix: passed over
    good, first[3] = out, -1
    status, out = B.shared(prefix_table=first, table=table)
    assert status == CACHE
    for s in range(len(qs)):
        if qs[s]:
            see = (np.arange(ctx[s]) <= B.positions(s)[:, None, None]) & (np.arange(ctx[s]) // 64 != 3)
            compare(B.rows(s, out), B.rows(s, B.q), B.k[s], B.v[s], np.broadcast_to(see, (qs[s], kv, ctx[s])), B.scale)
    first[3] = B.P.table[0, 3]
    status, out = B.shared(prefix_table=first, table=table, ctx=[prefix + qs[0] - 1] + ctx[1:])
    assert status == CACHE and (out[: qs[0]] == 7).all() and np.array_equal(out[qs[0]:], good[qs[0]:])


@pytest.mark.gpu
def test_shared_prefix_of_none_is_the_plain_call(dev):  # noqa: F811
    B = Batch(dev, [1, 40], [300, 500], 2, 4, 64, 32, seed=1)
    assert np.array_equal(B.shared(prefix=0)[1], B.plain()[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dim,G,qs,ctx", [(64, 7, [1, 1, 1, 1], [900, 700, 650, 800]), (128, 4, [200, 90, 131, 1], [900, 750, 1500, 700]), (256, 2, [200] * 4, [900, 850, 1300, 870])])
def test_shared_prefix_values_out_of_range(dev, dim, G, qs, ctx):  # noqa: F811
    B = Batch(dev, qs, ctx, 2, G, dim, 64, prefix=640, seed=dim)
    status, good = B.shared()
    assert status == OK
    n, n_tok = len(qs), sum(qs)
    rows = lambda *seqs: np.isin(np.repeat(np.arange(n), qs), seqs)  # noqa: E731
    for at in range(n + 1):
        for value in (-1, -2 ** 31, n_tok + 1, 2 ** 31 - 1):
            start = B.start.copy()
            start[at] = value
            status, out = B.shared(start=start)
            kept = rows(*[s for s in range(n) if s != at and s + 1 != at])
            assert status == CACHE and np.array_equal(out[kept], good[kept]) and (out[~kept] == 7).all(), (at, value)
    for s in range(n):  # a context out of range, or one whose tokens begin inside the prefix
        for value in (-1, 10 ** 6, 639, 640 + qs[s] - 1):
            c = np.array(ctx)
            c[s] = value
            status, out = B.shared(ctx=c)
            assert status == CACHE and np.array_equal(out[~rows(s)], good[~rows(s)]) and (out[rows(s)] == 7).all(), (s, value)
    # a page of the prefix out of range: its positions are not seen, by any sequence
    table = B.P.table[0, :10].clone()
    table[3] = -1
    status, out = B.shared(prefix_table=table)
    assert status == CACHE
    for s in range(n):
        key = np.arange(ctx[s])
        see = (key <= B.positions(s)[:, None, None]) & (key // 64 != 3)
        compare(B.rows(s, out), B.rows(s, B.q), B.k[s], B.v[s], np.broadcast_to(see, (qs[s], 2, ctx[s])), B.scale)
    assert B.shared()[0] == OK


@pytest.mark.gpu
def test_rows_of_no_sequence_hold_anything(dev):  # noqa: F811
    """Tokens behind the last sequence's are not written, and what stands in their queries reaches no other row."""
    for qs, ctx in (([1, 1, 1, 0], [700, 650, 800, 0]), ([70, 30, 90, 0], [750, 700, 900, 0])):
        B = Batch(dev, qs, ctx, 2, 3, 64, 32, prefix=610, seed=2)
        B.q = np.concatenate([B.q, np.full((5, B.width), np.nan, np.float32)])
        B.ctxs[3] = 610
        status, out = B.shared()
        assert status == OK and (out[-5:] == 7).all() and np.isfinite(out).all()
        means = B.means(32)
        status, out, chosen = B.blocks(means, 32, 4, 1, 1)
        assert status == OK and (out[-5:] == 7).all() and np.isfinite(out).all() and (chosen[-5:] == -7).all()


# ---- over blocks --------------------------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,page,block", [(64, 1, 32, 32), (64, 3, 128, 64), (128, 2, 64, 64), (128, 5, 1024, 256), (256, 2, 128, 32), (256, 1, 64, 64)])
def test_means_are_the_blocks(dev, dim, kv, page, block):  # noqa: F811
    ctx = [2 * page + block - 1, block, 3 * page, 1]
    B = Batch(dev, [1] * 4, ctx, kv, 1, dim, page, seed=dim + kv, spread=1e3)
    got = B.means(block)
    table, left = B.P.table.cpu().numpy(), np.ones(got.shape[:2], bool)
    for s, c in enumerate(ctx):
        for b in range(c // block):
            want = B.k[s][b * block: (b + 1) * block].astype(np.float64).mean(0).astype(np.float32).astype(np.float16)
            at = table[s, b * block // page], b * block % page // block
            assert np.array_equal(got[at].cpu().numpy(), want), (s, b)
            left[at] = False
    assert (got.cpu().numpy()[left] == 3).all()  # blocks without their last position, and pages of no one
    # one token at a time: only the one that ends a block changes it
    again = torch.full_like(got, 3.0)
    for p in range(block + 1):
        B.means(block, [2], [p], out=again)
    assert torch.equal(again[table[2, 0], 0], got[table[2, 0], 0])
    again[table[2, 0], 0] = 3
    assert (again == 3).all()
    assert dev.sync_status(stream()) == OK
    # padding tokens are passed over; a sequence, position or page out of range is refused, and the others served
    for seq, pos, table_value in ((4, 0, None), (2, 3 * page, None), (2, -1, None), (2, block - 1, 10 ** 6)):
        fresh, kept = torch.full_like(got, 3.0), B.P.table.clone()
        if table_value is not None:
            B.P.table[2, 0] = table_value
        B.means(block, [-1, seq, 1], [-5, pos, block - 1], out=fresh)
        assert dev.sync_status(stream()) == CACHE
        B.P.table.copy_(kept)
        assert torch.equal(fresh[table[1, 0], 0], got[table[1, 0], 0])
        fresh[table[1, 0], 0] = 3
        assert (fresh == 3).all()


BLOCKS = [  # (tokens, contexts, page, block, top, first, last)
    ([1, 1, 1, 1, 1], [1, 32, 33, 700, 0], 32, 32, 4, 0, 0), ([1] * 6, [900, 64, 65, 1400, 31, 257], 64, 64, 3, 1, 1), ([1], [5000], 128, 32, 16, 2, 3),
    ([70, 33, 0, 1, 5, 150], [70, 300, 50, 200, 3, 150], 32, 32, 2, 1, 0), ([300], [2100], 128, 64, 8, 0, 2), ([40, 40], [1000, 1000], 64, 32, 1, 0, 0),
    ([1, 2], [3000, 3100], 1024, 512, 2, 1, 0), ([3], [900], 32, 32, 64, 0, 0), ([1, 1], [9000, 100], 32, 32, 100, 7, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,G,pad", [(64, 2, 7, 0), (128, 2, 6, 4), (256, 1, 3, 0), (64, 3, 1, 1), (128, 1, 19, 0)])
@pytest.mark.parametrize("call", range(len(BLOCKS)))
def test_blocks_are_chosen_and_attended(dev, dim, kv, G, pad, call):  # noqa: F811
    qs, ctx, page, block, top, first, last = BLOCKS[call]
    B = Batch(dev, qs, ctx, kv, G, dim, page, seed=dim + call, pad=pad)
    for sign in (1, -1):
        B.scale = sign * dim ** -0.5
        status, out, chosen = B.blocks(B.means(block), block, top, first, last)
        assert status == OK and (out[:, B.heads * dim:] == 7).all()
        for s in range(len(qs)):
            if qs[s]:
                want, see = B.choose(s, block, top, first, last)
                assert np.array_equal(chosen[B.start[s]:B.start[s + 1]], want)
                compare(B.rows(s, out), B.rows(s, B.q), B.k[s], B.v[s], see, B.scale)


@pytest.mark.gpu
def test_blocks_that_hold_everything_are_the_whole_context(dev):  # noqa: F811
    B = Batch(dev, [1, 50, 3], [700, 333, 64], 2, 4, 128, 64, seed=5)
    status, out, chosen = B.blocks(B.means(64), 64, 32, 0, 0)
    assert status == OK
    for s in range(3):
        see = np.arange(B.ctxs[s]) <= B.positions(s)[:, None, None]
        compare(B.rows(s, out), B.rows(s, B.q), B.k[s], B.v[s], np.broadcast_to(see, (B.qs[s], 2, B.ctxs[s])), B.scale)
        own = B.positions(s) // 64
        assert np.array_equal(chosen[B.start[s]:B.start[s + 1], 0], np.where(np.arange(32) < own[:, None], np.arange(32), -1))


MANY_TOKENS = [  # (head_dim, KV heads, queries of each, tokens, contexts, page, block, top, first, last)
    (64, 2, 7, [1, 300, 5, 0, 40], [800, 900, 5, 40, 1200], 64, 32, 5, 1, 1), (128, 2, 6, [520], [1531], 64, 64, 4, 0, 2), (128, 8, 1, [4] * 20, [1000 + 7 * i for i in range(20)], 128, 128, 2, 1, 0),
    (128, 2, 3, [70, 250], [3000, 260], 32, 32, 30, 2, 3), (256, 4, 2, [100, 1, 17, 200], [100, 700, 900, 1100], 64, 32, 6, 0, 0), (64, 3, 9, [200, 201], [700, 800], 32, 32, 65, 1, 0),
    (64, 2, 8, [2, 600], [2000, 640], 1024, 64, 3, 1, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,G,qs,ctx,page,block,top,first,last", MANY_TOKENS)
def test_blocks_of_many_tokens(dev, dim, kv, G, qs, ctx, page, block, top, first, last):  # noqa: F811
    """Two (token, KV head)s a CU and more, four and more: 16 tokens' choice together, a wave a list."""
    B = Batch(dev, qs, ctx, kv, G, dim, page, seed=dim + kv, pad=4)
    means = B.means(block)
    status, out, chosen = B.blocks(means, block, top, first, last)
    assert status == OK and (out[:, B.heads * dim:] == 7).all()
    for s in range(len(qs)):
        if qs[s]:
            want, see = B.choose(s, block, top, first, last)
            assert np.array_equal(chosen[B.start[s]:B.start[s + 1]], want)
            compare(B.rows(s, out), B.rows(s, B.q), B.k[s], B.v[s], see, B.scale)
    good, picked, edge = out, chosen, qs[0]
    for value in (-1, 10 ** 6):  # the first out of range: the others as before
        status, out, chosen = B.blocks(means, block, top, first, last, ctx=[value] + ctx[1:])
        assert status == CACHE and (out[:edge] == 7).all() and np.array_equal(out[edge:], good[edge:]) and np.array_equal(chosen[edge:], picked[edge:])
    B.q = np.concatenate([B.q, np.full((40, B.width), np.nan, np.float32)])  # rows of no sequence
    status, out, chosen = B.blocks(means, block, top, first, last)
    assert status == OK and (out[-40:] == 7).all() and (chosen[-40:] == -7).all() and np.array_equal(out[:-40], good) and np.array_equal(chosen[:-40], picked)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,G,qs,ctx", [(128, 6, [40], [3]), (256, 3, [1, 70, 5], [0, 2, 40]), (64, 7, [300, 40], [20, 0]), (128, 4, [600], [130]), (64, 8, [520, 30], [3, 100]),
                                          (256, 2, [520], [1]), (128, 9, [520], [260])])
def test_blocks_of_more_tokens_than_positions(dev, dim, G, qs, ctx):  # noqa: F811
    """Tokens before position 0 see nothing and choose nothing."""
    B = Batch(dev, qs, ctx, 2, G, dim, 64, seed=dim)
    status, out, chosen = B.blocks(B.means(32), 32, 2, 1, 0)
    assert status == OK
    for s in range(len(qs)):
        want, see = B.choose(s, 32, 2, 1, 0)
        assert np.array_equal(chosen[B.start[s]:B.start[s + 1]], want) and (B.rows(s, out)[B.positions(s) < 0] == 0).all()
        if ctx[s]:
            compare(B.rows(s, out), B.rows(s, B.q), B.k[s], B.v[s], see, B.scale)


@pytest.mark.gpu
@pytest.mark.parametrize("blocks,top", [(20, 5), (300, 64), (1500, 16), (1500, 1000)])
def test_equal_scores_take_the_first_blocks(dev, blocks, top):  # noqa: F811
    """Means of small whole numbers, so that sums are exact and many scores equal."""
    rng = np.random.default_rng(blocks)
    B = Batch(dev, [1, 1], [32 * blocks + 7, 32 * blocks], 1, 2, 64, 32, seed=blocks)
    B.q = rng.integers(-2, 3, B.q.shape).astype(np.float32)
    B.q[1] = 0  # all equal
    per = -(-B.ctxs[0] // 32)
    means = torch.zeros(B.P.cache.n_pages, 1, 1, 64, dtype=torch.float16, device="cuda")
    value = rng.integers(-1, 2, (2, per, 64)).astype(np.float16)
    value[0, 3::7] = value[0, 3]
    for s in range(2):
        means[B.P.table[s].long()[:per], 0, 0] = cuda(value[s])
    status, out, chosen = B.blocks(means, 32, top, 0, 0)
    assert status == OK
    for s in range(2):
        own = (B.ctxs[s] - 1) // 32
        score = value[s, :own].astype(np.float64) @ B.q[s].reshape(2, 64).astype(np.float64).sum(0)
        assert np.array_equal(chosen[s, 0], np.sort(np.argsort(-score, kind="stable")[:top]))


@pytest.mark.gpu
def test_blocks_of_a_context_past_the_scores_that_lds_holds(dev):  # noqa: F811
    n = 17000  # blocks
    cache = chart.KvCache4(dev, n, 32, 1, 64)
    rng = np.random.default_rng(3)
    table = torch.arange(n, dtype=torch.int32, device="cuda")[None].contiguous()
    k = torch.randn(n * 32, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    seq, pos = torch.zeros(n * 32, dtype=torch.int32, device="cuda"), torch.arange(n * 32, dtype=torch.int32, device="cuda")
    tokens = dict(seq_ptr=ptr(seq), pos_ptr=ptr(pos), n_tok=n * 32, table_ptr=ptr(table), n_seq=1, table_stride=n, stream=stream())
    cache.append_dev(None, k_ptr=ptr(k), v_ptr=ptr(k), **tokens)
    means = torch.zeros(n, 1, 1, 64, dtype=torch.float16, device="cuda")
    cache.block_means_dev(ptr(means), block_len=32, **tokens)
    for ctx in (n * 32, n * 32 - 40):
        q, out = cuda(rng.standard_normal((1, 64)).astype(np.float32)), torch.zeros(1, 64, device="cuda")
        start, c, chosen = cuda(np.array([0, 1], np.int32)), cuda(np.array([ctx], np.int32)), torch.zeros(1, 1, 8, dtype=torch.int32, device="cuda")
        cache.attn_blocks_dev(ptr(q), ptr(out), means_ptr=ptr(means), block_len=32, n_top=8, n_first=1, n_last=2, n_heads=1, n_tok=1, n_seq=1, q_start_ptr=ptr(start),
                              ctx_ptr=ptr(c), table_ptr=ptr(table), table_stride=n, max_q=1, max_ctx=ctx, scale=0.125, chosen_ptr=ptr(chosen), stream=stream())
        assert dev.sync_status(stream()) == OK
        own = (ctx - 1) // 32
        score = means[1:own - 2, 0, 0].double().cpu().numpy() @ q[0].double().cpu().numpy()
        want = 1 + np.sort(np.argsort(-score, kind="stable")[:8])
        assert np.array_equal(chosen[0, 0].cpu().numpy(), want)
        key = np.concatenate([np.arange(b * 32, min(ctx, b * 32 + 32)) for b in [0, *want, own - 2, own - 1, own]])
        K = quantize4(k.cpu().numpy()[key])[:, None]
        compare(out.cpu().numpy()[:, None], q.cpu().numpy()[:, None], K, K, np.ones((1, 1, len(key)), bool), 0.125)


@pytest.mark.gpu
@pytest.mark.parametrize("qs,ctx", [([1, 1, 1, 1], [900, 700, 650, 800]), ([70, 90, 31, 1], [900, 750, 1500, 700])])
def test_blocks_values_out_of_range(dev, qs, ctx):  # noqa: F811
    B = Batch(dev, qs, ctx, 2, 3, 64, 64, seed=7)
    means = B.means(32)
    status, good, picked = B.blocks(means, 32, 4, 1, 1)
    assert status == OK
    n, n_tok = len(qs), sum(qs)
    rows = lambda *seqs: np.isin(np.repeat(np.arange(n), qs), seqs)  # noqa: E731
    for at in range(n + 1):
        for value in (-1, -2 ** 31, n_tok + 1, 2 ** 31 - 1):
            start = B.start.copy()
            start[at] = value
            status, out, chosen = B.blocks(means, 32, 4, 1, 1, start=start)
            kept = rows(*[s for s in range(n) if s != at and s + 1 != at])
            assert status == CACHE and np.array_equal(out[kept], good[kept]) and (out[~kept] == 7).all(), (at, value)
            assert np.array_equal(chosen[kept], picked[kept]) and (chosen[~kept] == -7).all()
    for s, value in ((0, -1), (1, 10 ** 6), (n - 1, -2 ** 31)):
        c = np.array(ctx)
        c[s] = value
        status, out, chosen = B.blocks(means, 32, 4, 1, 1, ctx=c)
        assert status == CACHE and np.array_equal(out[~rows(s)], good[~rows(s)]) and (out[rows(s)] == 7).all(), (s, value)
    # a page out of range: its blocks score lowest, and where one is read all the same its positions are not seen
    table = B.P.table.clone()
    table[0, 0] = -9
    status, out, chosen = B.blocks(means, 32, 4, 1, 1, table=table)
    assert status == CACHE and np.array_equal(out[~rows(0)], good[~rows(0)])
    first = slice(0, qs[0])
    score_free = B.choose(0, 32, 4, 2, 1)  # blocks 0 and 1 are out: as if the first two were read anyway
    assert np.array_equal(chosen[first], score_free[0])
    compare(B.rows(0, out), B.rows(0, B.q), B.k[0], B.v[0], score_free[1] & (np.arange(ctx[0]) >= 64), B.scale)
    # NaN in a query or a mean: the lowest score, and nobody else's
    q = B.q.copy()
    q[0, 5] = np.nan
    status, out, chosen = B.blocks(means, 32, 4, 1, 1, q=q)
    assert np.array_equal(out[1:], good[1:]) and np.array_equal(chosen[1:], picked[1:]) and np.array_equal(chosen[0, 1], picked[0, 1])
    assert np.array_equal(chosen[0, 0], np.arange(1, 5))
    m = means.clone()
    m[int(B.P.table[0, 2]), 0, 0, 3] = np.nan  # block 4 of sequence 0
    status, out, chosen = B.blocks(m, 32, 4, 1, 1)
    assert status == OK and not (chosen[first, 0] == 4).any() and np.array_equal(chosen[first, 1], picked[first, 1])
    assert B.blocks(means, 32, 4, 1, 1)[0] == OK


@pytest.mark.gpu
def test_part_attention_is_the_same_each_time_and_on_any_stream(dev):  # noqa: F811
    for qs, ctx in (([1, 1, 1], [5000, 4100, 4500]), ([200, 1, 70], [4900, 4100, 4500])):
        B = Batch(dev, qs, ctx, 2, 6, 128, 64, prefix=4099, seed=8)
        means = B.means(64)
        want = B.shared()[1], *B.blocks(means, 64, 8, 1, 1)[1:]
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        for st in (None, side.cuda_stream, None):
            got = B.shared(stream=st)[1], *B.blocks(means, 64, 8, 1, 1, stream=st)[1:]
            assert all(np.array_equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dim,G,qs,ctx", [(64, 7, [1, 1, 1], [1900, 1570, 2600]), (128, 6, [90, 1, 33], [2000, 1700, 1600]), (256, 4, [64], [1700])])
def test_part_attention_replayed_as_a_graph(dev, dim, G, qs, ctx):  # noqa: F811
    """Append, the means of the blocks that its tokens end, attention over blocks and behind the prefix, in a graph: every
    replay, with eager work of the same context that outgrows its scratch between, leaves what the eager calls leave."""
    d = chart.Device(0)
    B = Batch(d, qs, ctx, 2, G, dim, 64, prefix=1500, seed=dim)
    large = Batch(d, [500, 300], [3000, 2900], 2, G, dim, 64, prefix=2000, seed=1)
    n, cache = sum(qs), B.P.cache
    rng = np.random.default_rng(0)
    k, v = (cuda(rng.standard_normal((n, 2 * dim)).astype(np.float32)) for _ in range(2))
    seq, pos = cuda(np.repeat(np.arange(len(qs)), qs).astype(np.int32)), cuda(np.concatenate([B.positions(s) for s in range(len(qs))]).astype(np.int32))
    means, prefix = B.means(32), B.P.table[0, :24].clone()
    out, args = B.arrays()
    out2, chosen = torch.zeros_like(out), torch.zeros(n, 2, 6, dtype=torch.int32, device="cuda")
    arrays = B.keep

    def run():
        a = args | {"stream": stream()}
        tokens = dict(seq_ptr=ptr(seq), pos_ptr=ptr(pos), n_tok=n, table_ptr=ptr(B.P.table), n_seq=len(qs), table_stride=B.P.per, stream=stream())
        cache.append_dev(None, k_ptr=ptr(k), v_ptr=ptr(v), **tokens)
        cache.block_means_dev(ptr(means), block_len=32, **tokens)
        cache.attn_blocks_dev(ptr(arrays[3]), ptr(out), means_ptr=ptr(means), block_len=32, n_top=6, n_first=1, n_last=1, chosen_ptr=ptr(chosen), **a)
        cache.attn_shared_dev(ptr(arrays[3]), ptr(out2), prefix_len=1500, prefix_table_ptr=ptr(prefix), **a)

    run()
    torch.cuda.synchronize()
    want = [t.clone() for t in (out, out2, chosen, means)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    big_means = large.means(32)
    for i in range(4):
        for t in (out, out2, chosen):
            t.zero_()
        k.mul_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((out, out2, chosen, means), want)), i
        large.shared()
        large.blocks(big_means, 32, 12, 1, 1)
        large.plain()
    assert d.sync_status(stream()) == OK
    d.close()


@pytest.mark.gpu
def test_blocks_of_a_cache_past_4_gib(dev):  # noqa: F811
    kv, dim, page = 8, 256, 32
    n_pages = (5 << 30) // (36 * dim * kv)
    B = Batch.__new__(Batch)
    B.d, B.qs, B.ctxs, B.kv, B.heads, B.dim, B.width, B.scale, B.prefix = dev, [1], [160], kv, 2 * kv, dim, 2 * kv * dim, dim ** -0.5, 40
    B.P = Paged.__new__(Paged)
    B.P.cache, B.P.n_seq, B.P.per = chart.KvCache4(dev, n_pages, page, kv, dim), 1, 5
    B.P.table = cuda(n_pages - 1 - 2 * np.arange(5, dtype=np.int32)[None])
    rng = np.random.default_rng(5)
    k, v = rng.standard_normal((2, 160, kv, dim)).astype(np.float32)
    B.P.append(np.zeros(160), np.arange(160), k, v)
    B.k, B.v, B.start, B.q = [quantize4(k)], [quantize4(v)], np.array([0, 1], np.int32), rng.standard_normal((1, B.width)).astype(np.float32)
    status, out, chosen = B.blocks(B.means(32), 32, 2, 0, 0)
    want, see = B.choose(0, 32, 2, 0, 0)
    assert status == OK and np.array_equal(chosen, want)
    compare(B.rows(0, out), B.rows(0, B.q), B.k[0], B.v[0], see, B.scale)
    status, out = B.shared()
    assert status == OK
    compare(B.rows(0, out), B.rows(0, B.q), B.k[0], B.v[0], np.ones((1, kv, 160), bool), B.scale)


@pytest.mark.gpu
def test_part_attention_refusals(dev):  # noqa: F811
    B = Batch(dev, [1], [64], 1, 1, 64, 64, seed=1)
    L, z, cache = dev.lib, torch.zeros(512, device="cuda"), B.P.cache
    half = torch.zeros(cache.n_pages * 64 * 2 + 8, dtype=torch.float16, device="cuda")
    i = cuda(np.array([0, 1, 64, 0], np.int32))

    def attn(**kw):
        return _lib.Kv4Attn(*(kw.get(n, v) for n, v in (("n_seq", 1), ("n_tok", 1), ("n_heads", 1), ("max_q", 1), ("max_ctx", 64), ("start", ptr(i)), ("ctx", ptr(i) + 8),
                                                        ("table", ptr(B.P.table)), ("stride", 1), ("scale", 1.0), ("window", 0), ("sinks", 0))))

    def shared(prefix=32, table=ptr(B.P.table), q=ptr(z), qs=64, out=ptr(z) + 1024, os=64, **kw):
        return L.ah_kv4_attn_shared_dev(dev.h, cache.h, ctypes.byref(attn(**kw)), prefix, table, q, qs, out, os, stream())

    def blocks(q=ptr(z), qs=64, out=ptr(z) + 1024, os=64, len=32, top=1, first=0, last=0, means=ptr(half), **kw):  # noqa: A002
        return L.ah_kv4_attn_blocks_dev(dev.h, cache.h, ctypes.byref(attn(**kw)), ctypes.byref(_lib.Kv4Blocks(len, top, first, last, means)), q, qs, out, os, None,
                                        stream())

    assert shared() == OK and blocks() == OK
    both = (dict(window=1), dict(sinks=1), dict(start=None), dict(ctx=None), dict(table=None), dict(n_seq=65536), dict(n_tok=1 << 31), dict(n_heads=65537), dict(stride=0),
            dict(q=None), dict(out=None), dict(qs=63), dict(os=63), dict(out=ptr(z)), dict(out=ptr(z) + 128))
    for bad in (*both, dict(prefix=1 << 31), dict(n_tok=1 << 24, n_heads=64, qs=4096, os=4096)):
        assert shared(**bad) == INVALID, bad
    for bad in (*both, dict(len=16), dict(len=48), dict(len=128), dict(len=0), dict(top=0), dict(top=4097), dict(first=4097), dict(last=4097), dict(means=None),
                dict(means=ptr(half) + 2)):
        assert blocks(**bad) == INVALID, bad
    for empty in (dict(n_seq=0), dict(n_tok=0), dict(n_heads=0), dict(max_q=0)):
        assert shared(**empty) == OK and blocks(**empty) == OK
    t = _lib.Kv4Tokens(ptr(i), ptr(i), 1, ptr(B.P.table), 1, 1)
    assert L.ah_kv4_block_means_dev(dev.h, cache.h, ctypes.byref(t), 32, ptr(half), stream()) == OK
    for n, p in ((16, ptr(half)), (128, ptr(half)), (48, ptr(half)), (32, None), (32, ptr(half) + 2)):
        assert L.ah_kv4_block_means_dev(dev.h, cache.h, ctypes.byref(t), n, p, stream()) == INVALID
    assert dev.sync_status(stream()) == OK


def test_null_arguments_are_refused_without_a_gpu():
    L = _lib.load()
    a, t, b = _lib.Kv4Attn(), _lib.Kv4Tokens(), _lib.Kv4Blocks()
    assert L.ah_kv4_attn_shared_dev(None, None, ctypes.byref(a), 1, None, None, 0, None, 0, None) == INVALID
    assert L.ah_kv4_block_means_dev(None, None, ctypes.byref(t), 32, None, None) == INVALID
    assert L.ah_kv4_attn_blocks_dev(None, None, ctypes.byref(a), ctypes.byref(b), None, 0, None, 0, None, None) == INVALID
    assert ctypes.sizeof(_lib.Kv4Blocks) == 5 * 8
