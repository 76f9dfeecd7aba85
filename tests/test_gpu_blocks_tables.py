"""Attention over blocks where the page tables are wider than the contexts (a server's are as wide as the longest context
allowed) and where the contexts are longer than the call planned for."""
import ctypes

import numpy as np
import pytest

from apeiron_amd import chart
from test_gpu_part_attention import Batch, compare
from test_gpu_token_ops import OK, cuda, dev, ptr  # noqa: F401

torch = pytest.importorskip("torch")


def wide(table, pages):
    """The same sequences' pages in a table of that many; the places behind them are of no page."""
    t = torch.full((table.shape[0], pages), 1 << 30, dtype=torch.int32, device="cuda")
    t[:, : table.shape[1]] = table
    return t


WIDE = [  # (head_dim, KV heads, queries of each, tokens, contexts, page, block, top, first, last)
    (64, 2, 7, [1, 1, 1], [900, 64, 1400], 64, 32, 4, 1, 1), (128, 2, 6, [1] * 40, [300 + 90 * i for i in range(40)], 64, 64, 8, 1, 1),
    (64, 2, 7, [600, 40], [2000, 900], 128, 64, 6, 1, 1), (128, 2, 6, [520], [1531], 64, 64, 4, 0, 2), (256, 4, 2, [100, 1, 217], [400, 700, 1100], 64, 32, 6, 0, 0),
    (64, 3, 9, [200, 201], [700, 800], 32, 32, 65, 1, 0), (128, 2, 3, [70, 250], [3000, 260], 32, 32, 30, 2, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,G,qs,ctx,page,block,top,first,last", WIDE)
def test_a_table_wider_than_its_contexts_changes_nothing(dim, kv, G, qs, ctx, page, block, top, first, last):
    """The same values bit for bit, and no byte more of scratch (but for lists that a narrow table cuts short)."""
    d = chart.Device(0)
    B = Batch(d, qs, ctx, kv, G, dim, page, seed=dim + kv)
    means = B.means(block)

    def held():
        n = ctypes.c_size_t()
        assert d.lib.ah_ctx_scratch_bytes(d.h, ctypes.byref(n)) == OK
        return n.value

    status, out, chosen = B.blocks(means, block, top, first, last)
    before, more = held(), 5 * sum(qs) * kv * (top + first + last + 2) if top + first + last >= B.P.per * page // block else 0
    assert status == OK
    for pages in (B.P.per + 1, 2048, 1 << 17):
        t = wide(B.P.table, pages)
        status, o, c = B.blocks(means, block, top, first, last, table=t, table_stride=pages)
        assert status == OK and np.array_equal(o, out) and np.array_equal(c, chosen) and held() <= before + more, pages
    d.close()


LONGER = [  # (head_dim, KV heads, queries of each, tokens, contexts, page, block, top, first, last)
    (64, 2, 2, [1, 1, 1], [20011, 9000, 8320], 64, 32, 8, 1, 1), (64, 1, 3, [1, 2], [31000, 17000], 1024, 32, 100, 3, 2), (128, 2, 1, [1], [20000], 32, 32, 300, 0, 0),
    (64, 2, 1, [280], [20011], 64, 32, 8, 1, 1), (128, 2, 2, [250, 40], [9000, 18000], 128, 32, 20, 0, 3), (256, 4, 1, [30, 250], [40, 19000], 64, 32, 3, 2, 0),
    (64, 2, 1, [270], [20000], 64, 32, 90, 1, 0), (128, 2, 1, [260], [26000], 64, 32, 595, 0, 1), (128, 2, 1, [260], [25000], 64, 32, 596, 0, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,G,qs,ctx,page,block,top,first,last", LONGER)
def test_contexts_longer_than_planned_are_served_whole(dev, dim, kv, G, qs, ctx, page, block, top, first, last):  # noqa: F811
    """The choice by passes, over what a call that plans for less keeps in LDS."""
    B = Batch(dev, qs, ctx, kv, G, dim, page, seed=dim + kv)
    means = B.means(block)
    want = [B.choose(s, block, top, first, last) for s in range(len(qs))]
    for max_ctx in (max(ctx), 0, 1, 3 * block, 300 * block, 400 * block, 10 ** 9):
        status, out, chosen = B.blocks(means, block, top, first, last, max_ctx=max_ctx)
        assert status == OK
        for s in range(len(qs)):
            assert np.array_equal(chosen[B.start[s]:B.start[s + 1]], want[s][0]), max_ctx
            if max_ctx in (0, max(ctx)):
                compare(B.rows(s, out), B.rows(s, B.q), B.k[s], B.v[s], want[s][1], B.scale)


@pytest.mark.gpu
@pytest.mark.parametrize("blocks,top,n", [(700, 5, 1), (700, 64, 1), (1500, 65, 1), (1500, 1000, 1), (700, 5, 300), (800, 64, 300), (800, 70, 300)])
def test_equal_scores_take_the_first_blocks_by_passes_too(dev, blocks, top, n):  # noqa: F811
    """Means of small whole numbers, so that sums are exact and many scores equal; one of NaN, which is chosen last."""
    rng = np.random.default_rng(blocks + top)
    B = Batch(dev, [n], [32 * blocks + 7], 2, 2, 64, 32, seed=blocks)
    B.q = rng.integers(-2, 3, B.q.shape).astype(np.float32)
    B.q[-1] = 0  # all equal
    per = -(-B.ctxs[0] // 32)
    means = torch.zeros(B.P.cache.n_pages, 1, 2, 64, dtype=torch.float16, device="cuda")
    value = rng.integers(-1, 2, (per, 2, 64)).astype(np.float16)
    value[3::7] = value[3]
    value[10] = np.nan
    means[B.P.table[0].long()[:per], 0] = cuda(value)
    for max_ctx in (1, B.ctxs[0]):
        status, out, chosen = B.blocks(means, 32, top, 0, 0, max_ctx=max_ctx)
        assert status == OK
        for t, pos in enumerate(B.positions(0)):
            for h in range(2):
                score = value[: pos // 32, h].astype(np.float64) @ B.q[t, 128 * h:128 * h + 128].reshape(2, 64).astype(np.float64).sum(0)
                score[10] = -np.inf
                assert np.array_equal(chosen[t, h], np.sort(np.argsort(-score, kind="stable")[:top])), (t, h, max_ctx)


@pytest.mark.gpu
def test_tens_of_thousands_of_idle_sequences_and_many_kv_heads(dev):  # noqa: F811
    """As without them, where they would be too many tiles of 16 tokens for a launch."""
    B = Batch(dev, [8], [290], 80, 1, 64, 32, seed=3)
    means = B.means(32)
    status, want, chosen = B.blocks(means, 32, 3, 1, 0)
    assert status == OK
    n_seq = 65535
    start, c = np.full(n_seq + 1, 8, np.int32), np.zeros(n_seq, np.int32)
    start[0], c[0] = 0, 290
    table = torch.zeros(n_seq, B.P.per, dtype=torch.int32, device="cuda")
    table[0] = B.P.table[0]
    status, out, picked = B.blocks(means, 32, 3, 1, 0, start=start, ctx=c, table=table, n_seq=n_seq)
    assert status == OK and np.array_equal(picked, chosen)
    see = B.choose(0, 32, 3, 1, 0)[1]
    for x in (out, want):
        compare(B.rows(0, x), B.rows(0, B.q), B.k[0], B.v[0], see, B.scale)
