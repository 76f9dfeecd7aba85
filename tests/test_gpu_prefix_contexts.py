"""Sequences behind a common prefix whose contexts end before it, or that have no tokens: on every route that the call may
take (each sequence for itself, units of 16, 32 and 128 rows of the prefix, 8, 16 and 128 of what follows it)."""
import numpy as np
import pytest

from test_gpu_part_attention import Batch
from test_gpu_token_ops import CACHE, OK, dev  # noqa: F401

torch = pytest.importorskip("torch")

ROUTES = [  # (head_dim, KV heads, queries of each, tokens, contexts, prefix)
    (64, 2, 7, [3, 1, 5], [700, 641, 650], 640),              # each for itself, 16 rows
    (64, 2, 2, [3, 1, 4], [700, 641, 650], 640),              # each for itself, 8 rows
    (128, 2, 4, [2, 1, 2], [5000, 4801, 4802], 4800),         # 16 rows of the prefix, 8 behind it
    (256, 2, 3, [9, 1, 2], [700, 641, 650], 640),             # 16 and 16
    (128, 2, 6, [20, 1, 130], [5000, 4801, 4930], 4800),      # 32
    (64, 2, 7, [200, 90, 31, 1], [900, 750, 700, 650], 640),  # 128 of the prefix
    (128, 8, 16, [16] * 30, [2070 + i for i in range(30)], 2048), (64, 32, 16, [9, 16, 12] * 13, [150 + i for i in range(39)], 100)]  # 128 and 128


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,G,qs,ctx,prefix", ROUTES)
def test_fewer_positions_than_tokens_behind_a_prefix_are_refused(dev, dim, kv, G, qs, ctx, prefix):  # noqa: F811
    """Tokens at positions before 0, or before the prefix's end: not written, and the others as before."""
    B = Batch(dev, qs, ctx, kv, G, dim, 64, prefix=prefix, seed=dim)
    status, good = B.shared()
    assert status == OK
    last = len(qs) - 1
    for s in (0, 1, last):
        for value in sorted({0, qs[s] // 2, qs[s] - 1, qs[s], prefix // 2, prefix, prefix + qs[s] - 1}):
            c = np.array(ctx)
            c[s] = value
            status, out = B.shared(ctx=c)
            rows = np.arange(B.start[s], B.start[s + 1])
            assert status == CACHE and (out[rows] == 7).all(), (s, value)
            assert np.array_equal(np.delete(out, rows, 0), np.delete(good, rows, 0)), (s, value)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,kv,G,qs,ctx,prefix", ROUTES)
def test_sequences_without_tokens_behind_a_prefix_are_passed_over(dev, dim, kv, G, qs, ctx, prefix):  # noqa: F811
    """Idle slots of a batch, whatever their contexts: the call is served as without them."""
    idle = 0, 2, len(qs) + 2
    qs, ctx = [0, qs[0], 0, *qs[1:], 0], [prefix, ctx[0], prefix, *ctx[1:], prefix]
    B = Batch(dev, qs, ctx, kv, G, dim, 64, prefix=prefix, seed=dim)
    status, want = B.shared()
    assert status == OK and (want[:, : B.heads * dim] != 7).all()
    for values, expect in (((0, 0, 0), OK), ((1, prefix - 1, 0), OK), ((0, -1, prefix), CACHE), ((10 ** 6, 0, 0), CACHE)):
        c = np.array(ctx)
        c[list(idle)] = values
        status, out = B.shared(ctx=c)
        assert status == expect and np.array_equal(out, want), values
