"""How far attention is from 64 bits, as a root mean square over a call: a bound that a lost half of q or of a weight
breaks (shown on the CPU), over every kernel and every way of joining pieces.

A call's error relative to its outputs, in units of u = 2^-24 (f32's rounding): a score of S powers of two is rounded on its
way to the exponential (2 S, its largest taken), exp2, the halves of q and of a weight and the f32 products take a
few each (8), and sums over c keys about sqrt(c) (half a unit each, at random).
"""
import numpy as np
import pytest

from test_gpu_token_ops import OK, Paged, U, cuda, dev, filled, ptr, quantize4, stream  # noqa: F401

torch = pytest.importorskip("torch")


def exact(q, k, v, scale, nq, c, half_q=False, half_p=False):
    """f64 attention of one sequence's nq rows [nq][heads][dim] over k, v [c][kv][dim], and its largest score in powers of
    two; half_*: q or the weights as one f16 (as if their low halves were lost)."""
    heads, kv = q.shape[1], k.shape[1]
    see = np.arange(c)[None] <= (c - nq + np.arange(nq))[:, None]
    out, S = np.zeros(q.shape), 0.0
    for h in range(heads):
        x = q[:, h].astype(np.float64)
        if half_q:
            up = 2.0 ** (13 - np.floor(np.log2(np.abs(x).max(-1, keepdims=True))))
            x = (x * up).astype(np.float16).astype(np.float64) / up
        s = np.where(see, x @ k[:c, h * kv // heads].astype(np.float64).T * scale * np.log2(np.e), -np.inf)
        S = max(S, np.abs(s[see]).max())
        p = np.exp2(s - s.max(-1, keepdims=True))
        w = (p * 2.0 ** 11).astype(np.float16).astype(np.float64) / 2.0 ** 11 if half_p else p
        out[:, h] = w @ v[:c, h * kv // heads].astype(np.float64) / p.sum(-1, keepdims=True)
    return out, S


def bound(S, c):
    return U * (8 + 2 * S + np.sqrt(c))


# (KV heads, heads of each, tokens and contexts): single tokens whole, in pieces, in two levels of pieces; a few tokens;
# chunks whole, in pieces, even and uneven; chunks beside single tokens
CALLS = {"one": (2, 6, [1], [129]), "one in pieces": (2, 6, [1], [5000]), "one in groups of pieces": (1, 4, [1], [60000]), "few": (2, 4, [5, 3, 1], [700, 2100, 64]),
         "chunk": (2, 7, [300], [700]), "prompt": (1, 6, [1100], [1100]), "even": (2, 4, [100] * 9, [900] * 9), "uneven": (2, 3, [200, 61, 140], [3000, 300, 1400]),
         "mixed": (1, 7, [200] + [1] * 30, [900] + [400] * 30)}


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("call", CALLS)
def test_root_mean_square_error(dev, dim, call):  # noqa: F811
    kv, G, qs, ctx = CALLS[call]
    P, k, v = filled(dev, ctx, 64, kv, dim, seed=dim, spread=1.5)
    rng = np.random.default_rng(dim)
    q = rng.standard_normal((sum(qs), kv * G, dim)).astype(np.float32)
    start = np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)
    dq, ds, dc = cuda(q), cuda(start), cuda(np.asarray(ctx, np.int32))
    out = torch.full_like(dq, 7.0)
    P.cache.attn_dev(ptr(dq), ptr(out), n_heads=kv * G, n_tok=sum(qs), n_seq=len(qs), q_start_ptr=ptr(ds), ctx_ptr=ptr(dc), table_ptr=ptr(P.table),
                     table_stride=P.per, max_q=max(qs), max_ctx=max(ctx), scale=dim ** -0.5, stream=stream())
    assert dev.sync_status(stream()) == OK
    got = out.cpu().numpy()
    for s, (n, c) in enumerate(zip(qs, ctx)):
        rows = slice(start[s], start[s + 1])
        ref, S = exact(q[rows], k[s], v[s], dim ** -0.5, n, c)
        err = np.linalg.norm(got[rows] - ref) / np.linalg.norm(ref)
        assert err <= bound(S, c), (s, err, bound(S, c))


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,c", [(1, 129), (1, 5000), (5, 700), (60, 300), (1, 60000)])
def test_the_bound_notices_a_lost_half(dim, n, c):
    rng = np.random.default_rng(dim + c)
    q = rng.standard_normal((n, 2, dim)).astype(np.float32)
    k, v = quantize4((1.5 * rng.standard_normal((c, 1, dim))).astype(np.float32)), quantize4(rng.standard_normal((c, 1, dim)).astype(np.float32))
    ref, S = exact(q, k, v, dim ** -0.5, n, c)
    for lost in (dict(half_q=True), dict(half_p=True)):
        err = np.linalg.norm(exact(q, k, v, dim ** -0.5, n, c, **lost)[0] - ref) / np.linalg.norm(ref)
        assert err > 2 * bound(S, c), (lost, err, bound(S, c))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,G", [(136, 8), (1, 4)], ids=["chunk", "token"])
def test_a_long_tail_of_small_weights(dev, dim, n, G):  # noqa: F811
    """One key's weight and 40000 others of 2^-20 to 2^-24 of it, every value 1: the output is 1.  The running sums stay between
    one and two times the large weight, so an addition rounds by up to half of 2 u, 2 u / sqrt(12) at random.  They see an
    addition for every 16 keys (of the weights' halves: two) and, of the weights themselves, one for 32 at the most: in all
    2 u sqrt(c (1/16 + 1/16 + 1/32) / 12), 2.5 times which is allowed.  (One addition a key, each of less than the sum's
    last place, would lose or gain up to u of the sum every time.)"""
    c = 40037
    rng = np.random.default_rng(dim)
    k, v = np.zeros((c, 1, dim), np.float32), np.ones((c, 1, dim), np.float32)
    k[:, 0, 0] = rng.uniform(0, 4, c)
    k[n % 7, 0, 0] = 24.0
    P = Paged(dev, 1, c, 1024, 1, dim)
    P.append(np.zeros(c), np.arange(c), k, v)
    q = np.zeros((n, G, dim), np.float32)
    q[..., 0] = rng.uniform(0.97, 1.03, (n, G))
    dq, ds, dc = cuda(q), cuda(np.array([0, n], np.int32)), cuda(np.array([c], np.int32))
    out = torch.full_like(dq, 7.0)
    # (a bound of 64 keys: the context in one piece, one running maximum for all of it or for a wave's share)
    P.cache.attn_dev(ptr(dq), ptr(out), n_heads=G, n_tok=n, n_seq=1, q_start_ptr=ptr(ds), ctx_ptr=ptr(dc), table_ptr=ptr(P.table), table_stride=P.per, max_q=n,
                     max_ctx=64, scale=float(np.log(2.0)), stream=stream())
    assert dev.sync_status(stream()) == OK
    err = out.cpu().numpy().astype(np.float64) - 1
    assert np.sqrt((err ** 2).mean()) <= 2.5 * 2 * U * np.sqrt(c * (5 / 32) / 12), (err.mean(), err.std())
