"""The operators between a token's projections against plain 64-bit implementations: residual + norm +
quantizer, rotary positions, the 4-bit cache, attention over it, sampling.

Tolerances are derived from the arithmetic (u = 2^-24, f32's rounding):
  norm       y = (s R) g takes three roundings (R's own included): 4 u |y|.  The QuantAct is compared bit for bit
             with the oracle's on the y that came back.
  rope       cosine, sine, two products and a sum are rounded: 4 u (|a| + |b|) m, and the f64 angle's own error,
             8 * 2^-53 pos theta (|a| + |b|) m.
  cache      codes are compared exactly (numpy's f32 operations are the definition's).
  attention  a score errs by the two halves of q (2^-21 of the row's largest |q| against sum |k|) and the f32 sums of
             2 D products; the weights by that times 2, exp2 and its argument's rounding (|score| u); the output by
             the weights' two halves and the f32 sums over the keys.  All relative to sum p |v| / sum p.
  sampling   weights err by exp's last bit and its argument's rounding, under 2^-17; the random numbers stand in the
             middle of a token's interval and the limits between two tokens, so the token is certain.
"""
import ctypes

import numpy as np
import pytest

import oracle
from apeiron_amd import chart

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
OK, NONFINITE, RANGE, INVALID, CACHE = 0, 10, 11, 21, 27


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "GPU tests need the MI355X"
    d = chart.Device(0)
    yield d
    d.close()


def stream():
    return torch.cuda.current_stream().cuda_stream


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


# ---- norm -----------------------------------------------------------------------------------------


def norm(dev, x, r, g, eps=1e-6, inplace=False):
    n_tok, n = x.shape
    dx, dr, dg = cuda(x), None if r is None else cuda(r), cuda(g)
    s = (dx if r is None else dr) if inplace else torch.full((n_tok, n), 7.0, device="cuda")
    y = torch.full((n_tok, n), 7.0, device="cuda")
    codes = torch.full((n_tok, n), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((n_tok, -(-n // 32)), 99, dtype=torch.int64, device="cuda")
    values = torch.full((n_tok, n), 7.0, dtype=torch.bfloat16, device="cuda")
    chart.norm_quant_dev(dev, ptr(dx), ptr(dg), eps, n_tok, n, residual_ptr=ptr(dr), sum_ptr=ptr(s), y_ptr=ptr(y), codes_ptr=ptr(codes),
                         scales_ptr=ptr(scales), values_ptr=ptr(values), stream=stream())
    st = dev.sync_status(stream())
    return st, s.cpu().numpy(), y.cpu().numpy(), codes.cpu().numpy(), scales.cpu().numpy(), values.float().cpu().numpy()


@pytest.mark.parametrize("n_tok,n,res", [(1, 1, True), (3, 7, False), (1, 31, True), (5, 32, True), (2, 33, False), (7, 896, True),
                                         (4, 1531, True), (2, 512, True), (3, 513, False), (2, 4097, True), (1, 8192, True), (2, 8193, True),
                                         (1, 16387, True), (1, 32768, True), (300, 64, True)])
def test_norm_matches_f64_and_the_quantizer(dev, n_tok, n, res):
    rng = np.random.default_rng(n * 7 + n_tok)
    x = rng.standard_normal((n_tok, n)).astype(np.float32)
    r = (rng.standard_normal((n_tok, n)) * 30).astype(np.float32) if res else None
    g = (1 + 0.3 * rng.standard_normal(n)).astype(np.float32)
    st, s, y, codes, scales, values = norm(dev, x, r, g, inplace=n % 2 == 0)
    assert st == OK
    want = x if r is None else x + r  # one f32 addition
    assert np.array_equal(s, want)
    v = want.astype(np.float64)
    ref = v / np.sqrt((v * v).mean(-1, keepdims=True) + 1e-6) * g
    assert (np.abs(y - ref) <= 4 * U * np.abs(ref)).all()
    for t in range(n_tok):
        ost, oc, osc = oracle.quant_act_f32(y[t])
        assert ost == 0 and np.array_equal(codes[t], oc) and np.array_equal(scales[t], osc)
        real = oc.astype(np.float64) * np.repeat(osc, 32)[:n].astype(np.float64) * 2.0 ** -32
        assert np.array_equal(values[t].astype(np.float64), real)


def test_norm_extremes_and_refusals(dev):
    g = np.ones(70, np.float32)
    # a row of zeros, one whose squares would leave f32, and one whose squares vanish in it
    x = np.zeros((3, 70), np.float32)
    x[1], x[2] = 1e25, 1e-25
    st, s, y, codes, scales, values = norm(dev, x, None, g, eps=1e-6)
    assert st == OK and np.array_equal(y[0], np.zeros(70)) and np.abs(y[1] - 1).max() <= 4 * U
    assert np.abs(y[2] - 1e-22).max() <= 4 * U * 1e-22 and (codes[0] == 0).all() and (scales[0] == 0).all()
    for bad in (np.nan, np.inf, -np.inf):
        x = np.ones((2, 70), np.float32)
        x[1, 40] = bad
        assert norm(dev, x, None, g)[0] == NONFINITE
    assert norm(dev, np.ones((1, 70), np.float32), None, g * 1e12)[0] == RANGE
    L, x = dev.lib, torch.ones(64, device="cuda")
    c = torch.zeros(64, dtype=torch.int8, device="cuda")
    assert L.ah_norm_quant_dev(dev.h, ptr(x), None, ptr(x), 1e-6, 1, 64, None, None, ptr(c), None, None, None) == INVALID
    assert L.ah_norm_quant_dev(dev.h, ptr(x), None, ptr(x), -1.0, 1, 64, None, ptr(x), None, None, None, None) == INVALID
    assert L.ah_norm_quant_dev(dev.h, ptr(x), None, ptr(x), float("nan"), 1, 64, None, ptr(x), None, None, None, None) == INVALID
    assert L.ah_norm_quant_dev(dev.h, ptr(x), None, ptr(x), 1e-6, 1, 32769, None, ptr(x), None, None, None, None) == INVALID
    assert L.ah_norm_quant_dev(dev.h, ptr(x), None, None, 1e-6, 1, 64, None, ptr(x), None, None, None, None) == INVALID
    assert L.ah_norm_quant_dev(dev.h, None, None, None, 1e-6, 0, 64, None, None, None, None, None, None) == OK
    assert dev.sync_status() == OK


# ---- rotary positions -----------------------------------------------------------------------------


def frequencies(rot, base, scaling):
    theta = np.array([base ** (-2.0 * j / rot) for j in range(rot // 2)])
    if scaling is None:
        return theta, 1.0
    kind, f, *rest = scaling
    if kind == "linear":
        return theta / f, 1.0
    if kind == "ntk":
        return np.array([(base * f ** (rot / (rot - 2))) ** (-2.0 * j / rot) for j in range(rot // 2)]), 1.0
    low, high, original = rest
    g = np.clip((original * theta / (2 * np.pi) - low) / (high - low), 0, 1)
    return theta * ((1 - g) / f + g), 0.1 * np.log(f) + 1


def rotate(x, pos, theta, m, rot, layout):
    """f64 rotation of x [tok][head][dim] and the tolerance."""
    x = x.astype(np.float64)
    a = (pos.astype(np.float64)[:, None] * theta)[:, None]
    c, s = m * np.cos(a), m * np.sin(a)
    y, tol = x.copy(), np.zeros_like(x)
    i, j = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    t = (np.abs(x[..., i]) + np.abs(x[..., j])) * m * (4 * U + 8 * 2.0 ** -53 * np.abs(a))
    tol[..., i] = tol[..., j] = t
    return y, tol


SCALINGS = [None, ("linear", 4.0), ("ntk", 8.0), ("bands", 8.0, 1.0, 32.0, 4096.0)]


@pytest.mark.parametrize("dim,rot,layout", [(128, 128, "half"), (64, 32, "interleaved"), (64, 20, "half"), (100, 100, "half"), (10, 6, "interleaved"),
                                            (256, 64, "half"), (512, 512, "interleaved"), (2, 2, "half")])
@pytest.mark.parametrize("scaling", SCALINGS)
def test_rope_matches_f64(dev, dim, rot, layout, scaling):
    if scaling and scaling[0] == "ntk" and rot == 2:
        pytest.skip("no frequency but the first")
    rng = np.random.default_rng(dim + rot)
    n_tok, heads, xs = 5, 3, 3 * dim + 6
    rope = chart.Rope(dev, dim, rot, layout=layout, base=1e6, scaling=scaling)
    theta, m = frequencies(rot, 1e6, scaling)
    got_theta, got_m = rope.info()
    assert np.abs(got_theta / theta - 1).max() <= 64 * 2.0 ** -53 and abs(got_m - m) <= 4 * 2.0 ** -53
    x = rng.standard_normal((n_tok, xs)).astype(np.float32)
    pos = np.array([0, 1, 131071, -3, 1 << 20], np.int32)
    dx, dp, dy = cuda(x), cuda(pos), torch.full((n_tok, heads * dim), 7.0, device="cuda")
    rope.rotate_dev(ptr(dx), ptr(dy), heads, ptr(dp), n_tok, x_stride=xs, stream=stream())
    ref, tol = rotate(x[:, :heads * dim].reshape(n_tok, heads, dim), pos, got_theta, got_m, rot, layout)
    y = dy.cpu().numpy().reshape(n_tok, heads, dim)
    assert (np.abs(y - ref) <= tol).all(), np.abs(y - ref).max()
    rope.rotate_dev(ptr(dx), ptr(dx), heads, ptr(dp), n_tok, x_stride=xs, y_stride=xs, stream=stream())  # in place
    z = dx.cpu().numpy()
    assert np.array_equal(z[:, :heads * dim], y.reshape(n_tok, -1)) and np.array_equal(z[:, heads * dim:], x[:, heads * dim:])
    rope.free()


def test_rope_refusals(dev):
    for bad in (dict(head_dim=64, rot_dim=66), dict(head_dim=64, rot_dim=7), dict(head_dim=514), dict(head_dim=64, base=0.0),
                dict(head_dim=64, base=float("inf")), dict(head_dim=64, scaling=("linear", 0.0)), dict(head_dim=64, rot_dim=2, scaling=("ntk", 2.0)),
                dict(head_dim=64, scaling=("bands", 2.0, 4.0, 4.0, 100.0)), dict(head_dim=64, scaling=("bands", 2.0, 1.0, 4.0, 0.0)),
                dict(head_dim=64, rot_dim=0)):
        with pytest.raises(chart.MatvecError) as e:
            chart.Rope(dev, **bad)
        assert e.value.status == INVALID, bad
    rope, x = chart.Rope(dev, 64), torch.zeros(4, 64, device="cuda")
    for kw in (dict(x_stride=63), dict(y_stride=63), dict(x_stride=64, y_stride=128)):
        with pytest.raises(chart.MatvecError):
            rope.rotate_dev(ptr(x), ptr(x), 1, ptr(x), 2, **kw)
    rope.rotate_dev(None, None, 1, None, 0)


# ---- the cache ------------------------------------------------------------------------------------


def quantize4(x):
    """The cache's values for f32 rows (last axis whole blocks), by the definition in f32."""
    b = x.reshape(*x.shape[:-1], -1, 32).astype(np.float32)
    hi, lo = b.max(-1, keepdims=True), b.min(-1, keepdims=True)
    d = (np.where(hi >= -lo, hi, lo) * np.float32(-0.125)).astype(np.float32)
    e = np.maximum(np.frexp(d)[1] - 8, -24)
    d = np.clip(np.ldexp(np.rint(np.ldexp(d, -e)), e), -8160, 8160).astype(np.float32)
    assert np.array_equal(d.astype(np.float16).astype(np.float32), d)
    with np.errstate(over="ignore"):
        c = np.clip(np.rint((b / np.where(d == 0, np.float32(1), d)).astype(np.float32)), -8, 7) * (d != 0)
    v = (c * d).reshape(x.shape)
    assert np.array_equal(v.astype(np.float16).astype(np.float32), v)  # every value is an f16
    return v


class Paged:
    """A cache and a shuffled page table for n_seq sequences of up to `length` positions."""

    def __init__(self, dev, n_seq, length, page, kv, dim, extra=2, seed=0):
        per = max(1, -(-length // page))
        self.cache = chart.KvCache4(dev, n_seq * per + extra, page, kv, dim)
        self.table = cuda(np.random.default_rng(seed).permutation(n_seq * per + extra)[: n_seq * per].reshape(n_seq, per).astype(np.int32))
        self.n_seq, self.per = n_seq, per

    def where(self, seq, pos):
        self.keep = cuda(np.asarray(seq, np.int32)), cuda(np.asarray(pos, np.int32))
        return dict(seq_ptr=ptr(self.keep[0]), pos_ptr=ptr(self.keep[1]), n_tok=len(seq), table_ptr=ptr(self.table), n_seq=self.n_seq,
                    table_stride=self.per)

    def append(self, seq, pos, k, v, rope=None, **kw):
        dk, dv = cuda(k), cuda(v)
        self.cache.append_dev(rope, k_ptr=ptr(dk), v_ptr=ptr(dv), stream=stream(), **self.where(seq, pos), **kw)
        torch.cuda.synchronize()

    def read(self, seq, pos):
        k = torch.full((len(seq), self.cache.n_kv_heads, self.cache.head_dim), 7.0, dtype=torch.float16, device="cuda")
        v = k.clone()
        self.cache.read_dev(k_ptr=ptr(k), v_ptr=ptr(v), stream=stream(), **self.where(seq, pos))
        return k.float().cpu().numpy(), v.float().cpu().numpy()


@pytest.mark.parametrize("dim,kv,page", [(64, 1, 32), (64, 3, 128), (128, 2, 64), (128, 1, 1024), (256, 2, 32), (256, 5, 64)])
def test_cache_holds_the_formats_values(dev, dim, kv, page):
    rng = np.random.default_rng(dim + kv)
    length = page + 45
    P = Paged(dev, 2, length, page, kv, dim)
    n = 2 * length
    seq, pos = np.repeat([0, 1], length), np.tile(np.arange(length), 2)
    order = rng.permutation(n)  # any order of tokens
    k, v = (rng.standard_normal((n, kv, dim)) * np.exp(rng.standard_normal((n, kv, dim)))).astype(np.float32), rng.standard_normal((n, kv, dim)).astype(np.float32)
    k[3], k[4], k[5] = 0, 1e-7, 3e38  # zeros, values at f16's smallest step, values past its range
    k[6, :, 5] = 1e6
    v[7] = 2.0 ** -14 * rng.standard_normal((kv, dim))
    k[8] = np.where(np.arange(dim) % 2, 5.0, -5.0)  # both signs of the largest magnitude
    P.append(seq[order], pos[order], k[order], v[order])
    gk, gv = P.read(seq, pos)
    assert dev.sync_status(stream()) == OK
    assert np.array_equal(gk, quantize4(k)) and np.array_equal(gv, quantize4(v))
    # a position written again holds the new values, its neighbours the old ones
    P.append([1], [33], v[:1], k[1:2])
    k[length + 33], v[length + 33] = v[0], k[1]
    gk, gv = P.read(seq, pos)
    assert np.array_equal(gk, quantize4(k)) and np.array_equal(gv, quantize4(v))


@pytest.mark.parametrize("dim,rot,layout,scaling", [(128, 128, "half", None), (64, 32, "half", ("linear", 2.0)), (256, 64, "interleaved", ("bands", 8.0, 1.0, 32.0, 4096.0)),
                                                    (64, 20, "half", None)])
def test_append_rotates_and_quantizes(dev, dim, rot, layout, scaling):
    rng = np.random.default_rng(rot)
    n, heads, kv = 9, 5, 2
    rope = chart.Rope(dev, dim, rot, layout=layout, base=1e4, scaling=scaling)
    width = (heads + 2 * kv) * dim + 10  # q, k and v as one projection's row
    x = rng.standard_normal((n, width)).astype(np.float32)
    pos = np.array([0, 1, 31, 32, 63, 64, 90, 33, 2], np.int32)
    P = Paged(dev, n, 96, 32, kv, dim)
    dx, dp = cuda(x), cuda(pos)
    out = torch.full((n, heads * dim + 4), 7.0, device="cuda")
    tokens = P.where(np.arange(n), pos)
    args = dict(q_ptr=ptr(dx), n_heads=heads, q_stride=width, k_ptr=ptr(dx) + 4 * heads * dim, k_stride=width,
                v_ptr=ptr(dx) + 4 * (heads + kv) * dim, v_stride=width, stream=stream(), **tokens)
    P.cache.append_dev(rope, q_out_ptr=ptr(out), q_out_stride=heads * dim + 4, **args)
    torch.cuda.synchronize()
    both = torch.empty(n, (heads + kv) * dim, device="cuda")
    rope.rotate_dev(ptr(dx), ptr(both), heads + kv, ptr(dp), n, x_stride=width, stream=stream())
    both = both.cpu().numpy()
    got = out.cpu().numpy()
    assert np.array_equal(got[:, :heads * dim], both[:, :heads * dim]) and (got[:, heads * dim:] == 7).all()
    gk, gv = P.read(np.arange(n), pos)
    assert np.array_equal(gk, quantize4(both[:, heads * dim:].reshape(n, kv, dim)))
    assert np.array_equal(gv, quantize4(x[:, (heads + kv) * dim:(heads + 2 * kv) * dim].reshape(n, kv, dim)))
    P.cache.append_dev(rope, q_out_ptr=ptr(dx), q_out_stride=width, **args)  # q in place
    assert np.array_equal(dx.cpu().numpy()[:, :heads * dim], both[:, :heads * dim])
    assert dev.sync_status(stream()) == OK


def test_cache_refusals(dev):
    for bad in ((0, 32, 1, 64), (4, 16, 1, 64), (4, 48, 1, 64), (4, 2048, 1, 64), (4, 32, 0, 64), (4, 32, 1, 96), (4, 32, 5000, 64)):
        with pytest.raises(chart.MatvecError) as e:
            chart.KvCache4(dev, *bad)
        assert e.value.status == INVALID, bad
    P = Paged(dev, 2, 64, 32, 1, 64)
    assert P.cache.info() == (6 * 36 * 64, 6, 32, 1, 64)
    k = np.ones((4, 1, 64), np.float32)
    P.append([0, 1], [5, 6], k[:2], k[:2])
    assert dev.sync_status(stream()) == OK
    # padding tokens are passed over; a sequence, position or page outside is refused and passed over
    P.append([-1, 0], [5, 7], 2 * k[:2], 2 * k[:2])
    assert dev.sync_status(stream()) == OK
    for seq, pos in (([2], [0]), ([0], [64]), ([0], [-1])):
        P.append(seq, pos, k[:1], k[:1])
        assert dev.sync_status(stream()) == CACHE, (seq, pos)
    P.table[1, 1] = 6
    P.append([1, 0], [33, 9], k[:2], k[:2])
    assert dev.sync_status(stream()) == CACHE
    gk, _ = P.read([0, 0, 0, 1, 1], [5, 7, 9, 33, 6])
    assert dev.sync_status(stream()) == CACHE
    assert np.array_equal(gk[:, 0, 0], [1, 2, 1, 0, 1])
    # a block with a value that is not finite is zeros, the other block is kept
    k[0, 0, 3] = np.nan
    k[1, 0, 40] = np.inf
    P.append([0, 0], [10, 11], k[:2], k[2:4])
    assert dev.sync_status(stream()) == NONFINITE
    gk, gv = P.read([0, 0], [10, 11])
    assert (gk[0, 0, :32] == 0).all() and (gk[0, 0, 32:] == 1).all() and (gk[1, 0, :32] == 1).all() and (gk[1, 0, 32:] == 0).all() and (gv == 1).all()
    d = torch.zeros(256, device="cuda")
    with pytest.raises(chart.MatvecError):
        P.cache.append_dev(chart.Rope(dev, 128), k_ptr=ptr(d), v_ptr=ptr(d), **P.where([0], [0]))
    with pytest.raises(chart.MatvecError):
        P.cache.append_dev(None, k_ptr=ptr(d), v_ptr=ptr(d), k_stride=32, **P.where([0], [0]))
    with pytest.raises(chart.MatvecError):
        P.cache.append_dev(None, k_ptr=ptr(d), v_ptr=ptr(d), q_ptr=ptr(d), n_heads=1, **P.where([0], [0]))


def test_cache_past_4_gib(dev):
    """Pages whose byte offsets need more than 32 bits, appended, read and attended."""
    kv, dim, page = 8, 256, 32
    n_pages = (5 << 30) // (36 * dim * kv)
    cache = chart.KvCache4(dev, n_pages, page, kv, dim)
    rng = np.random.default_rng(5)
    k, v = rng.standard_normal((2, 64, kv, dim)).astype(np.float32)
    P = Paged.__new__(Paged)
    P.cache, P.n_seq, P.per = cache, 1, 2
    P.table = cuda(np.array([[n_pages - 1, n_pages - 3]], np.int32))
    P.append(np.zeros(64), np.arange(64), k, v)
    gk, gv = P.read(np.zeros(64), np.arange(64))
    assert np.array_equal(gk, quantize4(k)) and np.array_equal(gv, quantize4(v))
    attend(dev, P, [1], [64], heads=16, scale=dim ** -0.5, k=[quantize4(k)], v=[quantize4(v)])


# ---- attention ------------------------------------------------------------------------------------


def attend(dev, P, qs, ctx, heads, scale, k, v, window=0, sinks=0, max_ctx=None, pad=0, q_scale=1.0, seed=0):
    """Runs a ragged batch and compares every row with f64 attention over the values k[s], v[s] [ctx][kv][dim]."""
    kv, dim = P.cache.n_kv_heads, P.cache.head_dim
    G, n_tok = heads // kv, sum(qs)
    rng = np.random.default_rng(seed)
    width = heads * dim + pad
    q = (rng.standard_normal((n_tok, width)) * q_scale).astype(np.float32)
    start = np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)
    dq, out = cuda(q), torch.full((n_tok, width), 7.0, device="cuda")
    ds, dc = cuda(start), cuda(np.asarray(ctx, np.int32))
    P.cache.attn_dev(ptr(dq), ptr(out), n_heads=heads, n_tok=n_tok, n_seq=len(qs), q_start_ptr=ptr(ds), ctx_ptr=ptr(dc), table_ptr=ptr(P.table),
                     table_stride=P.per, max_q=max(qs), max_ctx=max(ctx) if max_ctx is None else max_ctx, scale=scale, window=window, sinks=sinks,
                     q_stride=width, out_stride=width, stream=stream())
    assert dev.sync_status(stream()) == OK
    got = out.cpu().numpy()
    assert (got[:, heads * dim:] == 7).all()
    for s, (nq, c) in enumerate(zip(qs, ctx)):
        if nq == 0:
            continue
        x = q[start[s]:start[s + 1], :heads * dim].reshape(nq, heads, dim).astype(np.float64)
        o = got[start[s]:start[s + 1], :heads * dim].reshape(nq, heads, dim)
        pos, key = (c - nq + np.arange(nq))[:, None], np.arange(c)[None]
        see = key <= pos
        if window:
            see &= (key > pos - window) | (key < sinks)
        for h in range(heads):
            K, V = k[s][:c, h // G].astype(np.float64), v[s][:c, h // G].astype(np.float64)
            sc = x[:, h] @ K.T * scale
            top = np.where(see, sc, -np.inf).max(-1, keepdims=True, initial=-np.inf)
            p = np.where(see, np.exp(sc - np.where(np.isfinite(top), top, 0)), 0)
            den = p.sum(-1, keepdims=True)
            safe = np.where(den > 0, den, 1)
            ref, mag = p @ V / safe, p @ np.abs(V) / safe
            size = abs(scale) * np.where(see, np.abs(x[:, h]) @ np.abs(K).T, 0).max(-1, keepdims=True, initial=0)
            wide = abs(scale) * np.abs(x[:, h]).max(-1, keepdims=True) * np.where(see, np.abs(K).sum(-1)[None], 0).max(-1, keepdims=True, initial=0)
            rel = 2 * (2.0 ** -21 * wide + (2 * dim + 4) * U * size) + 2.0 ** -18 + 2 * (c + 64) * U
            err = np.abs(o[:, h] - ref)
            assert (err <= rel * mag).all(), (s, h, err.max(), (err / np.maximum(rel * mag, 1e-30)).max())


def filled(dev, ctx, page, kv, dim, seed=0, spread=1.0):
    """A cache with random keys and values of every sequence, and those values."""
    rng = np.random.default_rng(seed)
    P = Paged(dev, len(ctx), max(max(ctx), 1), page, kv, dim, seed=seed)
    ks, vs = [], []
    for s, c in enumerate(ctx):
        k, v = (rng.standard_normal((c, kv, dim)) * spread).astype(np.float32), rng.standard_normal((c, kv, dim)).astype(np.float32)
        if c:
            P.append(np.full(c, s), np.arange(c), k, v)
        ks.append(quantize4(k) if c else k)
        vs.append(quantize4(v) if c else v)
    return P, ks, vs


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kv,G,page", [(1, 1, 32), (2, 7, 64), (2, 6, 128), (3, 8, 32), (1, 19, 64)])
def test_attention_of_single_tokens(dev, dim, kv, G, page):
    ctx = [1, 2, 31, 32, 33, 64, 65, 129, 700, 0]
    P, k, v = filled(dev, ctx, page, kv, dim, seed=dim + G)
    attend(dev, P, [1] * len(ctx), ctx, kv * G, dim ** -0.5, k, v)


@pytest.mark.parametrize("dim,kv,G,page", [(64, 2, 7, 64), (128, 2, 6, 32), (128, 1, 1, 128), (256, 2, 3, 32), (64, 1, 8, 1024), (128, 2, 16, 64), (256, 1, 5, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (40, 0), (40, 3), (64, 33), (1000000, 5)])
def test_attention_of_chunks_causal_window_sinks(dev, dim, kv, G, page, window, sinks):
    # uneven chunks: whole prompts, chunks over a prefix, none, one token, and more tokens than positions (rows that
    # see nothing come out as zeros)
    qs, ctx = [70, 33, 0, 1, 5, 150], [70, 300, 50, 200, 3, 150]
    P, k, v = filled(dev, ctx, page, kv, dim, seed=dim + G)
    attend(dev, P, qs, ctx, kv * G, dim ** -0.5, k, v, window=window, sinks=sinks, pad=4)


@pytest.mark.parametrize("dim,kv,G", [(64, 2, 7), (128, 1, 4), (256, 1, 3), (64, 1, 12)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 2)])
def test_attention_of_chunks_among_single_tokens(dev, dim, kv, G, window, sinks):
    """Long chunks, short ones, single tokens and sequences without any in one call, more than a wave has lanes."""
    rng = np.random.default_rng(dim + G)
    qs = [1] * 70 + [0, 2, 0, 9]
    for at, n in ((0, 260), (13, 40), (69, 300)):
        qs[at] = n
    ctx = [int(n + rng.integers(0, 90)) for n in qs]
    P, k, v = filled(dev, ctx, 64, kv, dim, seed=dim)
    attend(dev, P, qs, ctx, kv * G, dim ** -0.5, k, v, window=window, sinks=sinks)


@pytest.mark.parametrize("dim,kv,G,n,q,c", [(64, 1, 7, 9, 100, 700), (128, 2, 4, 8, 64, 300), (256, 1, 2, 3, 128, 400), (128, 1, 3, 17, 43, 90)])
def test_attention_of_even_chunks(dev, dim, kv, G, n, q, c):
    P, k, v = filled(dev, [c] * n, 32, kv, dim, seed=n)
    attend(dev, P, [q] * n, [c] * n, kv * G, dim ** -0.5, k, v)


@pytest.mark.parametrize("dim,kv,G,n,q,c,pad", [(64, 2, 7, 1, 300, 700, 1), (64, 2, 2, 3, 1, 900, 3), (128, 1, 6, 2, 90, 500, 2), (256, 1, 3, 2, 5, 300, 1),
                                                (64, 1, 7, 1, 2048, 2048, 1)])
def test_attention_of_rows_off_the_16_byte_grid(dev, dim, kv, G, n, q, c, pad):
    P, k, v = filled(dev, [c] * n, 64, kv, dim, seed=pad)
    attend(dev, P, [q] * n, [c] * n, kv * G, dim ** -0.5, k, v, pad=pad)


@pytest.mark.parametrize("dim,G,qs,ctx", [(64, 7, [1, 1], [900, 70]), (64, 7, [600], [700]), (64, 7, [300, 120], [2000, 900]), (128, 6, [200, 1, 90], [3000, 800, 90]),
                                          (256, 4, [64], [1500])])
def test_operators_replayed_as_a_graph(dev, dim, G, qs, ctx):
    """Norm, append, attention (pieces joined in the launch and by another) and sampling captured in a row: every
    replay, with eager work of the same context and synchronizations between, leaves what the eager calls leave."""
    kv, n_tok, n, V = 2, sum(qs), len(qs), 7001
    heads, rng = kv * G, np.random.default_rng(dim + n_tok)
    P, _, _ = filled(dev, ctx, 64, kv, dim, seed=3)
    rope = chart.Rope(dev, dim)
    f32 = lambda *s: cuda(rng.standard_normal(s).astype(np.float32))  # noqa: E731
    x, gain, q, k, v, logits = f32(n_tok, 640), f32(640), f32(n_tok, heads * dim), f32(n_tok, kv * dim), f32(n_tok, kv * dim), f32(40, V)
    seq = cuda(np.repeat(np.arange(n), qs).astype(np.int32))
    pos = cuda(np.concatenate([c - m + np.arange(m) for m, c in zip(qs, ctx)]).astype(np.int32))
    start, cx = cuda(np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)), cuda(np.asarray(ctx, np.int32))
    u, p, top = cuda(rng.random(40).astype(np.float32)), cuda(rng.choice([1.0, 0.9], 40).astype(np.float32)), cuda(rng.choice([0, 1, 30, 300], 40).astype(np.int32))
    out = [torch.zeros(n_tok, 640, dtype=torch.int8, device="cuda"), torch.zeros(n_tok, 20, dtype=torch.int64, device="cuda"), torch.zeros_like(q),
           torch.zeros_like(q), torch.zeros(40, dtype=torch.int32, device="cuda"), torch.zeros(40, device="cuda")]

    def run():
        st = stream()
        chart.norm_quant_dev(dev, ptr(x), ptr(gain), 1e-6, n_tok, 640, codes_ptr=ptr(out[0]), scales_ptr=ptr(out[1]), stream=st)
        P.cache.append_dev(rope, q_ptr=ptr(q), n_heads=heads, q_out_ptr=ptr(out[2]), k_ptr=ptr(k), v_ptr=ptr(v), seq_ptr=ptr(seq), pos_ptr=ptr(pos), n_tok=n_tok,
                           table_ptr=ptr(P.table), n_seq=n, table_stride=P.per, stream=st)
        P.cache.attn_dev(ptr(out[2]), ptr(out[3]), n_heads=heads, n_tok=n_tok, n_seq=n, q_start_ptr=ptr(start), ctx_ptr=ptr(cx), table_ptr=ptr(P.table),
                         table_stride=P.per, max_q=max(qs), max_ctx=max(ctx), scale=dim ** -0.5, stream=st)
        chart.sample_dev(dev, ptr(logits), 40, V, ptr(u), ptr(out[4]), probs_ptr=ptr(out[5]), top_k_ptr=ptr(top), top_p_ptr=ptr(p), stream=st)

    run()
    torch.cuda.synchronize()
    want = [t.clone() for t in out]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        run()
    for i in range(5):
        for t in out:
            t.zero_()
        graph.replay()
        if i % 2:
            torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        torch.cuda.synchronize()
        chart.sample_dev(dev, ptr(logits), 40, V, ptr(u), ptr(out[4]), stream=stream())  # (the same scratch and counters)
        (f32(64, 64) @ f32(64, 64)).sum().item()
    assert dev.sync_status(stream()) == OK


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attention_of_large_scores_and_long_contexts(dev, dim):
    # scores of tens of units (few keys carry the row), q far from one, and a context cut in many pieces
    P, k, v = filled(dev, [5000, 4097], 64, 2, dim, seed=3, spread=4.0)
    attend(dev, P, [1, 2], [5000, 4097], 8, dim ** -0.5, k, v)
    attend(dev, P, [1, 2], [5000, 4097], 8, dim ** -0.5 * 1e-20, k, v, q_scale=1e20)
    attend(dev, P, [1, 2], [5000, 4097], 8, dim ** -0.5 * 1e20, k, v, q_scale=1e-20)
    attend(dev, P, [2, 1], [5000, 4097], 8, -dim ** -0.5, k, v, max_ctx=64)  # a bound that the contexts pass
    attend(dev, P, [1, 1], [5000, 4097], 8, 0.0, k, v, window=3000, sinks=7, max_ctx=1 << 40)


def test_attention_is_the_same_each_time_and_on_any_stream(dev):
    P, k, v = filled(dev, [900, 77], 64, 2, 128, seed=1)
    q = torch.randn(40, 12 * 128, device="cuda")
    start, ctx = cuda(np.array([0, 30, 40], np.int32)), cuda(np.array([900, 77], np.int32))
    outs = []
    for i in range(3):
        out = torch.zeros_like(q)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            P.cache.attn_dev(ptr(q), ptr(out), n_heads=12, n_tok=40, n_seq=2, q_start_ptr=ptr(start), ctx_ptr=ptr(ctx), table_ptr=ptr(P.table),
                             table_stride=P.per, max_q=30, max_ctx=900, scale=0.09, stream=side.cuda_stream)
        side.synchronize()
        outs.append(out.cpu())
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_attention_refusals_and_values_out_of_range(dev):
    P, k, v = filled(dev, [100, 100], 32, 1, 64, seed=2)
    q, out = torch.randn(4, 128, device="cuda"), torch.full((4, 128), 7.0, device="cuda")
    ctx = cuda(np.array([100, 100], np.int32))

    def run(start, ctx=ctx, table=P.table, max_q=2, q=q, **kw):
        out.fill_(7.0)
        ds = cuda(np.array(start, np.int32))
        a = dict(n_heads=2, n_tok=4, n_seq=2, q_start_ptr=ptr(ds), ctx_ptr=ptr(ctx), table_ptr=ptr(table), table_stride=P.per, max_q=max_q,
                 max_ctx=100, scale=0.125, stream=stream()) | kw
        P.cache.attn_dev(ptr(q), ptr(out), **a)
        return dev.sync_status(stream()), out.cpu().numpy().copy()

    st, good = run([0, 2, 4])
    assert st == OK
    # a sequence whose tokens or context are out of range is not written, the other is whole
    for start, c in (([0, 2, 5], [100, 100]), ([0, 2, 1], [100, 100]), ([0, 2, 4], [100, 129]), ([0, 2, 4], [100, -1])):
        st, o = run(start, ctx=cuda(np.array(c, np.int32)))
        assert st == CACHE and np.array_equal(o[:2], good[:2]) and (o[2:] == 7).all(), (start, c)
    st, o = run([0, 1, 4], max_q=2)
    assert st == CACHE and (o[1:] == 7).all()
    # a page outside: its positions are not seen
    table = P.table.clone()
    table[1, 1] = -1
    st, o = run([0, 2, 4], table=table)
    assert st == CACHE and np.array_equal(o[:2], good[:2]) and np.isfinite(o).all() and not np.array_equal(o[2:], good[2:])
    # a row of NaN is NaN, its neighbours are not touched
    bad = q.clone()
    bad[1, 70] = float("nan")
    st, o = run([0, 2, 4], q=bad)
    assert st == OK and np.isnan(o[1, 64:]).all() and np.array_equal(o[1, :64], good[1, :64]) and np.array_equal(o[[0, 2, 3]], good[[0, 2, 3]])
    for kw in (dict(n_heads=3, n_tok=4), dict(q_start_ptr=None), dict(ctx_ptr=None), dict(table_ptr=None), dict(table_stride=0), dict(q_stride=100),
               dict(out_stride=127), dict(n_seq=70000)):
        if kw.get("n_heads") == 3:
            P2 = chart.KvCache4(dev, 4, 32, 2, 64)
            with pytest.raises(chart.MatvecError):
                P2.attn_dev(ptr(q), ptr(out), **(dict(n_seq=2, q_start_ptr=1, ctx_ptr=1, table_ptr=1, table_stride=1, max_q=1, max_ctx=1, scale=1.0) | kw))
            continue
        with pytest.raises(chart.MatvecError) as e:
            run([0, 2, 4], **kw)
        assert e.value.status == INVALID, kw
    assert run([0, 0, 0], n_tok=0)[0] == OK and run([0, 2, 4], n_seq=0)[0] == OK


# ---- sampling -------------------------------------------------------------------------------------


def kept_weights(x, T, k, p, m):
    """f64 weights of a row's kept tokens, in index order, and the order (logit descending, index ascending)."""
    x = np.where(np.isnan(x), -np.inf, x).astype(np.float64)
    order = np.argsort(-x, kind="stable")
    if T == 0:
        w = np.zeros(len(x))
        w[order[0]] = 2.0 ** 32
        return w, order, w
    with np.errstate(invalid="ignore"):
        z = np.where(x == x[order[0]], 0.0, (x - x[order[0]]) / T)
    full = np.rint(2.0 ** 32 * np.exp(z))
    w = full[order].copy()
    w[k if 0 < k < len(x) else len(x):] = 0
    if p < 1:
        before = np.cumsum(w) - w
        w[1:][before[1:] >= p * w.sum()] = 0
    w[1:][w[1:] < m * 2.0 ** 32] = 0
    kept = np.zeros(len(x))
    kept[order] = w
    return kept, order, full


def sample(dev, x, u, T=None, k=None, p=None, m=None, stride=None):
    n, V = x.shape
    wide = np.full((n, stride or V), 50.0, np.float32)  # what lies past a row is never looked at
    wide[:, :V] = x
    t = [cuda(wide), cuda(np.asarray(u, np.float32))] + [None if a is None else cuda(np.broadcast_to(np.asarray(a, d), n).copy()) for a, d in
                                                       ((T, np.float32), (k, np.int32), (p, np.float32), (m, np.float32))]
    tok = torch.full((n,), -7, dtype=torch.int32, device="cuda")
    prob = torch.full((n,), 7.0, device="cuda")
    chart.sample_dev(dev, ptr(t[0]), n, V, ptr(t[1]), ptr(tok), row_stride=stride, probs_ptr=ptr(prob), temperature_ptr=ptr(t[2]), top_k_ptr=ptr(t[3]),
                     top_p_ptr=ptr(t[4]), min_p_ptr=ptr(t[5]), stream=stream())
    return dev.sync_status(stream()), tok.cpu().numpy(), prob.cpu().numpy()


def safe_p(x, T, k, p):
    """A top-p near p halfway between the masses before two ranks."""
    w, order, full = kept_weights(x, T, k, 1.0, 0.0)
    c = np.cumsum(w[order]) / w.sum()
    j = min(int(np.searchsorted(c, p)), len(c) - 2)
    while j + 2 < len(c) and c[j + 1] - c[j] < 1e-5:
        j += 1
    return float(np.float32((c[j] + c[j + 1]) / 2)) if c[j + 1] - c[j] >= 1e-5 else 1.0


@pytest.mark.parametrize("V", [1, 2, 63, 64, 1000, 1024, 1025, 4097, 32003, 151936])
@pytest.mark.parametrize("T,k,p,m", [(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (0.3, 20, 0.5, 0.0), (1.0, 0, 1.0, 0.07),
                                     (0.9, 1000, 0.95, 0.02), (0.0, 5, 0.5, 0.0), (1.0, 1, 1.0, 0.0), (2.0, 3, 0.0, 0.0)])
def test_sampling_draws_the_token_of_the_interval(dev, V, T, k, p, m):
    rng = np.random.default_rng(V + int(100 * T) + k)
    n = 6
    x = (rng.standard_normal((n, V)) * 2.5).astype(np.float32)
    x[1] = np.rint(x[1])             # many equal logits: the cuts fall inside a tie
    x[2, : V // 2] = -np.inf         # a grammar's mask
    x[3] += 1000.0
    x[4, rng.integers(V)] += 9.0
    u, ps, want, prob = [], [], [], []
    for i in range(n):
        pi = safe_p(x[i], T, k, p) if 0 < p < 1 and T > 0 and V > 2 else p
        w, order, _ = kept_weights(x[i], T, k, pi, m)
        run = np.cumsum(w)
        picks = np.nonzero(w > 2e-5 * run[-1])[0]
        t = int(rng.choice(picks))
        u.append((run[t] - w[t] / 2) / run[-1])
        ps.append(pi)
        want.append(t)
        prob.append(w[t] / run[-1])
    st, tok, got = sample(dev, x, u, T, k, ps, m, stride=V + 3)
    assert st == OK and tok.tolist() == want
    assert (np.abs(got - np.array(prob)) <= 2.0 ** -17 * np.array(prob)).all()


def test_sampling_ties_take_the_lowest_indices(dev):
    V = 5000
    x = np.zeros((1, V), np.float32)
    x[0, ::2] = -0.0  # equal to 0
    x[0, 4000:] = 3.0
    for k in (1, 2, 999, 1000, 1001, 1200):
        last = 4000 + k - 1 if k <= 1000 else k - 1001
        first = 4000 if k <= 1000 else 0
        w, order, _ = kept_weights(x[0], 1.0, k, 1.0, 0.0)
        assert np.nonzero(w)[0][0] == first
        st, tok, _ = sample(dev, x, [0.0], 1.0, k)
        assert st == OK and tok[0] == first
        st, tok, _ = sample(dev, x, [np.float32(1 - 2.0 ** -24)], 1.0, k)
        assert st == OK and tok[0] == (4999 if k > 1000 else last)
    # the mass of a tie cut inside: 1000 equal tokens, 0.2505 of them are 251
    st, tok, prob = sample(dev, x[:, 4000:], [0.99999], 1.0, None, 0.2505)
    assert st == OK and tok[0] == 250 and abs(prob[0] - 1 / 251) < 1e-8


@pytest.mark.parametrize("V,kind", [(1 << 20, "equal"), (70000, "equal"), (151936, "narrow"), (1 << 20, "normal"), (9000, "narrow"), (40000, "rounded")])
@pytest.mark.parametrize("k,p", [(0, 0.3), (5000, 1.0), (5000, 0.7), (300, 0.9), (0, 1.0), (3, 1.0), (100, 0.6), (16, 0.7)])
def test_sampling_of_flat_rows(dev, V, kind, k, p):
    """Limits that fall among hundreds to all of a row's tokens: long lists, and rows past the lists' room."""
    rng = np.random.default_rng(V + k)
    x = {"equal": lambda: np.zeros(V), "narrow": lambda: 1e-3 * rng.standard_normal(V), "normal": lambda: rng.standard_normal(V),
         "rounded": lambda: np.rint(2 * rng.standard_normal(V)) / 2}[kind]().astype(np.float32)[None]
    # within a tie the token is certain in the middle of its interval; the limits stand between two tokens (their
    # weights differ by less than exp's error, but not within a tie)
    pi = p
    if p < 1:
        w, order, _ = kept_weights(x[0], 0.9, k, 1.0, 0.0)
        n = int((w > 0).sum() * p)
        c = np.cumsum(w[order]) / w.sum()
        pi = float(np.float32((c[n] + c[n - 1]) / 2))
    w, order, _ = kept_weights(x[0], 0.9, k, pi, 0.0)
    run = np.cumsum(w)
    for q in (0.1, 0.95):
        t = int(np.searchsorted(run, q * run[-1]))
        u = (run[t] - w[t] / 2) / run[-1]
        st, tok, prob = sample(dev, x, [u], 0.9, k, pi)
        # f32 p and u, and exp's error over a million equal shares, move the token by a few places at most
        assert st == OK and w[tok[0]] > 0 and abs(run[tok[0]] - run[t]) <= (2.0 ** -18 * run[-1] + 2 * w.max())
        assert abs(prob[0] / (w[tok[0]] / run[-1]) - 1) <= 2.0 ** -17 + 4.0 / (w > 0).sum()


@pytest.mark.parametrize("rows,V", [(13, 151936), (300, 5000), (900, 2049), (3100, 2100)])
@pytest.mark.parametrize("order", ["random", "falling"])
def test_sampling_of_many_rows(dev, rows, V, order):
    """Many rows of mixed parameters in one call: few and several workgroups a row, rows that end early beside rows
    that do not, likely tokens spread over the row or next to each other (as in a vocabulary by frequency)."""
    rng = np.random.default_rng(rows)
    x = (2.5 * rng.standard_normal((rows, V))).astype(np.float32)
    if order == "falling":
        x = np.ascontiguousarray(np.sort(x, axis=1)[:, ::-1])
    T = rng.choice([0.0, 0.3, 0.7, 1.3], rows).astype(np.float32)
    k = rng.choice([0, 1, 2, 20, 56, 57, 64, 300, 1000], rows).astype(np.int32)
    p = rng.choice([1.0, 0.9, 0.5], rows).astype(np.float32)
    u, want, prob = [], [], []
    for i in range(rows):
        if T[i] > 0 and p[i] < 1:
            p[i] = safe_p(x[i], float(T[i]), int(k[i]), float(p[i]))
        w, _, _ = kept_weights(x[i], float(T[i]), int(k[i]), float(p[i]), 0.0)
        run = np.cumsum(w)
        t = int(rng.choice(np.nonzero(w > 2e-5 * run[-1])[0]))
        u.append((run[t] - w[t] / 2) / run[-1])
        want.append(t)
        prob.append(w[t] / run[-1])
    st, tok, got = sample(dev, x, u, T, k, p)
    assert st == OK and tok.tolist() == want
    assert (np.abs(got - np.array(prob)) <= 2.0 ** -17 * np.array(prob)).all()


def test_sampling_defaults_infinities_and_refusals(dev):
    rng = np.random.default_rng(0)
    x = rng.standard_normal((4, 3000)).astype(np.float32)
    w = kept_weights(x[0], 1.0, 0, 1.0, 0.0)[0]
    st, tok, prob = sample(dev, x[:1], [0.4])  # no parameters: the softmax itself
    assert st == OK and tok[0] == np.searchsorted(np.cumsum(w), 0.4 * w.sum()) and abs(prob[0] / (w[tok[0]] / w.sum()) - 1) < 2.0 ** -17
    x[1, [7, 9]] = np.inf  # two certain tokens
    assert [sample(dev, x[1:2], [u])[1][0] for u in (0.2, 0.8)] == [7, 9]
    assert sample(dev, x[1:2], [0.8], 0.0)[1][0] == 7
    y = x.copy()
    y[2, 5] = np.nan  # never drawn
    y[2, :5] = y[2, 6:] = -50.0
    y[2, 11] = 3.0
    st, tok, prob = sample(dev, y, [0.5] * 4)
    assert st == NONFINITE and tok[2] == 11
    y[3] = -np.inf
    st, tok, prob = sample(dev, y[3:], [0.5])
    assert st == NONFINITE and tok[0] == -1 and prob[0] == 0
    for bad in (-1.0, np.nan, np.inf):
        st, tok, prob = sample(dev, x[:1], [0.5], bad)
        assert st == RANGE and tok[0] == x[0].argmax() and prob[0] == 1
    # random numbers outside [0, 1) take the first and the last kept token
    last = np.nonzero(kept_weights(x[0], 1.0, 50, 1.0, 0.0)[0])[0]
    assert [int(sample(dev, x[:1], [u], 1.0, 50)[1][0]) for u in (-3.0, np.nan, 1.0, 7.0)] == [last[0], last[0], last[-1], last[-1]]
    assert sample(dev, x[:1], [0.5], 1e-30)[1][0] == x[0].argmax()
    assert sample(dev, x[:1], [0.9999], 1.0, None, None, 7.0)[1][0] == x[0].argmax()
    L, d = dev.lib, torch.zeros(64, device="cuda")
    for a in ((None, 8, 1, 8, None, ptr(d), ptr(d)), (ptr(d), 7, 1, 8, None, ptr(d), ptr(d)), (ptr(d), 8, 1, 0, None, ptr(d), ptr(d)),
              (ptr(d), 1 << 21, 1, (1 << 20) + 1, None, ptr(d), ptr(d)), (ptr(d), 8, 1, 8, None, None, ptr(d)), (ptr(d), 8, 1, 8, None, ptr(d), None)):
        assert L.ah_sample_dev(dev.h, *a, None, None) == INVALID, a
    assert L.ah_sample_dev(dev.h, None, 8, 0, 8, None, None, None, None, None) == OK
