"""A recurrent layer's operators against plain 64-bit implementations: the short causal convolution and the gated delta
rule, token by token and in chunks.

Tolerances (u = 2^-24, f32's rounding):
  conv   W products and the bias take W + 1 roundings of partial sums, each at most u sum |w x| + |bias|; SiLU's slope is
         at most 1.1, and its own exponential, sum and quotient take under 8 u of the result.
  delta  root mean square, relative to the values: a token's products of dk terms, exponentials and quotients leave about
         (16 + sqrt(dk)) u at random, and with keys of length one and rates up to one no step makes an earlier error
         larger, so that T tokens leave at most sqrt(T) of that.  An output is a sum of dk products q_i S_i, whose
         partial sums are rounded: its errors are relative to m = scale sqrt(sum (q_i S_i)^2), the root mean square of such
         a sum, not to the sum itself, which may all but cancel (one token behind an empty state: every output is a
         multiple of q . k).  A half of f32 lost in any product breaks it (below, on the CPU).  What is compared element
         for element is at most 64 times that from the formula's value, in units of the root mean square.
"""
import ctypes

import numpy as np
import pytest

from apeiron_amd import _lib, chart
from test_gpu_token_ops import CACHE, INVALID, NONFINITE, OK, U, cuda, dev, ptr, stream  # noqa: F401

torch = pytest.importorskip("torch")


def starts(qs):
    return np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)


# ---- the convolution --------------------------------------------------------------------------------


def conv_reference(x, w, bias, silu, qs, src, dst, state):
    state, out, mag = state.astype(np.float64), np.zeros(x.shape), np.zeros(x.shape)
    old, W = state.copy(), w.shape[1]
    for s, (a, n) in enumerate(zip(starts(qs), qs)):
        rows = np.concatenate([old[src[s]] if src[s] >= 0 else np.zeros_like(old[0]), x[a:a + n].astype(np.float64)])
        for t in range(n):
            out[a + t] = (rows[t:t + W] * w.T).sum(0) + (0 if bias is None else bias)
            mag[a + t] = (np.abs(rows[t:t + W] * w.T)).sum(0) + (0 if bias is None else np.abs(bias))
        if dst[s] >= 0:
            state[dst[s]] = rows[n:]
    return out / (1 + np.exp(-out)) if silu else out, mag, state


def conv(d, x, w, bias, silu, qs, src, dst, state, *, pad=0, start=None, max_q=None, st=None):
    n, C = x.shape
    dx = torch.full((n, C + pad), 5.0, device="cuda")
    dx[:, :C] = cuda(x)
    y = torch.full((n, C + pad), 7.0, device="cuda")
    ds, dw, db = cuda(state), cuda(w), None if bias is None else cuda(bias)
    arrays = cuda(starts(qs) if start is None else start), cuda(np.asarray(src, np.int32)), cuda(np.asarray(dst, np.int32))
    chart.conv_dev(d, ptr(dx), ptr(y), n_channels=C, width=w.shape[1], weight_ptr=ptr(dw), bias_ptr=ptr(db), silu=silu, state_ptr=ptr(ds), n_seq=len(qs),
                   n_tok=n, max_q=max(qs) if max_q is None else max_q, n_slots=len(state), q_start_ptr=ptr(arrays[0]), from_ptr=ptr(arrays[1]),
                   to_ptr=ptr(arrays[2]), x_stride=C + pad, y_stride=C + pad, stream=stream() if st is None else st)
    status = d.sync_status(stream() if st is None else st)
    assert (y[:, C:] == 7).all()
    return status, y[:, :C].cpu().numpy(), ds.cpu().numpy()


CONV_SEQS = {"one": ([1], [0], [0]), "begins": ([5], [-1], [1]), "dropped": ([2], [0], [-1]), "long": ([200], [0], [2]),
             "batch": ([1] * 9, list(range(9)), list(range(9))), "ragged": ([33, 0, 1, 64, 2, 3, 129, 0], [4, 5, -1, 0, 0, 1, 2, -1], [4, 8, 9, 10, 11, 1, 2, 12]),
             "even": ([40] * 6, [5, 4, -1, 3, 2, 1], [6, 7, 8, 9, 10, -1])}


@pytest.mark.gpu
@pytest.mark.parametrize("C,W,pad", [(1, 4, 0), (3, 2, 1), (64, 4, 0), (1024, 3, 4), (1025, 4, 3), (130, 8, 0), (2050, 5, 2)])
@pytest.mark.parametrize("seqs", CONV_SEQS)
def test_conv_matches_f64(dev, C, W, pad, seqs):  # noqa: F811
    qs, src, dst = CONV_SEQS[seqs]
    rng = np.random.default_rng(C * W + len(qs))
    f32 = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    x, w, bias, state = f32(sum(qs), C), f32(C, W), f32(C) if C % 2 else None, f32(13, W - 1, C)
    for silu in (True, False):
        status, y, kept = conv(dev, x, w, bias, silu, qs, src, dst, state, pad=pad)
        ref, mag, want = conv_reference(x, w, bias, silu, qs, src, dst, state)
        assert status == OK
        assert (np.abs(y - ref) <= 1.1 * (W + 1) * U * mag + 8 * U * np.abs(ref)).all()
        assert np.array_equal(kept, want.astype(np.float32))


@pytest.mark.gpu
def test_conv_in_parts_is_bit_for_bit_the_whole(dev):  # noqa: F811
    rng = np.random.default_rng(1)
    x, w, state = (rng.standard_normal(s).astype(np.float32) for s in ((150, 70), (70, 4), (1, 3, 70)))
    _, whole, last = conv(dev, x, w, None, True, [150], [0], [0], state)
    at, s = 0, state
    for n in (1, 1, 2, 37, 3, 64, 42):
        _, y, s = conv(dev, x[at:at + n], w, None, True, [n], [0], [0], s)
        assert np.array_equal(y, whole[at:at + n])
        at += n
    assert np.array_equal(s, last)


@pytest.mark.gpu
def test_conv_out_of_range_and_not_finite(dev):  # noqa: F811
    rng = np.random.default_rng(2)
    qs, src, dst = [40, 3, 70, 1], [0, 1, 2, 3], [0, 1, 2, 3]
    x, w, state = (rng.standard_normal(s).astype(np.float32) for s in ((114, 66), (66, 4), (4, 3, 66)))
    status, good, kept = conv(dev, x, w, None, True, qs, src, dst, state)
    assert status == OK
    first = starts(qs)
    for change, bad in (({"src": [0, 4, 2, 3]}, [1]), ({"dst": [0, 1, 2 ** 31 - 1, 3]}, [2]), ({"max_q": 64}, [2]),
                        ({"start": np.array([0, -3, 43, 113, 114], np.int32)}, [0, 1]), ({"start": np.array([0, 40, 43, 113, 115], np.int32)}, [3])):
        a = {"src": src, "dst": dst} | change
        status, y, s = conv(dev, x, w, None, True, qs, a.pop("src"), a.pop("dst"), state, **a)
        assert status == CACHE, change
        for i in range(4):
            rows = slice(first[i], first[i + 1])
            assert (y[rows] == 7).all() if i in bad else np.array_equal(y[rows], good[rows]), (change, i)
            assert np.array_equal(s[i], state[i] if i in bad else kept[i]), (change, i)
    # a value that is not finite reaches its own channel's next tokens alone
    for v in (np.nan, np.inf):
        z = x.copy()
        z[50, 9] = v
        status, y, _ = conv(dev, z, w, None, True, qs, src, dst, state)
        same = np.ones(y.shape, bool)
        same[50:54, 9] = False
        assert status == NONFINITE and np.array_equal(y[same], good[same])
    assert conv(dev, x, w, None, True, qs, src, dst, state)[0] == OK


# ---- the gated delta rule -----------------------------------------------------------------------------


def delta_reference(q, k, v, a, b, A, dt, scale, eps, qs, src, dst, state, lose=None):
    """f64; lose: rounds the factors of the products with S (to show what a lost half costs)."""
    q, k, v, a, b = (x.astype(np.float64) for x in (q, k, v, a, b))
    lose = lose or (lambda x: x)
    r = v.shape[1] // q.shape[1]
    if eps >= 0:
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + eps) for x in (q, k))
    q, k = np.repeat(q, r, 1), np.repeat(k, r, 1)
    if A is not None:
        a = -np.exp(A.astype(np.float64)) * np.logaddexp(a + dt, 0)
        b = 1 / (1 + np.exp(-b))
    old, state, out, mag = state.astype(np.float64), state.astype(np.float64), np.zeros(v.shape), np.zeros(v.shape)
    for s, (at, n) in enumerate(zip(starts(qs), qs)):
        S = old[src[s]].copy() if src[s] >= 0 else np.zeros_like(old[0])
        for t in range(at, at + n):
            S *= np.exp(a[t])[:, None, None]
            u = b[t][:, None] * (v[t] - np.einsum("hkv,hk->hv", lose(S), lose(k[t])))
            S += k[t][:, :, None] * u[:, None, :]
            out[t] = np.einsum("hkv,hk->hv", lose(S), lose(q[t])) * scale
            mag[t] = np.sqrt(np.einsum("hkv,hk->hv", S * S, q[t] ** 2)) * scale
        if dst[s] >= 0:
            state[dst[s]] = S
    return out, state, mag


class Rule:
    """Inputs of a call: heads H over K of dk by dv; kind: how the keys, gates and decays lie."""

    def __init__(self, qs, K, H, dk, dv, seed=0, kind="plain", slots=0):
        rng = np.random.default_rng(seed)
        f32 = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        n = sum(qs)
        self.qs, self.scale, self.eps = qs, dk ** -0.5, 1e-6
        self.q, self.k, self.v, self.a, self.b = f32(n, K, dk), f32(n, K, dk), f32(n, H, dv), f32(n, H), f32(n, H)
        self.A, self.dt = rng.uniform(0, 2.7, H).astype(np.float32), rng.uniform(-6, -2, H).astype(np.float32)
        self.state = f32(max(slots, 1), H, dk, dv)
        if kind == "alike":  # keys near each other, rates near one, hardly any decay
            self.k = (self.k[:1] + 0.05 * self.k).astype(np.float32)
            self.b += 4
            self.dt -= 6
        if kind == "given":  # decays and rates themselves; keys of any length up to one
            self.A = self.dt = None
            self.a, self.b = -rng.exponential(0.3, (n, H)).astype(np.float32), rng.uniform(0, 1, (n, H)).astype(np.float32)
            self.eps = -1.0
            self.k /= 1.5 * np.sqrt(dk, dtype=np.float32)
            self.k /= np.maximum(1, np.sqrt((self.k ** 2).sum(-1, keepdims=True)))
        if kind == "strong":  # decays that forget everything, at once or in a few tokens, and none at all
            self.A = self.dt = None
            self.a = rng.choice([0.0, -1e-3, -3.0, -80.0, -1e4, -np.inf], (n, H), p=[.3, .3, .2, .1, .05, .05]).astype(np.float32)
            self.b = rng.choice([0.0, 0.5, 1.0], (n, H)).astype(np.float32)
        if kind == "large":  # values and states far from one, differently for every head
            f = np.exp2(rng.integers(-40, 40, H)).astype(np.float32)
            self.v *= f[:, None]
            self.state *= f[:, None, None]
            self.q *= np.float32(2.0 ** 30)
            self.k *= np.float32(2.0 ** -20)
            self.eps = 1e-30

    def reference(self, src, dst, lose=None):
        return delta_reference(self.q, self.k, self.v, self.a, self.b, self.A, self.dt, self.scale, self.eps, self.qs, src, dst, self.state, lose)

    def __call__(self, d, src, dst, *, pad=0, start=None, max_q=None, st=None):
        n, K, dk = self.q.shape
        H, dv = self.v.shape[1:]

        def rows(x):
            y = torch.full((n, x[0].size if n else 1) if not pad else (n, x[0].size + pad), 5.0, device="cuda")
            y[:, : y.shape[1] - pad] = cuda(x.reshape(n, -1))
            return y

        q, k, v, a, b = (rows(x) for x in (self.q, self.k, self.v, self.a, self.b))
        out, ds = torch.full((n, H * dv + pad), 7.0, device="cuda"), cuda(self.state)
        A, dt = (None if x is None else cuda(x) for x in (self.A, self.dt))
        i32 = lambda x: cuda(np.asarray(x, np.int32))  # noqa: E731
        arrays = i32(starts(self.qs) if start is None else start), i32(src), i32(dst)
        s = stream() if st is None else st
        chart.delta_rule_dev(d, ptr(q), ptr(k), ptr(v), ptr(a), ptr(b), ptr(out), n_heads=H, n_k_heads=K, k_dim=dk, v_dim=dv, scale=self.scale, norm_eps=self.eps,
                             a_log_ptr=ptr(A), dt_bias_ptr=ptr(dt), state_ptr=ptr(ds), n_seq=len(self.qs), n_tok=n, max_q=max(self.qs) if max_q is None else max_q,
                             n_slots=len(self.state), q_start_ptr=ptr(arrays[0]), from_ptr=ptr(arrays[1]), to_ptr=ptr(arrays[2]), q_stride=K * dk + pad,
                             k_stride=K * dk + pad, v_stride=H * dv + pad, a_stride=H + pad, b_stride=H + pad, out_stride=H * dv + pad, stream=s)
        status = d.sync_status(s)
        assert (out[:, H * dv:] == 7).all()
        return status, out[:, : H * dv].reshape(n, H, dv).cpu().numpy(), ds.cpu().numpy()


def delta_bound(dk, tokens):
    return U * (16 + np.sqrt(dk)) * np.sqrt(max(tokens, 1))


def close(got, ref, tol, per=(), mag=None):
    """Root mean square and element for element, for every index of the axes `per` by itself, in units of mag (ref itself)."""
    mag = ref if mag is None else mag
    for at in np.ndindex(*(got.shape[i] for i in per)):
        i = [slice(None)] * got.ndim
        for axis, j in zip(per, at):
            i[axis] = j
        g, r, m = got[tuple(i)].astype(np.float64), ref[tuple(i)], mag[tuple(i)]
        size = np.sqrt((m * m).mean()) if r.size else 0.0
        assert np.sqrt(((g - r) ** 2).mean()) <= tol * size if r.size else True, (at, np.sqrt(((g - r) ** 2).mean()) / max(size, 1e-300), tol)
        assert (np.abs(g - r) <= 64 * tol * np.maximum(size, np.abs(r))).all(), (at, (np.abs(g - r) / max(size, 1e-300)).max(), tol)


RAGGED = [65, 0, 1, 64, 130, 2, 63, 17, 200], [3, 5, -1, 0, 0, 1, 2, -1, 4], [3, 6, 7, 8, 9, 1, 2, -1, 10]
DELTA_SEQS = {"one": ([1], [0], [0]), "begins": ([1], [-1], [0]), "few": ([3, 1, 2], [0, -1, 2], [0, 1, 2]), "batch": ([1] * 20, list(range(20)), list(range(20))),
              "chunk": ([64], [0], [1]), "over": ([65], [0], [0]), "long": ([500], [-1], [0]), "even": ([100] * 4, [0, -1, 2, 3], [4, 5, 6, -1]), "ragged": RAGGED}


@pytest.mark.gpu
@pytest.mark.parametrize("K,H,dk,dv", [(1, 1, 64, 64), (2, 4, 128, 128), (3, 3, 64, 128), (2, 2, 128, 64), (1, 3, 128, 256), (1, 2, 64, 256)])
@pytest.mark.parametrize("seqs", DELTA_SEQS)
def test_delta_rule_matches_f64(dev, K, H, dk, dv, seqs):  # noqa: F811
    qs, src, dst = DELTA_SEQS[seqs]
    R = Rule(qs, K, H, dk, dv, seed=dk + H + len(qs), slots=20)
    status, out, state = R(dev, src, dst, pad=4 * (dv == 128))
    ref, want, mag = R.reference(src, dst)
    assert status == OK
    tol = delta_bound(dk, max(qs))
    close(out, ref, tol, per=(1,), mag=mag)
    close(state, want, tol, per=(0, 1))
    untouched = [i for i in range(20) if i not in dst]
    assert np.array_equal(state[untouched], R.state[untouched])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["alike", "given", "strong", "large"])
@pytest.mark.parametrize("qs", [[1, 1, 1], [7, 300, 64], [129, 128, 127]])
def test_delta_rule_of_unusual_inputs(dev, kind, qs):  # noqa: F811
    R = Rule(qs, 2, 4, 128, 128, seed=len(kind), kind=kind, slots=3)
    status, out, state = R(dev, [0, 1, -1], [0, 1, 2])
    ref, want, mag = R.reference([0, 1, -1], [0, 1, 2])
    assert status == OK
    tol = delta_bound(128, max(qs))
    close(out, ref, tol, per=(1,), mag=mag)
    close(state, want, tol, per=(0, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [1, 2, 3])
def test_delta_rule_of_rows_off_the_16_byte_grid(dev, pad):  # noqa: F811
    qs = [70, 1, 131]
    R = Rule(qs, 1, 2, 64, 64, seed=pad, slots=3)
    status, out, state = R(dev, [0, 1, 2], [2, -1, 0], pad=pad)
    ref, want, mag = R.reference([0, 1, 2], [2, -1, 0])
    assert status == OK
    close(out, ref, delta_bound(64, 131), per=(1,), mag=mag)
    close(state, want, delta_bound(64, 131), per=(0, 1))


@pytest.mark.gpu
def test_delta_rule_is_the_same_each_time_in_any_batch_and_on_any_stream(dev):  # noqa: F811
    qs = [150, 1, 64, 33]
    R = Rule(qs, 2, 2, 128, 128, seed=9, slots=8)
    _, out, state = R(dev, [0, 1, 2, 3], [4, 5, 6, 7])
    side = torch.cuda.Stream()
    for st in (None, side.cuda_stream):
        torch.cuda.synchronize()
        status, o, s = R(dev, [0, 1, 2, 3], [4, 5, 6, 7], st=st)
        assert status == OK and np.array_equal(o, out) and np.array_equal(s, state)
    for i, at in enumerate(starts(qs)[:-1]):  # a sequence by itself
        one = Rule([qs[i]], 2, 2, 128, 128, slots=8)
        rows = slice(at, at + qs[i])
        one.q, one.k, one.v, one.a, one.b, one.A, one.dt, one.state = R.q[rows], R.k[rows], R.v[rows], R.a[rows], R.b[rows], R.A, R.dt, R.state
        _, o, s = one(dev, [i], [4 + i])
        ref, want, mag = one.reference([i], [4 + i])
        close(o, ref, delta_bound(128, qs[i]), per=(1,), mag=mag)
        close(s, want, delta_bound(128, qs[i]), per=(0, 1))


def on_the_gpu(R, src, dst):
    """R.reference for thousands of tokens: the same steps in f64 tensors of the GPU."""
    f = lambda x: cuda(x).double()  # noqa: E731
    q, k, v, a, b, state = f(R.q), f(R.k), f(R.v), f(R.a), f(R.b), f(R.state)
    r = v.shape[1] // q.shape[1]
    q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + R.eps) for x in (q, k))
    q, k = q.repeat_interleave(r, 1), k.repeat_interleave(r, 1)
    keep, b = torch.exp(-torch.exp(f(R.A)) * torch.nn.functional.softplus(a + f(R.dt))), torch.sigmoid(b)
    out, mag, old = torch.zeros_like(v), torch.zeros_like(v), state.clone()
    for s, (at, n) in enumerate(zip(starts(R.qs), R.qs)):
        S = old[src[s]].clone() if src[s] >= 0 else torch.zeros_like(old[0])
        for t in range(at, at + n):
            S *= keep[t, :, None, None]
            u = b[t, :, None] * (v[t] - (S * k[t, :, :, None]).sum(1))
            S += k[t, :, :, None] * u[:, None, :]
            o = S * q[t, :, :, None]
            out[t], mag[t] = o.sum(1) * R.scale, torch.sqrt((o * o).sum(1)) * R.scale
        if dst[s] >= 0:
            state[dst[s]] = S
    return out.cpu().numpy(), state.cpu().numpy(), mag.cpu().numpy()


# (heads of q and k, heads, k_dim, v_dim, tokens; the arrays' rows): sequences whose chunks' blocks come to 192 MB and more
LONG = [(8, 16, 128, 128, [5700], 5700), (8, 8, 128, 128, [5610, 5610], 11220), (8, 8, 128, 128, [5600, 90], 11200), (16, 32, 64, 64, [5200], 5200),
        (4, 8, 64, 256, [12700], 12700), (4, 16, 128, 128, [130], 8000)]


@pytest.mark.gpu
@pytest.mark.parametrize("K,H,dk,dv,qs,rows", LONG)
def test_delta_rule_of_long_sequences(dev, K, H, dk, dv, qs, rows):  # noqa: F811
    """Chunks in groups; rows behind the last sequence, in a batch that could be even, stay as they were."""
    n, longest = sum(qs), max(rows // len(qs), max(qs))
    R = Rule([rows], K, H, dk, dv, seed=rows, slots=4)
    src, dst = ([3], [0]) if len(qs) == 1 else ([1, -1], [1, 0])  # (the first of two in place)
    R.qs = qs
    status, out, state = R(dev, src, dst, max_q=longest)
    assert status == OK and (out[n:] == 7).all()
    ref, want, mag = on_the_gpu(R, src, dst)
    close(out[:n], ref[:n], delta_bound(dk, max(qs)), per=(1,), mag=mag[:n])
    close(state, want, delta_bound(dk, max(qs)), per=(0, 1))
    if len(qs) == 2:  # one of them out of range: the other as before
        first, second = slice(0, qs[0]), slice(qs[0], n)
        for a, b, good, bad, slot, left in (([4, -1], dst, second, first, 0, 1), (src, [1, 4], first, second, 1, 0)):
            status, o, s = R(dev, a, b, max_q=longest)
            assert status == CACHE and np.array_equal(o[good], out[good]) and (o[bad] == 7).all()
            assert np.array_equal(s[slot], state[slot]) and np.array_equal(s[left], R.state[left])
        x = R.v.copy()
        R.v[qs[0] - 70, 2, 5] = np.nan  # (in the first's last chunks: its earlier outputs and the other's are as before)
        status, o, s = R(dev, src, dst, max_q=longest)
        R.v = x
        same = np.ones(o.shape, bool)
        same[(qs[0] - 70) // 64 * 64:qs[0], 2] = False
        assert status == NONFINITE and np.array_equal(o[same], out[same]) and np.array_equal(s[0], state[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (64, 256), (128, 64)])
@pytest.mark.parametrize("H,qs", [(64, [24, 25, 90, 1, 130, 0, 65, 24, 2]), (64, [25] * 8), (64, [24] * 8), (48, [16, 17, 3, 100, 15, 1]), (3, [1] * 40 + [70, 1, 1, 9, 66, 8]), (4, [1] * 100 + [70] + [2, 0] * 30 + [130, 17, 90] + [1] * 70 + [65]), (2, [33] * 70 + [1, 200])])
def test_delta_rule_of_many_heads(dev, dk, dv, H, qs):  # noqa: F811
    """The lengths around which sequences go by tokens or by chunks, the chain's wider columns, many single tokens."""
    R = Rule(qs, H // 3 if H % 3 == 0 else H // 2, H, dk, dv, seed=H + dk, slots=len(qs) + 2)
    src, dst = [i if i % 3 else -1 for i in range(len(qs))], [i if i % 5 else -1 for i in range(len(qs))]
    status, out, state = R(dev, src, dst)
    ref, want, mag = on_the_gpu(R, src, dst)
    assert status == OK
    close(out, ref, delta_bound(dk, max(qs)), mag=mag)
    close(state, want, delta_bound(dk, max(qs)))


@pytest.mark.gpu
def test_a_group_of_chunks_replayed_as_a_graph(dev):  # noqa: F811
    """A long sequence captured: what passes from launch to launch in the scratch is made anew by every replay."""
    d2, n, H = chart.Device(0), 5700, 16
    rng = np.random.default_rng(2)
    f32 = lambda *s: cuda(rng.standard_normal(s).astype(np.float32))  # noqa: E731
    x, ab, out, state = f32(n, 3 * H * 128), f32(n, 2 * H), torch.zeros(n, H * 128, device="cuda"), f32(2, H, 128, 128)
    gate, kept, i = (f32(H), f32(H) - 4), state.clone(), cuda(np.array([0, n, 0, 1], np.int32))

    def run(d):
        chart.delta_rule_dev(d, ptr(x), ptr(x) + 4 * H * 128, ptr(x) + 8 * H * 128, ptr(ab), ptr(ab) + 4 * H, ptr(out), n_heads=H, n_k_heads=H, k_dim=128, v_dim=128,
                             a_log_ptr=ptr(gate[0]), dt_bias_ptr=ptr(gate[1]), scale=0.1, norm_eps=1e-6, state_ptr=ptr(state), q_stride=3 * H * 128, k_stride=3 * H * 128,
                             v_stride=3 * H * 128, a_stride=2 * H, b_stride=2 * H, n_seq=1, n_tok=n, max_q=n, n_slots=2, q_start_ptr=ptr(i), from_ptr=ptr(i) + 8,
                             to_ptr=ptr(i) + 8, stream=stream())

    want = []
    for _ in range(3):
        run(dev)
        torch.cuda.synchronize()
        want.append((out.clone(), state.clone()))
    state.copy_(kept)
    run(d2)
    torch.cuda.synchronize()
    state.copy_(kept)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(d2)
    state.copy_(kept)
    other = Rule([300, 200], 2, 4, 128, 128, seed=3, slots=2)
    for o, s in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, o) and torch.equal(state, s)
        out.zero_()
        assert other(d2, [0, 1], [0, 1])[0] == OK
    assert d2.sync_status(stream()) == OK
    d2.close()


@pytest.mark.gpu
def test_delta_rule_out_of_range_and_not_finite(dev):  # noqa: F811
    qs, src, dst = [70, 3, 129, 1], [0, 1, 2, 3], [0, 1, 2, 3]
    R = Rule(qs, 1, 2, 64, 64, seed=4, slots=4)
    status, good, kept = R(dev, src, dst)
    assert status == OK
    first = starts(qs)
    for change, bad in (({"src": [0, 4, 2, 3]}, [1]), ({"dst": [0, 1, 2 ** 31 - 1, 3]}, [2]), ({"max_q": 100}, [2]), ({"start": [0, -3, 73, 202, 203]}, [0, 1]),
                        ({"start": [0, 70, 73, 202, 204]}, [3]), ({"start": [0, 2 ** 31 - 1, 73, 202, 203]}, [0, 1]), ({"start": [-2 ** 31, 70, 73, 202, 203]}, [0])):
        a = {"src": src, "dst": dst} | change
        status, o, s = R(dev, a.pop("src"), a.pop("dst"), **a)
        assert status == CACHE, change
        for i in range(4):
            rows = slice(first[i], first[i + 1])
            assert (o[rows] == 7).all() if i in bad else np.array_equal(o[rows], good[rows]), (change, i)
            assert np.array_equal(s[i], R.state[i] if i in bad else kept[i]), (change, i)
    # a value that is not finite: its head's later tokens alone, and the chunk of 64 that it stands in
    for name, at in (("v", (180, 1, 7)), ("a", (180, 1)), ("b", (180, 1))):
        x = getattr(R, name)
        for value in (np.nan, np.inf):
            z = x.copy()
            z[at] = value
            setattr(R, name, z)
            status, o, s = R(dev, src, dst)
            setattr(R, name, x)
            if value == np.inf and name == "b":  # (a rate of one)
                assert status == OK
                continue
            same = np.ones(o.shape, bool)
            same[73 + 64:202, 1] = False
            assert status == NONFINITE or (value == np.inf and name == "a")
            assert np.array_equal(o[same], good[same]) and np.array_equal(s[[0, 1, 3]], kept[[0, 1, 3]]) and np.array_equal(s[2, 0], kept[2, 0]), (name, value)
    assert R(dev, src, dst)[0] == OK


@pytest.mark.gpu
def test_state_operators_replayed_as_a_graph(dev):  # noqa: F811
    """A recurrent layer's step and a chunk of its prompt captured: every replay, with eager calls of other sizes
    between, carries the states on as eager calls do."""
    d2 = chart.Device(0)
    K, H, dk, dv = 2, 4, 128, 128
    C = 2 * K * dk + H * dv
    for qs in ([1, 1, 1], [150, 1, 70]):
        n, S = sum(qs), len(qs)
        rng = np.random.default_rng(n)
        f32 = lambda *s: cuda(rng.standard_normal(s).astype(np.float32))  # noqa: E731
        x, w, ab, A, dt = f32(n, C), f32(C, 4) * 0.5, f32(n, 2 * H), f32(H), f32(H) - 4
        i32 = lambda v: cuda(np.asarray(v, np.int32))  # noqa: E731
        start, slots = i32(starts(qs)), i32(range(S))
        y, out, tail, state = torch.zeros(n, C, device="cuda"), torch.zeros(n, H * dv, device="cuda"), f32(S, 3, C), f32(S, H, dk, dv)
        kept = tail.clone(), state.clone()

        def step(d):
            seqs = dict(n_seq=S, n_tok=n, max_q=max(qs), n_slots=S, q_start_ptr=ptr(start), from_ptr=ptr(slots), to_ptr=ptr(slots), stream=stream())
            chart.conv_dev(d, ptr(x), ptr(y), n_channels=C, width=4, weight_ptr=ptr(w), silu=True, state_ptr=ptr(tail), **seqs)
            chart.delta_rule_dev(d, ptr(y), ptr(y) + 4 * K * dk, ptr(y) + 8 * K * dk, ptr(ab), ptr(ab) + 4 * H, ptr(out), n_heads=H, n_k_heads=K, k_dim=dk, v_dim=dv,
                                 a_log_ptr=ptr(A), dt_bias_ptr=ptr(dt), scale=dk ** -0.5, norm_eps=1e-6, state_ptr=ptr(state), q_stride=C, k_stride=C, v_stride=C,
                                 a_stride=2 * H, b_stride=2 * H, **seqs)

        want = []
        for _ in range(4):
            step(dev)
            torch.cuda.synchronize()
            want.append((out.clone(), tail.clone(), state.clone()))
        tail.copy_(kept[0]), state.copy_(kept[1])
        step(d2)  # grows the scratch
        torch.cuda.synchronize()
        tail.copy_(kept[0]), state.copy_(kept[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(d2)
        tail.copy_(kept[0]), state.copy_(kept[1])
        big = Rule([700, 300], 2, 4, 128, 128, seed=3, slots=2)
        for o, t, s in want:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, o) and torch.equal(tail, t) and torch.equal(state, s)
            out.zero_()
            assert big(d2, [0, 1], [0, 1])[0] == OK
    d2.close()


@pytest.mark.gpu
def test_state_refusals(dev):  # noqa: F811
    L, z = dev.lib, torch.zeros(4096, device="cuda")
    i = torch.zeros(8, dtype=torch.int32, device="cuda")

    def seqs(**kw):
        return ctypes.byref(_lib.StateSeqs(*(kw.get(n, v) for n, v in (("n_seq", 1), ("n_tok", 1), ("max_q", 1), ("n_slots", 1), ("start", ptr(i)), ("src", ptr(i)),
                                                                       ("dst", ptr(i))))))

    def conv_call(s=None, x=ptr(z), xs=64, y=ptr(z) + 8192, ys=64, **kw):
        c = _lib.Conv(*(kw.get(n, v) for n, v in (("C", 64), ("W", 4), ("w", ptr(z)), ("b", None), ("silu", 1), ("state", ptr(z) + 4096))))
        return L.ah_conv_dev(dev.h, s or seqs(), ctypes.byref(c), x, xs, y, ys, stream())

    assert conv_call() == OK
    for bad in (dict(W=1), dict(W=9), dict(C=1 << 21), dict(w=None), dict(state=None), dict(x=None), dict(y=None), dict(xs=63), dict(ys=63), dict(y=ptr(z)),
                dict(y=ptr(z) + 252), dict(s=seqs(start=None)), dict(s=seqs(src=None)), dict(s=seqs(dst=None)), dict(s=seqs(n_seq=65536)),
                dict(s=seqs(n_tok=1 << 31)), dict(s=seqs(n_slots=1 << 31))):
        assert conv_call(**bad) == INVALID, bad
    assert conv_call(C=0) == OK and conv_call(s=seqs(n_seq=0, start=None)) == OK

    def delta_call(s=None, q=ptr(z), k=ptr(z), v=ptr(z), a=ptr(z), b=ptr(z), out=ptr(z) + 8192, st=(64,) * 6, **kw):
        r = _lib.DeltaRule(*(kw.get(n, v) for n, v in (("H", 1), ("K", 1), ("dk", 64), ("dv", 64), ("A", None), ("dt", None), ("scale", 1.0), ("eps", -1.0),
                                                       ("state", ptr(state)))))
        return L.ah_delta_rule_dev(dev.h, s or seqs(), ctypes.byref(r), q, st[0], k, st[1], v, st[2], a, st[3], b, st[4], out, st[5], stream())

    state = torch.zeros(64 * 64, device="cuda")
    assert delta_call() == OK
    for bad in (dict(dk=32), dict(dk=256), dict(dv=32), dict(dv=96), dict(K=0), dict(H=3, K=2), dict(H=4097), dict(A=ptr(z)), dict(dt=ptr(z)), dict(state=None), dict(q=None),
                dict(k=None), dict(v=None), dict(a=None), dict(b=None), dict(out=None), dict(out=ptr(z)), dict(out=ptr(z) + 128), dict(st=(63, 64, 64, 64, 64, 64)),
                dict(st=(64, 63, 64, 64, 64, 64)), dict(st=(64, 64, 63, 64, 64, 64)), dict(st=(64, 64, 64, 0, 64, 64)), dict(st=(64, 64, 64, 64, 0, 64)),
                dict(st=(64, 64, 64, 64, 64, 63)), dict(s=seqs(start=None)), dict(s=seqs(n_seq=65536))):
        assert delta_call(**bad) == INVALID, bad
    assert delta_call(H=0) == OK and delta_call(s=seqs(n_seq=0, start=None)) == OK
    assert dev.sync_status(stream()) == OK


def test_null_arguments_are_refused_without_a_gpu():
    L, s = _lib.load(), _lib.StateSeqs()
    assert L.ah_conv_dev(None, ctypes.byref(s), ctypes.byref(_lib.Conv()), None, 0, None, 0, None) == INVALID
    assert L.ah_delta_rule_dev(None, ctypes.byref(s), ctypes.byref(_lib.DeltaRule()), *[None, 0] * 6, None) == INVALID
    assert ctypes.sizeof(_lib.StateSeqs) == 7 * 8 and ctypes.sizeof(_lib.Conv) == 6 * 8 and ctypes.sizeof(_lib.DeltaRule) == 8 * 8


@pytest.mark.parametrize("qs", [[1, 3], [200]])
def test_a_lost_half_breaks_the_bound(qs):
    n = len(qs)
    R = Rule(qs, 1, 2, 64, 64, seed=6, slots=n)
    src = list(range(n))
    ref, _, mag = R.reference(src, src)
    err = lambda x: np.sqrt(((x - ref) ** 2).mean() / (mag * mag).mean())  # noqa: E731
    half, single = (R.reference(src, src, lose=lambda x: x.astype(t).astype(np.float64))[0] for t in (np.float16, np.float32))
    assert err(half) > 3 * delta_bound(64, max(qs)) and err(single) < delta_bound(64, max(qs))
