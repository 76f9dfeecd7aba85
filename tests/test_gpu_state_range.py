"""The recurrent layer's operators over the whole range of their inputs: activations far from zero, rows of very different
lengths in one chunk.

Tolerances (u = 2^-24, f32's rounding):
  SiLU   v / (1 + e^-v): the exponential takes up to 2 u (v_exp_f32's last place) and two roundings, the sum, the quotient's
         product and its Newton step one each: 6 u of the result, and half of f32's smallest number (2^-150), where it is
         below the normal ones.  With a bias of zero and one weight of one the value before it is the input itself.
  delta  as in tests/test_gpu_state_ops.py: a key's or query's own length is no part of the rule where they are divided by it,
         and where they are not, outputs and their tolerance are as long as the query.  So it is held by every token.
         By chunks a token's part of the state, u = beta (v - S^T k), is held to 2^-31 of the largest |S| and 2^-37 of the
         largest |beta v| of its chunk: an output of keys and queries of length one is off by at most scale times that for
         each of up to 64 tokens since a decay that cleared the state, a state's element by that for each.
"""
import numpy as np
import pytest

from test_gpu_state_ops import NONFINITE, OK, Rule, U, close, conv, delta_bound, dev  # noqa: F401

torch = pytest.importorskip("torch")


@pytest.mark.gpu
@pytest.mark.parametrize("qs", [[1] * 40, [40], [9, 1, 30]])
def test_silu_of_any_finite_value(dev, qs):  # noqa: F811
    rng = np.random.default_rng(len(qs))
    C = 130
    x = rng.uniform(-110, 110, (40, C)).astype(np.float32)
    x[0] = rng.uniform(-89, -87, C)
    x[1] = rng.uniform(-75, -68, C)
    edges = [88, 88.73, 89, 100, 104, 126, 128, 130, 1e4, 1e30, 3e38, 3.4028234663852886e38, 2.0 ** -126, 1e-45, 0]
    x[2, :30] = np.float32(edges + [-v for v in edges])
    x[3], x[4] = -np.exp(rng.uniform(0, 88, C)), np.exp(rng.uniform(0, 88, C))
    w = np.zeros((C, 4), np.float32)
    w[:, 3] = 1
    src = list(range(len(qs)))
    status, y, _ = conv(dev, x, w, None, True, qs, src, src, np.zeros((len(qs), 3, C), np.float32))
    v = x.astype(np.float64)
    with np.errstate(over="ignore"):
        ref = v / (1 + np.exp(-v))
    assert status == OK
    assert (np.abs(y - ref) <= 6 * U * np.abs(ref) + 2.0 ** -150).all()


@pytest.mark.gpu
@pytest.mark.parametrize("K,H,dk,dv", [(2, 4, 128, 128), (1, 2, 64, 256), (3, 3, 128, 64)])
@pytest.mark.parametrize("qs", [[1, 1, 1], [9, 8, 10], [7, 300, 64], [129, 128, 127]])
@pytest.mark.parametrize("norm", [True, False])
def test_delta_rule_of_rows_of_very_different_lengths(dev, K, H, dk, dv, qs, norm):  # noqa: F811
    R = Rule(qs, K, H, dk, dv, seed=dk + dv + len(qs), kind="plain" if norm else "given", slots=3)
    rng = np.random.default_rng(sum(qs))
    n = sum(qs)
    if norm:
        R.eps = 1e-30
        R.k *= np.exp2(rng.integers(-32, 33, (n, K, 1))).astype(np.float32)
        R.q *= np.exp2(rng.integers(-32, 33, (n, K, 1))).astype(np.float32)
    else:  # (keys no longer than one)
        R.k *= np.exp2(rng.integers(-24, 1, (n, K, 1))).astype(np.float32)
        R.q *= np.exp2(rng.integers(-32, 33, (n, K, 1))).astype(np.float32)
    status, out, state = R(dev, [0, 1, -1], [0, 1, 2])
    ref, want, mag = R.reference([0, 1, -1], [0, 1, 2])
    assert status == OK
    tol = delta_bound(dk, max(qs))
    close(out, ref, tol, per=(0, 1), mag=mag)
    close(state, want, tol, per=(0, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("qs,at", [([3], 2), ([8, 1], 7), ([64], 63), ([100, 20], 99), ([130], 10)])
def test_a_state_that_leaves_f32_is_refused(dev, qs, at):  # noqa: F811
    """What a token adds, k (beta (v - S^T k))^T, overflows where both factors are finite and no query reads it."""
    R = Rule(qs, 2, 2, 64, 64, seed=1, kind="given", slots=2)
    R.q[:] = 0
    R.a[:], R.b[:] = 0, 1
    src = list(range(len(qs)))
    status, _, good = R(dev, src, src)
    assert status == OK
    R.k[at, 1, 3], R.v[at, 1, 5] = 16, 1e38
    status, out, state = R(dev, src, src)
    assert status == NONFINITE and not np.isfinite(state[0, 1]).all()
    assert np.array_equal(state[0, 0], good[0, 0]) and np.array_equal(state[1:], good[1:]) and (out[:, 0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["q", "k"])
@pytest.mark.parametrize("qs,at", [([3, 2], 1), ([64, 3], 40), ([130, 70], 70)])
def test_rows_whose_squares_leave_f32_are_refused(dev, name, qs, at):  # noqa: F811
    """A row that is divided by its length, the sum of whose squares is not finite in f32: no row of zeros in its place."""
    R = Rule(qs, 2, 2, 64, 64, seed=2, slots=2)
    status, good, kept = R(dev, [0, 1], [0, 1])
    assert status == OK
    x = getattr(R, name).copy()
    for value, expect in ((1e18, OK), (3e19, NONFINITE), (-3e38, NONFINITE)):
        getattr(R, name)[at, 1] = value
        status, out, state = R(dev, [0, 1], [0, 1])
        assert status == expect, value
        same = np.ones(out.shape, bool)
        same[at // 64 * 64:qs[0], 1] = False
        assert np.array_equal(out[same], good[same]) and np.array_equal(state[1], kept[1]) and np.array_equal(state[0, 0], kept[0, 0])
        if expect == OK:
            ref, want, mag = R.reference([0, 1], [0, 1])
            close(out, ref, delta_bound(64, max(qs)), per=(1,), mag=mag)
            close(state, want, delta_bound(64, max(qs)), per=(0, 1))
    getattr(R, name)[:] = x
    assert R(dev, [0, 1], [0, 1])[0] == OK


@pytest.mark.gpu
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64)])
@pytest.mark.parametrize("at", [5, 16, 40])
@pytest.mark.parametrize("shrink", [10, 24])
def test_small_values_behind_a_decay_that_clears_a_large_state(dev, dk, dv, at, shrink):  # noqa: F811
    R = Rule([64], 2, 2, dk, dv, seed=at + shrink, kind="given", slots=1)
    R.eps = 1e-6
    R.a[at] = -np.inf
    R.v[at:] *= np.float32(2.0 ** -shrink)
    status, out, state = R(dev, [0], [0])
    ref, want, mag = R.reference([0], [0])
    assert status == OK
    tol, top = delta_bound(dk, 64), 2.0 ** -31 * np.abs(R.state).max() + 2.0 ** -37 * np.abs(R.v).max()
    close(out[:at], ref[:at], tol, per=(1,), mag=mag[:at])
    size = lambda x, axis: np.sqrt((x * x).mean(axis, keepdims=True))  # noqa: E731
    assert (np.abs(out - ref)[at:] <= 64 * tol * size(mag[at:], 2) + 64 * R.scale * top).all()
    assert (np.abs(state - want) <= 64 * tol * size(want, (2, 3)) + 64 * top).all()
