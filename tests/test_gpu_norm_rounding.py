"""The norm's y is the exact value's nearest f32 number: R and the products are formed in 64 bits and rounded once, so a
code of the quantizer differs from the exact y's only where that lies within half of f32's last place of a boundary."""
import numpy as np
import pytest

from test_gpu_token_ops import OK, dev, norm  # noqa: F401

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_tok,n", [(1, 1), (3, 7), (40, 896), (9, 1531), (5, 8193), (2, 32768)])
@pytest.mark.parametrize("size", [1.0, 1e-12, 1e15])
def test_y_is_rounded_once(dev, n_tok, n, size):  # noqa: F811
    rng = np.random.default_rng(n)
    x = (size * rng.standard_normal((n_tok, n))).astype(np.float32)
    g = (1 + 0.3 * rng.standard_normal(n)).astype(np.float32)
    st, s, y, codes, scales, values = norm(dev, x, None, g, eps=1e-6 * size * size)
    assert st == OK and np.array_equal(s, x)
    v = x.astype(np.longdouble)
    eps = np.longdouble(np.float32(1e-6 * size * size))
    ref = v / np.sqrt((v * v).mean(-1, keepdims=True) + eps) * g.astype(np.longdouble)
    half = np.spacing(np.abs(y)).astype(np.longdouble) / 2
    assert (np.abs(y - ref) <= half * (1 + 2.0 ** -20)).all()
