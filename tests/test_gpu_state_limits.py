"""The gated delta rule at the limits of a launch: batches of tens of thousands of sequences, and those that are too large."""
import ctypes

import numpy as np
import pytest

from apeiron_amd import _lib, chart
from test_gpu_state_ops import INVALID, OK, U, dev, ptr, stream  # noqa: F401

torch = pytest.importorskip("torch")


@pytest.mark.gpu
def test_a_chunk_among_tens_of_thousands_of_sequences(dev):  # noqa: F811
    """Idle ones and single tokens.  From an empty state a token's output is scale (q . k) beta v: dk + 4 roundings of the sum of
    |q k|."""
    n_seq, H, dk, dv, long, at = 65535, 9, 64, 256, 70, 30001
    qs = np.zeros(n_seq, np.int64)
    qs[::16], qs[at] = 1, long
    starts = np.concatenate([[0], np.cumsum(qs)])
    n, at = int(starts[-1]), int(starts[at])
    g = torch.Generator("cuda").manual_seed(1)
    q, k = (torch.randn(n, dk, device="cuda", generator=g) / 8 for _ in range(2))
    v, b = torch.randn(n, H * dv, device="cuda", generator=g), torch.rand(n, H, device="cuda", generator=g)
    a = -torch.rand(n, H, device="cuda", generator=g)
    q_start = torch.from_numpy(starts).int().cuda()
    none = torch.full((n_seq,), -1, dtype=torch.int32, device="cuda")
    out, state = torch.full((n, H * dv), 7.0, device="cuda"), torch.zeros(H * dk * dv, device="cuda")
    chart.delta_rule_dev(dev, ptr(q), ptr(k), ptr(v), ptr(a), ptr(b), ptr(out), n_heads=H, n_k_heads=1, k_dim=dk, v_dim=dv, scale=0.5, state_ptr=ptr(state), n_seq=n_seq,
                         n_tok=n, max_q=long, n_slots=1, q_start_ptr=ptr(q_start), from_ptr=ptr(none), to_ptr=ptr(none), stream=stream())
    assert dev.sync_status(stream()) == OK
    first = torch.ones(n, dtype=torch.bool, device="cuda")
    first[at + 1:at + long] = False
    dot, size = (q.double() * k.double()).sum(1), (q * k).abs().double().sum(1)
    for h in range(H):
        w = 0.5 * b[:, h].double()
        got, want = out[:, dv * h:dv * h + dv].double(), (w * dot)[:, None] * v[:, dv * h:dv * h + dv].double()
        off = (got - want).abs() <= ((dk + 4) * U * w * size)[:, None] * v[:, dv * h:dv * h + dv].abs().double()
        assert off[first].all(), h
    S = np.zeros((dk, dv))  # the long one, head 3
    f = lambda x: x[at:at + long].double().cpu().numpy()  # noqa: E731
    Q, K, V, A, Bt, got = f(q), f(k), f(v)[:, 3 * dv:4 * dv], f(a)[:, 3], f(b)[:, 3], f(out)[:, 3 * dv:4 * dv]
    for t in range(long):
        S *= np.exp(A[t])
        S += np.outer(K[t], Bt[t] * (V[t] - K[t] @ S))
        mag = 0.5 * np.sqrt((S * S * Q[t][:, None] ** 2).sum(0))
        assert np.sqrt(((got[t] - 0.5 * Q[t] @ S) ** 2).mean()) <= U * (16 + 8) * np.sqrt(t + 1) * np.sqrt((mag * mag).mean())


@pytest.mark.gpu
def test_more_workgroups_than_a_launch_holds_are_refused(dev):  # noqa: F811
    z, none, zero = torch.zeros(4096, device="cuda"), torch.full((65536,), -1, dtype=torch.int32, device="cuda"), torch.zeros(65536, dtype=torch.int32, device="cuda")
    for n_seq, H, dv, n_tok, max_q in ((65535, 4096, 256, 1, 1), (65535, 257, 128, 1, 1), (65535, 4096, 64, 1 << 20, 1 << 10), (65535, 4096, 64, 65535 * 64, 64)):
        # (sequences without tokens or slots: no row is read; the output's place is no one's)
        s = _lib.StateSeqs(n_seq, n_tok, max_q, 1, ptr(zero), ptr(none), ptr(none))
        r = _lib.DeltaRule(H, 1, 64, dv, None, None, 1.0, -1.0, ptr(z))
        call = dev.lib.ah_delta_rule_dev(dev.h, ctypes.byref(s), ctypes.byref(r), ptr(z), 64, ptr(z), 64, ptr(z), H * dv, ptr(z), H, ptr(z), H, 1 << 46, H * dv, stream())
        assert call == INVALID, (n_seq, H, dv)
    assert dev.sync_status(stream()) == OK
