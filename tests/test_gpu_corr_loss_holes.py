"""Left-out query rows that are not finite, spread over frames of many tiles: the
gradient kernel streams such rows as zeros, decided by row data that is on its way
with the tiles.  Oracle and tolerances of test_gpu_corr_loss.py."""
import numpy as np
import pytest
import torch

from test_gpu_corr_loss import PAIR, TYPES, _check, _problem, _run

pytestmark = pytest.mark.gpu


def _holes(rng, P, rows):
    """A third of the rows, runs and single ones, in every tile."""
    out = rng.random((rows, P)) < 0.2
    out[:, 64:70] = True
    out[:, 200:330] |= rng.random((rows, 130)) < 0.7
    return out


@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("P,Q,D", [(700, 150, 64), (450, 600, 128), (611, 90, 200), (2560, 300, 128)])
@pytest.mark.parametrize("K", [0, 3])
def test_separate_features(K, P, Q, D, dtype, positive):
    dt = TYPES[dtype]
    a, b, f1, f2, idx, logits, g = _problem(P + D, dt, K, 4, 2, P, 2, Q, D)
    f1[:], f2[:] = [0, 1, 0, 1], [0, 1, 1, 0]
    rng = np.random.default_rng(P)
    out = _holes(rng, P, 2)
    idx[idx < 0] = Q - 1 if K == 0 else -1
    for e in range(4):
        idx[e, out[f1[e]]] = -1
    if positive:
        g = np.abs(g)
    hole = torch.from_numpy(out).to(a.device)
    clean = a.clone()
    clean[hole] = 0.0
    a = a.clone()
    a[hole] = float("nan")
    a[hole & (torch.arange(P, device=a.device) % 3 == 0)] = float("inf")
    loss, grads = _run(a, b, f1, f2, idx, logits, g, False, 1 / 16, 1.0)
    _check(dt, clean, b, f1, f2, idx, logits, g, False, 1 / 16, 1.0, loss, grads)
    assert not grads[0][hole].any()


@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("P,D", [(520, 128), (700, 32), (450, 256)])
def test_shared_features(P, D, dtype, positive):
    """Frames 0 and 2 are queries only (the edge back to 0 has no target), 1 and 3
    a pair of their own."""
    dt = TYPES[dtype]
    f1, f2 = np.array([0, 2, 1, 1, 3], np.int32), np.array([1, 1, 0, 3, 1], np.int32)
    a, _, _, _, idx, logits, g = _problem(P, dt, 2, 5, 4, P, 4, P, D, shared=True)
    out = _holes(np.random.default_rng(D), P, 4)
    out[[1, 3]] = False
    for e in range(5):
        idx[e, out[f1[e]]] = -1
    idx[2] = -1
    if positive:
        g = np.abs(g)
    hole = torch.from_numpy(out).to(a.device)
    clean = a.clone()
    clean[hole] = 0.0
    a = a.clone()
    a[hole] = float("nan")
    loss, grads = _run(a, a, f1, f2, idx, logits, g, True, 1 / 16, 1.0)
    _check(dt, clean, clean, f1, f2, idx, logits, g, True, 1 / 16, 1.0, loss, grads, PAIR)
