"""The gradients of the correlation losses are off by the rounding of the result, not by
that of the weights.

The second product takes the weights ds = g (p - pi) in the features' type.  Where a
half tile holds a target they are two numbers of it, so a target's weight, which is
most of a row's, keeps twice the bits (2^-22 or 2^-16: nothing here).  The other
weights are g p, rounded by at most half a step h each, independently: their share of
the error's square is at most sum (h g p)^2 |f|^2.  Bound, in the 2-norm: the root of
the sum of the squares of the rounding of the exact result and twice that share, and
2 % for the fp32 sums (below 2^-17 of their terms).  With weights of one number the
error was 1.2 to 1.45 times the rounding of the result."""
import numpy as np
import pytest
import torch

from gpu_util import host
from oracle import corr_loss as oc
from test_gpu_corr_loss import TYPES, _problem, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shared,sign", [(False, True), (True, True), (True, False)])
@pytest.mark.parametrize("K,P,Q,D", [(0, 700, 700, 128), (4, 450, 450, 64), (16, 330, 330, 200), (1, 520, 520, 32)])
def test_error_is_that_of_the_result(K, P, Q, D, shared, sign, dtype):
    dt = TYPES[dtype]
    a, b, f1, f2, idx, logits, g = _problem(P + K, dt, K, 4, 3, P, 3, Q, D, shared=shared)
    f1[:], f2[:] = [0, 1, 2, 0], [1, 0, 1, 2]      # one edge and its reverse
    if not sign:
        g = np.abs(g)
    loss, grads = _run(a, b, f1, f2, idx, logits, g, shared, 1 / 16, 1.0)
    A, B, h = host(a.double()), host(b.double()), torch.finfo(dt).eps / 2
    _, d1, d2, per_edge = oc.corr_loss(A, B, f1, f2, idx, logits, 1 / 16, 1.0, g)
    share = [0.0, 0.0]
    for e, (_, p, q, _) in enumerate(per_edge):
        w = np.where(q.max(1, keepdims=True) > 0, h * np.abs(g[e])[:, None] * p / 16, 0.0) ** 2
        share[0] += (w @ (B[f2[e]] ** 2).sum(1)).sum()
        share[1] += (w.T @ (A[f1[e]] ** 2).sum(1)).sum()
    if shared:
        d1, share = d1 + d2, [sum(share)]
    for got, want, s in zip(grads, (d1, d2), share):
        own = host(torch.from_numpy(want).to(dt).double()) - want
        off = host(got.double()) - want
        bound = 1.02 * np.sqrt((own ** 2).sum() + 4 * s)
        assert np.sqrt((off ** 2).sum()) <= bound, np.sqrt((off ** 2).sum() / (own ** 2).sum())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K,T", [(0, 1.0), (1, 1.0), (2, 2.0)])
def test_small_losses_of_large_logits(K, T, dtype):
    """Each row's target is its own copy among the keys, the features small whole
    numbers: all products and their sums are exact in fp32, the logits about 1000 and
    the losses next to nothing.  What is left: at most Q + 8 roundings of a sum that is
    2^(half a step of the largest logit), and as many units for the hardware's
    exponential and logarithm: T^2 (Q + 16) 2^-24; roundings of the logits or of lse
    themselves would be 6e-5 each."""
    dt = TYPES[dtype]
    rng = np.random.default_rng(K)
    a = torch.from_numpy(rng.integers(-3, 4, (2, 150, 128))).to(dt).to("cuda:0")
    f = np.array([0, 1], np.int32)
    idx = np.zeros((2, 150, max(1, K)), np.int32)
    idx[..., 0] = np.arange(150)
    logits = np.zeros(idx.shape, np.float32) if K else None
    if K == 2:
        idx[..., 1], logits[..., 1] = 7, -np.inf
    g = np.ones((2, 150), np.float32)
    loss, _ = _run(a, a.clone(), f, f, idx, logits, g, False, 2.0, T)
    want = oc.corr_loss(host(a.double()), host(a.double()), f, f, idx, logits, 2.0, T)
    off = np.abs(host(loss.double()) - want)
    assert off.max() <= T * T * (150 + 16) * 2.0 ** -24, off.max()
