"""The correlation losses' gradients over the range of upstream gradients, checked
whatever comes out.  Oracle and tolerances of test_gpu_corr_loss.py."""
import numpy as np
import pytest
import torch

from gpu_util import host
from oracle import corr_loss as oc
from test_gpu_corr_loss import TYPES, _check, _problem, _run

pytestmark = pytest.mark.gpu


def _peaked(dt, gscale):
    """p near 1 at the target of most rows: the gradient is the small p - 1."""
    a, b, f1, f2, idx, _, g = _problem(5, dt, 0, 2, 2, 100, 2, 150, 128, gscale=gscale)
    b = b.clone()
    for e in range(2):
        for r in range(100):
            if idx[e, r, 0] >= 0 and f1[e] == 0:
                idx[e, r, 0] = r
    b[:, :100] = a[:1]
    return a, b, f1, f2, idx, None, g


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("gscale", [1e-7, 1e-3, 1.0, 1e3, 1e4])
def test_gradients_that_fit_the_type(dtype, gscale):
    dt = TYPES[dtype]
    p = _peaked(dt, gscale)
    a, b, f1, f2, idx, _, g = p
    _, d1, d2, _ = oc.corr_loss(host(a.double()), host(b.double()), f1, f2, idx, None, 1 / 16, 1.0, g)
    fits = max(np.abs(d1).max(), np.abs(d2).max()) < 0.9 * torch.finfo(dt).max
    assert fits or (dtype, gscale) == ("fp16", 1e4)
    loss, grads = _run(*p, False, 1 / 16, 1.0)
    assert torch.isfinite(loss).all()
    if fits:
        assert all(torch.isfinite(t).all() for t in grads)
        _check(dt, *p, False, 1 / 16, 1.0, loss, grads)


@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("shared", [False, True])
def test_upstream_gradients_times_a_power_of_two(shared, positive):
    """fp16 weights are scaled by a power of two a frame, so a loss scale of 2^k gives
    2^k times the result, infinite only past the type's range.  Not bit for bit: a
    streamed row's exponent log2 |g| - lse is rounded in fp32 with the scale in it
    (2^-24 of at most 60 + |lse|), so a weight may round to its other neighbour: eps
    of its value, and the sum by eps of the terms' sizes, then one rounding on each side."""
    dt, k = torch.float16, 18
    p = list(_peaked(dt, 1.0))
    if shared:
        p[1] = p[0]
        p[4] = np.minimum(p[4], 99)
    if positive:
        p[-1] = np.abs(p[-1])
    _, small = _run(*p, shared, 1 / 16, 1.0)
    a, b, f1, f2, idx, _, g = p
    A, B, eps = host(a.double()), host(b.double()), torch.finfo(dt).eps
    size = [np.zeros_like(A), np.zeros_like(A if shared else B)]
    for e, (ds, _, _, _) in enumerate(oc.corr_loss(A, B, f1, f2, idx, None, 1 / 16, 1.0, g)[3]):
        size[0][f1[e]] += np.abs(ds) @ np.abs(B[f2[e]])
        size[0 if shared else 1][f2[e]] += np.abs(ds).T @ np.abs(A[f1[e]])
    p[-1] = g * np.float32(2.0 ** k)
    _, large = _run(*p, shared, 1 / 16, 1.0)
    past = False
    for s, got, mag in zip(small, large, size):
        s, got = host(s.double()) * 2.0 ** k, host(got.double())
        bound = eps * (mag * 2.0 ** k + np.abs(s)) + 2.0 ** (k - 25)     # half the smallest step of the small one
        fits, over = np.abs(s) + bound <= 65504, np.abs(s) - bound > 65536
        assert fits.any()
        past |= over.any()
        assert (np.abs(got - s)[fits] <= bound[fits]).all()
        assert (got[over] == np.sign(s[over]) * np.inf).all()
    assert past or not shared    # (separate frames: no gradient reaches a quarter)
