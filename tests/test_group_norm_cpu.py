"""Group norm + activation without a GPU: the oracle's gradients against central
differences and torch's group norm, and every refusal of the entry points (all
of them made on the host, before anything is launched)."""
import ctypes

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import group_norm as og


@pytest.mark.parametrize("mode", range(5))
@pytest.mark.parametrize("shape,groups", [((2, 3, 5, 8), 2), ((1, 1, 1, 6), 3), ((2, 4, 3, 5), 5), ((1, 7, 2, 4), 1)])
def test_oracle_matches_torch_and_differences(shape, groups, mode):
    rng = np.random.default_rng(sum(shape) + mode)
    x, res, dy = rng.normal(size=shape) * 2 + 1, rng.normal(size=shape), rng.normal(size=shape)
    w, b = rng.normal(size=shape[-1]), rng.normal(size=shape[-1])
    y, n = og.group_norm_act(x, groups, w, b, mode, res)
    t = F.group_norm(torch.from_numpy(x).permute(0, 3, 1, 2), groups, torch.from_numpy(w), torch.from_numpy(b), 1e-5)
    np.testing.assert_allclose(n, t.permute(0, 2, 3, 1).numpy(), rtol=1e-12, atol=1e-12)
    dx, dres, dw, db = og.group_norm_act_backward(dy, x, groups, w, b, mode, res)
    # central differences: 64-bit rounding 1e-16 / h and curvature h^2, both far under 1e-6 at h = 1e-6
    h = 1e-6
    f = lambda x, w, b, r: (og.group_norm_act(x, groups, w, b, mode, r)[0] * dy).sum()
    vx, vw, vb, vr = (rng.normal(size=s.shape) for s in (x, w, b, res))
    tol = dict(rtol=2e-6, atol=2e-6)
    np.testing.assert_allclose((f(x + h * vx, w, b, res) - f(x - h * vx, w, b, res)) / (2 * h), (dx * vx).sum(), **tol)
    np.testing.assert_allclose((f(x, w + h * vw, b, res) - f(x, w - h * vw, b, res)) / (2 * h), (dw * vw).sum(), **tol)
    np.testing.assert_allclose((f(x, w, b + h * vb, res) - f(x, w, b - h * vb, res)) / (2 * h), (db * vb).sum(), **tol)
    if dres is not None:
        np.testing.assert_allclose((f(x, w, b, res + h * vr) - f(x, w, b, res - h * vr)) / (2 * h),
                                   (dres * vr).sum(), **tol)


def test_host_tensors_and_bad_arguments_are_refused():
    import droid_backends as nb
    x = torch.zeros((1, 8, 2, 2)).contiguous(memory_format=torch.channels_last)
    with pytest.raises(RuntimeError, match="HIP device"):
        nb.group_norm_act(x, 2)
    with pytest.raises(TypeError):
        nb.group_norm_act(np.zeros((1, 8, 2, 2), np.float32), 2)
    with pytest.raises(RuntimeError, match="HIP device"):
        nb.group_norm_act_backward(x, x, torch.zeros((1, 2, 2), dtype=torch.float64), 2)


OK = dict(dtype=0, x=16, res=16, out=16, w=None, b=None, wdt=1, stats=None, N=1, HW=4, C=8, G=2, mode=0, eps=1e-5,
          ws=16, wsb=1 << 20)


@pytest.mark.parametrize("change,says", [
    (dict(dtype=2), "dtype"), (dict(dtype=7), "dtype"), (dict(wdt=0, dtype=1), "weight"), (dict(wdt=2), "weight"),
    (dict(N=-1), "bad arguments"), (dict(HW=-4), "bad arguments"), (dict(C=0), "bad arguments"),
    (dict(C=520), "bad arguments"), (dict(G=3), "bad arguments"), (dict(G=0), "bad arguments"),
    (dict(mode=5), "bad arguments"), (dict(mode=-1), "bad arguments"), (dict(N=65535), "images"),
    (dict(x=None), "null map"), (dict(out=None), "null map"), (dict(mode=1, res=None), "null map"),
    (dict(mode=2, res=None), "null map"), (dict(ws=None), "workspace"), (dict(wsb=31), "workspace")])
def test_the_abi_refuses(change, says):
    """Pointers here are never read: each call ends at its check."""
    from droid_backends._lib import lib
    a = {**OK, **change}
    st = lib.droid_group_norm_act(a["dtype"], a["x"], a["res"], a["out"], a["w"], a["b"], a["wdt"], a["stats"],
                                  a["N"], a["HW"], a["C"], a["G"], a["mode"], a["eps"], a["ws"], a["wsb"], None)
    assert st != 0 and says in lib.droid_last_error().decode()
    st = lib.droid_group_norm_act_backward(a["dtype"], a["x"], a["res"], a["x"], a["w"], a["b"], a["wdt"], a["out"],
                                           a["out"], a["out"], None, None, a["N"], a["HW"], a["C"], a["G"], a["mode"],
                                           a["ws"], a["wsb"], None)
    assert st != 0 and says in lib.droid_last_error().decode()


def test_workspace_and_empty_maps():
    from droid_backends._lib import lib
    ws = lib.droid_group_norm_workspace
    assert ws(0, 1, 4, 8, 2, 0) == 2 * 16 and ws(0, 1, 4, 8, 2, 1) == (2 + 8) * 16
    assert ws(0, 0, 4, 8, 2, 0) == 0 and ws(0, 1, 0, 8, 2, 0) == 0 and ws(0, 1, 4, 8, 3, 0) == 0
    # nothing to normalise: accepted without a launch (there is no device here)
    for N, HW in ((0, 4), (2, 0)):
        assert lib.droid_group_norm_act(0, None, None, None, None, None, 1, None, N, HW, 8, 2, 0, 1e-5, None, 0,
                                        None) == 0
        assert lib.droid_group_norm_act_backward(0, None, None, None, None, None, 1, None, None, None, None, None,
                                                 N, HW, 8, 2, 0, None, 0, None) == 0
