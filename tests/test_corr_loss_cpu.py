"""The correlation losses without a GPU: the oracle against torch's cross
entropy / KL and central differences, the target helpers, and the entry points'
refusals (made on the host, before anything is launched)."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import corr_loss as oc


def _problem(seed, K, E=3, N1=2, P=7, N2=3, Q=11, D=8):
    rng = np.random.default_rng(seed)
    fmap1, fmap2 = rng.normal(size=(N1, P, D)), rng.normal(size=(N2, Q, D))
    f1, f2 = rng.integers(0, N1, E), rng.integers(0, N2, E)
    idx = np.stack([rng.permutation(Q)[:K] for _ in range(E * P)]).reshape(E, P, K)
    idx[0, 0] = -1
    idx[1, 2, 0] = -1
    return rng, fmap1, fmap2, f1, f2, idx


def test_oracle_cross_entropy_matches_torch():
    rng, a, b, f1, f2, idx = _problem(0, 1)
    g = rng.normal(size=idx.shape[:2])
    loss, d1, d2, _ = oc.corr_loss(a, b, f1, f2, idx, scale=0.7, g=g)
    ta, tb = torch.from_numpy(a).requires_grad_(), torch.from_numpy(b).requires_grad_()
    s = torch.einsum("epd,eqd->epq", ta[f1], tb[f2]) * 0.7
    t = torch.from_numpy(idx[..., 0])
    want = F.cross_entropy(s.reshape(-1, s.shape[-1]), t.reshape(-1), ignore_index=-1, reduction="none").view(t.shape)
    w1, w2 = torch.autograd.grad((want * torch.from_numpy(g)).sum(), [ta, tb])
    for x, y in ((loss, want), (d1, w1), (d2, w2)):
        np.testing.assert_allclose(x, y.detach().numpy(), rtol=1e-11, atol=1e-12)


@pytest.mark.parametrize("T", [1.0, 2.5])
def test_oracle_distillation_matches_torch_and_differences(T):
    rng, a, b, f1, f2, idx = _problem(1, 4)
    logits = 3 * rng.normal(size=idx.shape)
    logits[2, 3, 1] = -np.inf
    g = rng.normal(size=idx.shape[:2])
    loss, d1, d2, _ = oc.corr_loss(a, b, f1, f2, idx, logits, 0.7, T, g)
    s = torch.einsum("epd,eqd->epq", torch.from_numpy(a)[f1], torch.from_numpy(b)[f2]) * (0.7 / T)
    pi, used = oc.targets(idx, logits, T)
    q = torch.zeros_like(s).scatter_add(2, torch.from_numpy(np.maximum(idx, 0)), torch.from_numpy(pi))
    want = T * T * F.kl_div(torch.log_softmax(s, 2), q, reduction="none").sum(2)
    np.testing.assert_allclose(loss, np.where(used, want.numpy(), 0), rtol=1e-10, atol=1e-12)
    va, vb, h = rng.normal(size=a.shape), rng.normal(size=b.shape), 1e-6
    f = lambda x, y: (oc.corr_loss(x, y, f1, f2, idx, logits, 0.7, T) * g).sum()
    np.testing.assert_allclose((f(a + h * va, b) - f(a - h * va, b)) / (2 * h), (d1 * va).sum(), rtol=1e-6, atol=1e-6)
    np.testing.assert_allclose((f(a, b + h * vb) - f(a, b - h * vb)) / (2 * h), (d2 * vb).sum(), rtol=1e-6, atol=1e-6)


def test_target_helpers():
    from droid_mi355x import bilinear_targets, nearest_targets
    c = torch.tensor([[[0.0, 0.0], [3.4, 1.6], [4.0, 2.0], [4.2, 2.0], [-0.4, 0.3], [-3.0, 1.0], [float("nan"), 0.0],
                       [1e30, 0.0]]])
    ht, wd = 3, 5
    assert nearest_targets(c, ht, wd).tolist() == [[0, 2 * 5 + 3, 14, 14, 0, -1, -1, -1]]
    valid = torch.ones(1, 8)
    valid[0, 1] = 0
    assert nearest_targets(c, ht, wd, valid)[0, 1] == -1
    idx, logw = bilinear_targets(c, ht, wd, valid)
    assert idx.dtype == torch.int32 and logw.dtype == torch.float32 and idx.shape == (1, 8, 4)
    assert idx[0, 1].tolist() == [-1] * 4 and idx[0, 5].tolist() == [-1] * 4 and idx[0, 6].tolist() == [-1] * 4
    assert idx[0, 2].tolist() == [14, -1, -1, -1] and logw[0, 2, 0] == 0
    idx, logw = bilinear_targets(c, ht, wd)
    assert idx[0, 1].tolist() == [8, 9, 13, 14]
    np.testing.assert_allclose(logw[0, 1].exp().numpy(), [0.6 * 0.4, 0.4 * 0.4, 0.6 * 0.6, 0.4 * 0.6], rtol=1e-5)
    # weights outside the map are dropped, the rest renormalised by the loss
    assert (logw[idx < 0] == -np.inf).all()


def test_host_tensors_are_refused():
    import droid_backends as nb
    f = torch.zeros((2, 6, 8), dtype=torch.float16)
    e = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="HIP device"):
        nb.corr_loss_forward(f, None, e, e, torch.zeros((1, 6), dtype=torch.int32))
    with pytest.raises(RuntimeError, match="contiguous"):
        nb.corr_loss_forward(f.transpose(0, 1), None, e, e, torch.zeros((1, 6), dtype=torch.int32))


OK = dict(dtype=0, a=16, b=16, e1=16, e2=16, idx=16, lg=16, loss=16, lse=16, prob=16, E=2, N1=2, P=6, N2=2, Q=6, D=8,
          K=2, scale=0.1, T=1.0, ws=16, wsb=1 << 30)
NULLS = [dict(a=None), dict(b=None), dict(e1=None), dict(e2=None), dict(idx=None), dict(lse=None)]
BAD = [(dict(dtype=1), "float16 or bfloat16"), (dict(dtype=2), "float16 or bfloat16"), (dict(D=12), "bad arguments"),
       (dict(D=264), "bad arguments"), (dict(D=0), "bad arguments"), (dict(Q=0), "bad arguments"),
       (dict(E=-1), "bad arguments"), (dict(K=0), "bad arguments"), (dict(K=65), "bad arguments"),
       (dict(scale=0.0), "positive"), (dict(scale=-1.0), "positive"), (dict(scale=float("inf")), "positive"),
       (dict(T=0.0), "positive"), (dict(T=float("nan")), "positive"), (dict(a=24), "aligned"), (dict(b=8), "aligned"),
       (dict(ws=None), "workspace"), (dict(wsb=3), "workspace"), (dict(P=1 << 28, Q=1 << 28), "too large"),
       (dict(E=1 << 28), "too large")] + [(n, "null tensor") for n in NULLS]


def _forward(a):
    from droid_backends._lib import lib
    return lib.droid_corr_loss_forward(a["dtype"], a["a"], a["b"], a["e1"], a["e2"], a["idx"], a["lg"], a["loss"],
                                       a["lse"], a["prob"], a["E"], a["N1"], a["P"], a["N2"], a["Q"], a["D"], a["K"],
                                       a["scale"], a["T"], a["ws"], a["wsb"], None)


def _backward(a, d1=16, d2=16, shared=0):
    from droid_backends._lib import lib
    return lib.droid_corr_loss_backward(a["dtype"], a["a"], a["b"], a["e1"], a["e2"], a["idx"], a["prob"], a["lse"],
                                        a["loss"], d1, d2, shared, a["E"], a["N1"], a["P"], a["N2"], a["Q"], a["D"],
                                        a["K"], a["scale"], a["T"], a["ws"], a["wsb"], None)


@pytest.mark.parametrize("change,says", BAD)
def test_the_abi_refuses(change, says):
    """Pointers here are never read: each call ends at its check."""
    from droid_backends._lib import lib
    a = {**OK, **change}
    for call in (_forward, _backward):
        assert call(a) != 0 and says in lib.droid_last_error().decode(), call


def test_the_abi_refuses_more():
    from droid_backends._lib import lib
    says = lambda: lib.droid_last_error().decode()
    assert _forward({**OK, "loss": None}) != 0 and "null tensor" in says()
    assert _forward({**OK, "prob": None}) != 0 and "null tensor" in says()
    assert _forward({**OK, "lg": None}) != 0 and "one target" in says()
    assert _backward({**OK, "prob": None}) != 0 and "one target" in says()
    assert _backward(OK, None, None) != 0 and "null tensor" in says()
    assert _backward({**OK, "b": 32}, 16, None, 1) != 0 and "shared" in says()
    assert _backward(OK, 16, 16, 1) != 0 and "shared" in says()
    assert _backward({**OK, "Q": 7}, 16, None, 1) != 0 and "shared" in says()
    assert _backward({**OK, "E": 0}) != 0 and "no edges" in says()
    assert _forward({**OK, "E": 0}) == 0 and _forward({**OK, "P": 0}) == 0      # nothing to do
