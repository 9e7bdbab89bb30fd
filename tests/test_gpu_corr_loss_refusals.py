"""Calls of the correlation losses on device tensors that are refused before anything
is launched, and the largest edge list."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _call():
    f = torch.randn((2, 20, 16), device=DEV).half()
    e = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    return f, e, torch.zeros((2, 20, 3), dtype=torch.int32, device=DEV), torch.zeros((2, 20, 3), device=DEV)


def test_target_lists_of_no_or_too_many_places():
    import droid_backends as nb
    f, e, idx, logits = _call()
    _, lse, prob = nb.corr_loss_forward(f, None, e, e, idx, logits)
    g = torch.ones((2, 20), device=DEV)
    for K in (0, 65):
        i, w = (torch.zeros((2, 20, K), dtype=d, device=DEV) for d in (torch.int32, torch.float32))
        with pytest.raises(RuntimeError, match="targets a row"):
            nb.corr_loss_forward(f, None, e, e, i, w)
        with pytest.raises(RuntimeError, match="targets a row"):
            nb.corr_loss_backward(g, f, None, e, e, i, lse, w)
    for i in (idx[0, 0, 0], None):
        with pytest.raises(RuntimeError, match="idx must be"):
            nb.corr_loss_forward(f, None, e, e, i, logits)
        with pytest.raises(RuntimeError, match="idx must be"):
            nb.corr_loss_backward(g, f, None, e, e, i, lse, prob)


def test_edges_between_no_frames():
    import droid_backends as nb
    f, e, idx, _ = _call()
    for a, b in ((f[:0], f), (f, f[:0]), (f[:0], None)):
        with pytest.raises(RuntimeError, match="no frames"):
            nb.corr_loss_forward(a, b, e, e, idx[..., 0].contiguous())
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    loss, _, _ = nb.corr_loss_forward(f[:0], None, none, none, torch.empty((0, 20), dtype=torch.int32, device=DEV))
    assert loss.shape == (0, 20)


def test_the_largest_edge_list():
    """65536 edges of one-row frames, paired at random: softmax over one key, so the
    loss is |error| of s - s and the gradient p - 1 of p = 1."""
    from droid_mi355x import corr_cross_entropy
    g = torch.Generator(device=DEV).manual_seed(0)
    f = torch.randn((500, 1, 8), generator=g, device=DEV).half().requires_grad_()
    a, b = (torch.randint(0, 500, (65536,), generator=g, device=DEV, dtype=torch.int32) for _ in range(2))
    t = torch.zeros((65536, 1), dtype=torch.int32, device=DEV)
    loss = corr_cross_entropy(f, None, a, b, t)
    d, = torch.autograd.grad(loss.sum(), f)
    # s of 8 products in fp32, twice; p off by 2 (8 + 8 |lse|) 2^-24 at most, times 1/16 and the edges' sums
    assert (loss.abs() <= 64 * 2.0 ** -24 * 8).all()
    n = torch.bincount(torch.cat([a, b]), minlength=500).max()
    assert (d.float().abs() <= 64 * 2.0 ** -24 * 8 / 16 * n * f.abs().max() + 2.0 ** -24).all()
    more = torch.cat([a, a[:1]]), torch.cat([b, b[:1]]), torch.cat([t, t[:1]])
    with pytest.raises(RuntimeError, match="65536 edges"):
        torch.autograd.grad(corr_cross_entropy(f, None, *more).sum(), f)


@pytest.mark.parametrize("K", [0, 3])
def test_compiled_between_two_graphs(K):
    """torch.compile leaves the operator to the eager mode: the same loss and gradient."""
    from droid_mi355x import corr_cross_entropy, corr_distillation
    f, e, idx, logits = _call()

    def step(x):
        x = x * 2
        loss = (corr_distillation(x, None, e, e.flip(0), idx, logits) if K
                else corr_cross_entropy(x, None, e, e.flip(0), idx[..., 0].contiguous()))
        return loss.sum() * 3

    out = []
    for fn in (step, torch.compile(step, backend="eager")):
        x = f.clone().requires_grad_()
        y = fn(x)
        out.append((y.detach(), torch.autograd.grad(y, x)[0]))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1]) and out[0][1].any()
