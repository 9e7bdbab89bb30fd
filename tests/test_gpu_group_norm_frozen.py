"""Group norm with parameters that are not trained: the other gradients keep their bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("train_w,train_b", [(False, False), (True, False), (False, True)])
def test_frozen_parameters(mode, train_w, train_b, monkeypatch):
    import droid_backends as nb
    from droid_mi355x import group_norm_act
    g = torch.Generator(device=DEV).manual_seed(mode)
    x, r, dy = (torch.randn((2, 24, 9, 14), generator=g, device=DEV).contiguous(memory_format=torch.channels_last)
                for _ in range(3))
    w, b = (torch.randn(24, generator=g, device=DEV) for _ in range(2))
    made, call = [], nb._group_norm_act_backward

    def watch(*a):
        made.append(call(*a))
        return made[-1]

    monkeypatch.setattr(nb, "_group_norm_act_backward", watch)

    def grads(tw, tb):
        leaves = [t.clone().requires_grad_(on) for t, on in ((x, True), (w, tw), (b, tb), (r, mode != 0))]
        group_norm_act(leaves[0], 4, leaves[1], leaves[2], mode, leaves[3] if mode else None).backward(dy)
        return [t.grad for t in leaves]

    full, some = grads(True, True), grads(train_w, train_b)
    assert [t is not None for t in made[-1][2:]] == [train_w, train_b]
    for p, q in zip(full, some):
        assert q is None or torch.equal(p, q)
    assert (some[1] is not None) == train_w and (some[2] is not None) == train_b
