"""The encoder with group norm on the fused operators, and a training step over it:
features -> cross entropy / distillation over the correlation -> gradients.

Tolerances, relative in the 2-norm.  fp32: a convolution's K products (at most
1152) are off by at most K 2^-24 = 7e-5 of their terms; 15 layers, each
norm dividing by a spread no smaller than its terms' half: 15 * 2 * 7e-5 = 2e-3.
Gradients: ReLU arguments within that of zero change sign, at most a share of
2e-3 / 5 of the values in each of 15 layers, each at most its own gradient: the
2-norm moves by at most sqrt(15 * 4e-4) = 8e-2.  fp16 under autocast: 15 * 2
roundings of 2^-11 in the maps and as many in the weights, 2 * 15 * 2 * 2^-11 =
3e-2; the gradient's signs, sqrt(15 * 3e-2 / 5) = 0.3."""
import copy

import numpy as np
import pytest
import torch

from gpu_util import host
from oracle import corr_loss as oc

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _rel(got, want):
    want = want.double().cpu()
    return float((got.double().cpu() - want).norm() / want.norm())


def _encoder(seed, dim=64):
    from droid_mi355x.extractor import BasicEncoder
    torch.manual_seed(seed)
    enc = BasicEncoder(output_dim=dim, norm_fn="group")
    with torch.no_grad():
        for m in enc.modules():
            if isinstance(m, torch.nn.GroupNorm):
                m.weight.uniform_(0.5, 1.5)
                m.bias.uniform_(-0.5, 0.5)
    return enc


@pytest.mark.parametrize("b,n,h,w", [(1, 2, 64, 96), (2, 1, 40, 72)])
@pytest.mark.parametrize("autocast", [False, True])
def test_encoder_forward_and_gradients(b, n, h, w, autocast):
    enc = _encoder(1)
    x = torch.randn(b, n, 3, h, w)
    ref = copy.deepcopy(enc).double()
    want = ref.forward_reference(x.double())
    g = torch.randn(want.shape)
    want.backward(g.double())
    enc = enc.to(DEV)
    with torch.autocast("cuda", dtype=torch.float16, enabled=autocast):
        got = enc(x.to(DEV))
        plain = copy.deepcopy(enc).forward_reference(x.to(DEV))
    got.backward(g.to(DEV, got.dtype))
    assert got.dtype == plain.dtype and got.shape == want.shape and got.is_contiguous()
    assert _rel(got, want) < (3e-2 if autocast else 2e-3)
    for (name, p), q in zip(enc.named_parameters(), ref.parameters()):
        # a convolution's bias before a norm of its own channels has gradient ~ 0: no relative error
        if q.grad.norm() > 1e-3 * g.norm():
            assert _rel(p.grad, q.grad) < (0.3 if autocast else 8e-2), name
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.float16, enabled=autocast):
        again = enc(x.to(DEV))
    # (not bit for bit: the library may choose another convolution algorithm)
    assert again.dtype == got.dtype and _rel(again, want) < (3e-2 if autocast else 2e-3)


def test_encoder_types_it_leaves_to_the_plain_operators():
    enc = _encoder(2, 16)
    x = torch.randn(1, 1, 3, 32, 48)
    want = enc.double().forward_reference(x.double())
    assert torch.equal(enc(x.double()), want)                      # host
    assert _rel(enc.to(DEV)(x.double().to(DEV)), want) < 1e-12     # double on the GPU
    half = enc.half()
    assert _rel(half(x.half().to(DEV)), want) < 5e-2               # norm parameters in half too


@pytest.mark.parametrize("K", [0, 4])
def test_training_step(K):
    """Two directions of every neighbouring pair of four frames, targets from
    reprojected coordinates, the mean of the loss: the features' gradient against
    float64, and through the encoder against the float64 module."""
    from droid_mi355x import bilinear_targets, corr_cross_entropy, corr_distillation, nearest_targets
    enc = _encoder(3)
    n, h, w = 4, 64, 80
    ht, wd = h // 8, w // 8
    x = torch.randn(1, n, 3, h, w)
    f1 = torch.tensor([0, 1, 1, 2, 2, 3], dtype=torch.int32)
    f2 = torch.tensor([1, 0, 2, 1, 3, 2], dtype=torch.int32)
    yy, xx = torch.meshgrid(torch.arange(ht), torch.arange(wd), indexing="ij")
    flow = 1.7 * torch.randn(6, 1, 1, 2)
    coords = torch.stack([xx, yy], -1).float() + flow + 0.3 * torch.randn(6, ht, wd, 2)
    enc = enc.to(DEV)
    with torch.autocast("cuda", dtype=torch.float16):
        fmap = enc(x.to(DEV))
    assert fmap.dtype == torch.float16
    rows = fmap[0].permute(0, 2, 3, 1).contiguous()
    rows.retain_grad()
    e = (f1.to(DEV), f2.to(DEV))
    if K:
        idx, logits = bilinear_targets(coords.to(DEV), ht, wd)
        loss = corr_distillation(rows, None, *e, idx, logits)
        i, l = host(idx).reshape(6, -1, 4), host(logits).reshape(6, -1, 4)
    else:
        idx = nearest_targets(coords.to(DEV), ht, wd)
        loss = corr_cross_entropy(rows, None, *e, idx)
        i, l = host(idx).reshape(6, -1, 1), None
    assert loss.shape == (6, ht, wd)
    scale = 1024.0
    (loss.mean() * scale).backward()
    a = host(rows.detach().double()).reshape(n, ht * wd, -1)
    g = np.full((6, ht * wd), scale / (6 * ht * wd))
    want, d1, d2, _ = oc.corr_loss(a, a, f1.numpy(), f2.numpy(), i, l, 1 / 16, 1.0, g)
    np.testing.assert_allclose(host(loss).reshape(6, -1), want, rtol=1e-4, atol=1e-4)
    # weights and result rounded to fp16: 2^-11 of the terms each, which do not cancel to less than a quarter
    assert _rel(rows.grad.reshape(n, ht * wd, -1), torch.from_numpy(d1 + d2)) < 4 * 2 * 2.0 ** -11
    # the same features' gradient through the float64 module
    ref = copy.deepcopy(enc).double().cpu()
    for p in ref.parameters():
        p.grad = None
    out = ref.forward_reference(x.double())
    out.backward(torch.from_numpy(d1 + d2).view(1, n, ht, wd, -1).permute(0, 1, 4, 2, 3))
    for (name, p), q in zip(enc.named_parameters(), ref.parameters()):
        if q.grad.norm() > 1e-2 * ref.conv2.weight.grad.norm():
            assert _rel(p.grad, q.grad) < 0.3, name


@pytest.mark.parametrize("mode", range(5))
def test_second_derivatives(mode):
    """A backward pass under create_graph, differentiated again."""
    from droid_mi355x import group_norm_act
    from droid_mi355x.extractor import _group_norm_act_plain
    torch.manual_seed(mode)
    ins = [torch.randn(2, 12, 5, 7).contiguous(memory_format=torch.channels_last), torch.rand(12) + 0.5,
           torch.randn(12), torch.randn(2, 12, 5, 7).contiguous(memory_format=torch.channels_last)]
    g = torch.randn(2, 12, 5, 7)

    def second(fn, dev):
        x, w, b, r = (t.clone().to(dev).requires_grad_() for t in ins)
        y = fn(x, 3, w, b, mode, r if mode in (1, 2) else None, 1e-5)
        d, = torch.autograd.grad(y, [x], g.to(dev), create_graph=True)
        return torch.autograd.grad(d.square().sum(), [x, w])

    # a few dozen fp32 roundings of terms of one size on both sides
    for a, b in zip(second(group_norm_act, DEV), second(_group_norm_act_plain, "cpu")):
        assert _rel(a, b) < 1e-4
    # x and its residual the same tensor
    if mode in (1, 2):
        x = ins[0].clone().to(DEV).requires_grad_()
        y = group_norm_act(x, 3, None, None, mode, x)
        first, = torch.autograd.grad(y, [x], g.to(DEV), retain_graph=True)
        again, = torch.autograd.grad(y, [x], g.to(DEV), create_graph=True)
        assert _rel(again, first) < 1e-5


def test_saved_tensors_kept_on_the_host():
    """save_on_cpu hands back maps that are not channels_last."""
    from droid_backends import NORM_ADD_RELU
    from droid_mi355x import group_norm_act
    torch.manual_seed(0)
    x, r = (torch.randn(2, 24, 9, 7, device=DEV).contiguous(memory_format=torch.channels_last) for _ in range(2))
    w, b, g = torch.rand(24, device=DEV), torch.randn(24, device=DEV), torch.randn(2, 24, 9, 7, device=DEV)

    def grads():
        leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
        y = group_norm_act(leaves[0], 4, leaves[1], leaves[2], NORM_ADD_RELU, leaves[3])
        return y, leaves

    y, leaves = grads()
    want = torch.autograd.grad(y, leaves, g)
    with torch.autograd.graph.save_on_cpu():
        y, leaves = grads()
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, leaves, g), want))
