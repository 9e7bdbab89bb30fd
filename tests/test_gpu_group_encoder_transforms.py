"""What the encoder with group norm did before its norms were fused, it still does on
the GPU: forward mode, function transforms, traces, batched gradients, hooks and
replaced modules.  fp32 against the same modules run op by op in float64 on the
host, bounds of test_gpu_group_encoder.py: 2e-3 forward (tangents, whose ReLUs cut
by the same signs, as its gradients: 8e-2)."""
import copy

import pytest
import torch
from torch.autograd import forward_ad
from torch.nn.utils import prune

from test_gpu_group_encoder import DEV, _encoder, _rel

pytestmark = pytest.mark.gpu


def _frames(n=2):
    return torch.randn((1, n, 3, 40, 56), generator=torch.Generator().manual_seed(5))


def _tangent(enc, x, t):
    """The directional derivative in float64, through the reverse mode's double use."""
    ref = copy.deepcopy(enc).double().cpu()
    for p in ref.parameters():
        p.requires_grad_(False)
    return torch.autograd.functional.jvp(ref.forward_reference, x.double(), t.double())


@pytest.mark.parametrize("trainable", [False, True])
def test_forward_mode(trainable):
    enc, x = _encoder(1, 16).to(DEV).requires_grad_(trainable), _frames()
    t = torch.randn_like(x)
    want, tangent = _tangent(enc, x, t)
    with forward_ad.dual_level():
        y = forward_ad.unpack_dual(enc(forward_ad.make_dual(x.to(DEV), t.to(DEV))))
        assert y.tangent is not None and _rel(y.primal, want) < 2e-3 and _rel(y.tangent, tangent) < 8e-2
    y, dy = torch.func.jvp(enc, (x.to(DEV),), (t.to(DEV),))
    assert _rel(y, want) < 2e-3 and _rel(dy, tangent) < 8e-2


def test_function_transforms_and_traces():
    enc, x = _encoder(2, 16).to(DEV).requires_grad_(False), _frames(3)
    want = copy.deepcopy(enc).double().cpu().forward_reference(x.double())
    got = torch.func.vmap(lambda f: enc(f[None, None])[0, 0])(x[0].to(DEV))
    assert _rel(got, want[0]) < 2e-3
    traced = torch.jit.trace(enc, torch.randn_like(x).to(DEV), check_trace=False)
    assert _rel(traced(x.to(DEV)), want) < 2e-3
    g = torch.func.grad(lambda f: enc(f).square().sum())(x.to(DEV))
    leaf = x.double().requires_grad_()
    ref = copy.deepcopy(enc).double().cpu().forward_reference(leaf).square().sum()
    assert _rel(g, torch.autograd.grad(ref, leaf)[0]) < 8e-2


@pytest.mark.parametrize("mode", range(5))
def test_a_batch_of_upstream_gradients(mode):
    from droid_mi355x import group_norm_act
    g = torch.Generator().manual_seed(mode)
    x, r, w, b = (torch.randn(s, generator=g) for s in ((2, 12, 5, 7), (2, 12, 5, 7), (12,), (12,)))
    ups = torch.randn((3, 2, 12, 5, 7), generator=g).to(DEV)
    cl = torch.channels_last
    leaves = [t.to(DEV, memory_format=cl) if t.dim() == 4 else t.to(DEV) for t in (x, w, b, r)]
    leaves = [t.requires_grad_() for t in leaves][:4 if mode in (1, 2) else 3]
    y = group_norm_act(leaves[0], 3, leaves[1], leaves[2], mode, leaves[3] if mode in (1, 2) else None)
    batch = torch.autograd.grad(y, leaves, ups, is_grads_batched=True, retain_graph=True)
    for k in range(3):
        one = torch.autograd.grad(y, leaves, ups[k], retain_graph=True)
        for p, q in zip(batch, one):    # a few dozen fp32 roundings of terms of one size on both sides
            assert _rel(p[k], q) < 1e-4


def test_hooks_and_replaced_modules():
    enc, x = _encoder(3, 16).to(DEV), _frames().to(DEV)
    assert enc._fuses_group(x)
    plain = lambda: enc.forward_reference(x)
    blk = enc.layer2[0]
    spots = [enc.norm1, enc.relu1, blk.norm1, blk.norm2, blk.norm3, blk.relu, blk.downsample, enc.layer3[1].norm2]
    for m in spots:
        for hook in (m.register_forward_hook, m.register_forward_pre_hook):
            calls = []
            handle = hook(lambda *a: calls.append(1))
            enc(x)
            assert calls
            handle.remove()
        calls = []
        handle = m.register_full_backward_hook(lambda *a: calls.append(1)) if m is blk.downsample else None   # (the others feed an in-place ReLU)
        if handle:
            enc(x).sum().backward()
            assert calls
            handle.remove()
    calls = []
    handle = torch.nn.modules.module.register_module_forward_hook(lambda m, *a: calls.append(type(m)))
    enc(x)
    handle.remove()
    assert torch.nn.GroupNorm in calls
    assert enc._fuses_group(x)
    prune.random_unstructured(blk.norm1, "weight", 0.5)
    assert _rel(enc(x), plain()) < 2e-3
    prune.remove(blk.norm1, "weight")
    enc.layer1[0].norm2 = torch.nn.Identity()
    assert not enc._fuses_group(x) and _rel(enc(x), plain()) < 2e-3
    enc.layer1[0].norm2 = torch.nn.GroupNorm(4, 32, affine=False).to(DEV)
    assert enc._fuses_group(x) and _rel(enc(x), plain()) < 2e-3
    enc.layer1[0].relu = torch.nn.GELU()
    assert not enc._fuses_group(x) and _rel(enc(x), plain()) < 2e-3


def test_more_images_than_a_grid_has_rows():
    enc = _encoder(4, 16).to(DEV)
    assert not enc._fuses_group(torch.empty((1, 65535, 3, 1, 1), device=DEV))


def test_the_losses_refuse_a_batch_of_upstream_gradients():
    from droid_mi355x import corr_cross_entropy
    f = torch.randn((2, 30, 16), device=DEV).half().requires_grad_()
    e, t = torch.tensor([0, 1], dtype=torch.int32, device=DEV), torch.zeros((2, 30), dtype=torch.int32, device=DEV)
    loss = corr_cross_entropy(f, None, e, e.flip(0), t)
    with pytest.raises(RuntimeError, match="do not reach"):
        torch.autograd.grad(loss, f, torch.ones((3, 2, 30), device=DEV), is_grads_batched=True, retain_graph=True)
    assert torch.autograd.grad(loss, f, torch.ones((2, 30), device=DEV))[0].any()


def test_compiled():
    """torch.compile traces the modules one by one."""
    enc, x = _encoder(8, 16).to(DEV), _frames().to(DEV)
    want = copy.deepcopy(enc).double().cpu().forward_reference(x.double().cpu())
    got = torch.compile(enc, backend="eager")(x)
    assert _rel(got.detach(), want.detach()) < 2e-3
