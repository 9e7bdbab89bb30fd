"""What follows a tensor besides the tape: the operators' checks, without a GPU."""
import numpy as np
import pytest
import torch
from torch._subclasses import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils.flop_counter import FlopCounterMode

from droid_mi355x import corr_cross_entropy, corr_distillation, group_norm_act, tracing
from oracle import group_norm as og


def _seen(call):
    """What followed / refuse say inside `call`."""
    out = []

    def ask(*t):
        out.append(tracing.followed(*t) or tracing.batched(t[0]))
        try:
            (tracing.refuse_upstream if len(t) == 1 else tracing.refuse)("op", *t)
            out.append(False)
        except RuntimeError as e:
            assert "op: " in str(e)
            out.append(True)
        return t[0]

    call(ask)
    return tuple(out[:2])


def _dual(ask):
    with forward_ad.dual_level():
        x = torch.ones(2)
        ask(torch.zeros(2), forward_ad.make_dual(x, x))


def _level_only(ask):
    with forward_ad.dual_level():
        ask(torch.zeros(2))


def _fake(ask):
    with FakeTensorMode():
        ask(torch.ones(2))


def _fake_outside(ask):
    with FakeTensorMode():
        x = torch.ones(2)
    ask(x)


def _count(ask):
    with FlopCounterMode(display=False):
        ask(torch.ones(2))


def _batched(ask):
    class Op(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return x.clone()

        @staticmethod
        def backward(ctx, g):
            return ask(g)

    x = torch.ones(2, requires_grad=True)
    torch.autograd.grad(Op.apply(x), x, torch.ones(3, 2), is_grads_batched=True)


CALLS = {"nothing": (lambda ask: ask(torch.ones(2), None, torch.nn.Parameter(torch.ones(2))), (False, False)),
         "tangent": (_dual, (True, True)), "a level without tangents": (_level_only, (False, False)),
         "vmap": (lambda ask: torch.func.vmap(ask)(torch.ones(2, 2)), (True, True)),
         "func.grad": (lambda ask: torch.func.grad(lambda x: ask(x).sum())(torch.ones(2)), (True, True)),
         "jit.trace": (lambda ask: torch.jit.trace(ask, torch.ones(2), check_trace=False), (True, True)),
         "make_fx": (lambda ask: make_fx(lambda x: ask(x) + 1)(torch.ones(2)), (True, True)),
         "fake": (_fake, (True, True)), "fake tensor": (_fake_outside, (True, True)),
         "batched gradients": (_batched, (True, True)), "counter": (_count, (True, False))}


@pytest.mark.parametrize("name", list(CALLS))
def test_followed_and_refused(name):
    call, want = CALLS[name]
    assert _seen(call) == want


def test_the_losses_refuse():
    f = torch.zeros((2, 6, 8), dtype=torch.float16)
    e, t = torch.zeros(1, dtype=torch.int32), torch.zeros((1, 6), dtype=torch.int32)
    calls = [lambda f: corr_cross_entropy(f, None, e, e, t),
             lambda f: corr_distillation(f, f, e, e, t[..., None], torch.zeros(1, 6, 1))]
    for call in calls:
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="do not reach"):
                call(forward_ad.make_dual(f, f))
        with pytest.raises(RuntimeError, match="do not reach"):
            torch.func.vmap(call)(f[None])
        with pytest.raises(RuntimeError, match="do not reach"):
            torch.jit.trace(call, f)


@pytest.mark.parametrize("mode", range(5))
def test_group_norm_under_transforms(mode):
    """torch's operators: also on the host, where the operator itself has no path.
    Tangents against the float64 oracle's differences; a few dozen fp32 roundings
    of terms of one size, 2^-24 each: 1e-5 in the 2-norm."""
    g = torch.Generator().manual_seed(mode)
    x, t, r = (torch.randn((3, 2, 12, 5, 4), generator=g) for _ in range(3))
    f = lambda x: group_norm_act(x, 3, None, None, mode, r[0])
    rows = lambda v: v.double().permute(0, 2, 3, 1).numpy()
    h = 1e-6
    o = lambda s: og.group_norm_act(rows(x[0]) + s * h * rows(t[0]), 3, 1.0, 0.0, mode, rows(r[0]))[0]
    want = (o(1) - o(-1)) / (2 * h)
    with forward_ad.dual_level():
        y, dy = forward_ad.unpack_dual(f(forward_ad.make_dual(x[0], t[0])))
    for got in (dy, torch.func.jvp(f, (x[0],), (t[0],))[1]):
        assert np.linalg.norm(rows(got) - want) < 1e-5 * np.linalg.norm(want)
    torch.testing.assert_close(torch.func.vmap(f)(x)[0], y)
    torch.testing.assert_close(torch.compile(f, backend="eager", fullgraph=True)(x[0]), y)
    torch.testing.assert_close(torch.jit.trace(f, x[0], check_trace=False)(x[0]), y)
