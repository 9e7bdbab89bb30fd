"""Group norm + activation on the MI355X against the float64 oracle, forward and
backward.

Tolerances.  u = 2^-24 is fp32's largest rounding, h half a step of the output's
type.  n = fma(x - m, rw, b): the roundings of m, x - m, rw and the fma add up
to at most u (|m rw| + 3 |d rw| + |b| + |n|), d = x - mean; the residual adds
one more, SiLU's exp and reciprocal a few relative ones.  8 u of the sum of the
terms' sizes covers all of them, plus one rounding to the output's type (for
fp16 at least half its smallest subnormal, 2^-25).
dx = rw dn - (q1 + d q2): each product and sum one rounding; q1, q2 are means
of values summed in fp32 within a thread (at most 24 of them at these sizes)
and in 64 bits beyond: 32 u of the mean of the absolute values covers them.
dweight, dbias: the same sums, rounded to the parameter's type."""
import numpy as np
import pytest
import torch

from gpu_util import host
from oracle import group_norm as og

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _half_step(dt, v):
    return torch.finfo(dt).eps / 2 * np.abs(v) + (2.0 ** -25 if dt == torch.float16 else 2.0 ** -126)


def _map(rng, dt, N, C, H, W, mul=1.0, add=0.0):
    t = torch.from_numpy(rng.normal(size=(N, H, W, C)).astype(np.float32) * mul + add)
    return t.to(dt).to(DEV).permute(0, 3, 1, 2)


def _rows(t):
    return host(t.double()).transpose(0, 2, 3, 1)


def _inputs(dt, N, C, H, W, seed=0, mul=2.0, add=0.5, pdt=torch.float32):
    rng = np.random.default_rng(seed)
    x, res, dy = _map(rng, dt, N, C, H, W, mul, add), _map(rng, dt, N, C, H, W).relu(), _map(rng, dt, N, C, H, W)
    w = torch.from_numpy(1 + 0.3 * rng.normal(size=C)).to(pdt).to(DEV)
    b = torch.from_numpy(0.3 * rng.normal(size=C)).to(pdt).to(DEV)
    return x, res, dy, w, b


def _check(dt, x, res, dy, w, b, G, mode, y, dx, dres, dw, db, eps=1e-5):
    X, R, DY = _rows(x), _rows(res), _rows(dy)
    Wt = host(w.double()) if w is not None else np.ones(X.shape[3])
    B = host(b.double()) if b is not None else np.zeros(X.shape[3])
    N, H, W, C = X.shape
    per = lambda v: np.repeat(v, C // G, 1)[:, None, None, :]
    xhat, mean, rstd = og._normalise(X, G, eps)
    mean, rstd = per(mean), per(rstd)
    ref, n = og.group_norm_act(X, G, Wt, B, mode, R, eps)
    size = np.abs(mean * rstd * Wt) + 3 * np.abs(xhat * Wt) + np.abs(B) + np.abs(n) + np.abs(R)
    assert y.is_contiguous(memory_format=torch.channels_last) and y.dtype == dt
    assert (np.abs(_rows(y) - ref) <= 8 * U * size + _half_step(dt, ref)).all()
    if dx is None:
        return
    rdx, rdres, rdw, rdb = og.group_norm_act_backward(DY, X, G, Wt, B, mode, R, eps)
    if rdres is not None:
        assert np.array_equal(_rows(dres), rdres)          # dy or zero: exact
    dn = np.abs(DY) * (1.1 if mode == og.SILU else 1.0)     # |silu'| < 1.1
    gm = lambda v: per(v.reshape(N, H * W, G, C // G).mean((1, 3)))
    xs = np.abs(xhat) + np.abs(mean) * rstd                 # xhat with the size of x - mean's roundings
    terms = np.abs(Wt) * dn + gm(dn * np.abs(Wt)) * 5 + xs * gm(dn * np.abs(Wt) * xs) * 5
    slope = 8 * U * size * np.abs(DY * Wt) if mode == og.SILU else np.zeros_like(X)   # |silu''| < 1
    tol = rstd * (8 * U * terms + slope + gm(slope) + np.abs(xhat) * gm(slope * np.abs(xhat))) + _half_step(dt, rdx)
    assert (np.abs(_rows(dx) - rdx) <= tol).all()
    for got, want, v in ((dw, rdw, dn * (np.abs(xhat) + np.abs(mean) * rstd)), (db, rdb, dn)):
        if got is not None:
            bound = 32 * U * v.sum((0, 1, 2)) + _half_step(got.dtype, want)
            if mode == og.SILU:
                bound = bound + (8 * U * size * np.abs(DY) * (1 + np.abs(xhat))).sum((0, 1, 2))
            assert (np.abs(host(got.double()) - want) <= bound).all()


SHAPES = [(1, 1, 1, 1, 1), (2, 8, 1, 1, 2), (1, 8, 1, 3, 8), (2, 32, 5, 7, 8), (2, 32, 24, 40, 4), (3, 60, 13, 11, 12),
          (1, 511, 3, 5, 73), (1, 512, 9, 4, 1), (2, 48, 20, 37, 48), (5, 15, 17, 3, 5), (1, 128, 40, 64, 16),
          (4, 21, 44, 6, 7), (1, 3, 241, 7, 1)]


@pytest.mark.parametrize("mode", range(5))
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("N,C,H,W,G", SHAPES)
def test_forward_and_backward(N, C, H, W, G, dtype, mode):
    from droid_mi355x import group_norm_act
    dt = TYPES[dtype]
    x, res, dy, w, b = _inputs(dt, N, C, H, W, seed=N * C + H + mode)
    leaves = [t.requires_grad_() for t in (x, w, b, res)]
    y = group_norm_act(x, G, w, b, mode, res)
    with_res = mode in (og.RES_RELU, og.ADD_RELU)
    g = torch.autograd.grad(y, leaves if with_res else leaves[:3], dy)
    _check(dt, x.detach(), res.detach(), dy, w.detach(), b.detach(), G, mode, y.detach(), g[0],
           g[3] if with_res else None, g[1], g[2])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_far_mean_parameter_types_and_absent_parameters(dtype):
    """A mean far above the spread (the sums must not cancel), parameters of x's
    type, no parameters, only one of them, another eps."""
    import droid_backends as nb
    dt = TYPES[dtype]
    for pdt, has_w, has_b, eps in ((dt, True, True, 1e-5), (torch.float32, False, False, 1e-3),
                                   (torch.float32, True, False, 1e-5), (torch.float32, False, True, 1e-5)):
        x, res, dy, w, b = _inputs(dt, 2, 24, 19, 23, seed=3, mul=0.5, add=60.0, pdt=pdt)
        w, b = (w if has_w else None), (b if has_b else None)
        y, stats = nb.group_norm_act(x, 6, w, b, nb.NORM_RELU, eps=eps, return_stats=True)
        dx, dres, dw, db = nb.group_norm_act_backward(dy, x, stats, 6, w, b, nb.NORM_RELU)
        assert dres is None and (dw is None) == (not has_w) and (db is None) == (not has_b)
        _check(dt, x, res, dy, w, b, 6, og.RELU, y, dx, None, dw, db, eps)


def test_constant_groups_and_zero_residuals():
    """var = 0 (rstd = 1 / sqrt(eps)); residuals that are exactly zero beside cut
    values: relu(0 + relu(n <= 0)) passes no gradient."""
    import droid_backends as nb
    x, res, dy, w, b = _inputs(torch.float16, 2, 16, 6, 5, seed=9)
    x = x.clone(memory_format=torch.channels_last)
    x[0, :8] = 3.0
    res.zero_()
    for mode in range(5):
        y, stats = nb.group_norm_act(x, 2, w, b, mode, res, return_stats=True)
        dx, dres, dw, db = nb.group_norm_act_backward(dy, x, stats, 2, w, b, mode, res)
        # rstd = 316 multiplies the constant group's roundings: _check's bounds carry rstd
        _check(torch.float16, x, res, dy, w, b, 2, mode, y, dx, dres, dw, db)


@pytest.mark.parametrize("mode", range(5))
def test_nan_and_infinity_stay_in_their_group(mode):
    import droid_backends as nb
    x, res, dy, w, b = _inputs(torch.float32, 2, 16, 6, 5, seed=4)
    x = x.clone(memory_format=torch.channels_last)
    clean = nb.group_norm_act(x, 4, w, b, mode, res)
    x[0, 2, 3, 1], x[1, 15, 0, 0] = float("nan"), float("inf")
    y = nb.group_norm_act(x, 4, w, b, mode, res)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[0, :4], bad[1, 12:] = True, True
    assert torch.equal(y[~bad], clean[~bad]) and y[bad].isnan().all()


def test_in_place_and_repeatable():
    import droid_backends as nb
    x, res, dy, w, b = _inputs(torch.bfloat16, 3, 40, 31, 29, seed=5)
    y, stats = nb.group_norm_act(x, 5, w, b, nb.NORM_ADD_RELU, res, return_stats=True)
    g = nb.group_norm_act_backward(dy, x, stats, 5, w, b, nb.NORM_ADD_RELU, res)
    again = nb.group_norm_act_backward(dy, x, stats, 5, w, b, nb.NORM_ADD_RELU, res)
    assert all(torch.equal(p, q) for p, q in zip(g, again))       # fixed order of every sum
    for target in (0, 1):
        x1, r1 = x.clone(memory_format=torch.channels_last), res.clone(memory_format=torch.channels_last)
        out = nb.group_norm_act(x1, 5, w, b, nb.NORM_ADD_RELU, r1, out=(x1, r1)[target])
        assert out.data_ptr() == (x1, r1)[target].data_ptr() and torch.equal(out, y)


def test_other_stream_and_graph_replay():
    """On a side stream, and captured: replays on new inputs, with eager work
    between them, equal the eager results."""
    import droid_backends as nb
    a = [_inputs(torch.float16, 2, 32, 24, 40, seed=s) for s in range(3)]
    x, res, dy, w, b = a[0]
    x, res, dy = (t.clone(memory_format=torch.channels_last) for t in (x, res, dy))

    def both(x, res, dy):
        y, stats = nb.group_norm_act(x, 4, w, b, nb.NORM_RES_RELU, res, return_stats=True)
        return (y,) + nb.group_norm_act_backward(dy, x, stats, 4, w, b, nb.NORM_RES_RELU, res)

    want = [[t.clone() for t in both(*v[:3])] for v in a]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both(x, res, dy)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(got, want[0]))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = both(x, res, dy)
    for k in (1, 2, 0):
        for dst, src in zip((x, res, dy), a[k][:3]):
            dst.copy_(src)
        g.replay()
        both(*a[1][:3])
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want[k])), k


def test_refusals_on_the_device():
    import droid_backends as nb
    x, res, dy, w, b = _inputs(torch.float16, 1, 16, 4, 5)
    bad = [dict(x=x.contiguous()), dict(x=x.double()), dict(num_groups=3), dict(num_groups=0), dict(weight=w[:8]),
           dict(weight=w.double()), dict(bias=b.half()), dict(weight=w.cpu()), dict(mode=9),
           dict(mode=nb.NORM_RES_RELU), dict(mode=nb.NORM_RES_RELU, res=res.float()),
           dict(mode=nb.NORM_ADD_RELU, res=res[:, :8]), dict(out=torch.empty_like(x).float()),
           dict(x=x[:, :, ::2])]
    for kw in bad:
        with pytest.raises((RuntimeError, TypeError)):
            nb.group_norm_act(**{**dict(x=x, num_groups=2, weight=w, bias=b), **kw})
    _, stats = nb.group_norm_act(x, 2, w, b, return_stats=True)
    for st in (stats.float(), stats[:, :1], stats.cpu()):
        with pytest.raises(RuntimeError):
            nb.group_norm_act_backward(dy, x, st, 2, w, b)
    with pytest.raises(RuntimeError):
        nb.group_norm_act_backward(dy.float(), x, stats, 2, w, b)
    for shape in ((0, 16, 4, 5), (2, 16, 0, 5)):
        e = torch.empty(shape, dtype=torch.float16, device=DEV).contiguous(memory_format=torch.channels_last)
        y, st = nb.group_norm_act(e, 2, w, b, return_stats=True)
        assert y.shape == e.shape
        dx, _, dw, db = nb.group_norm_act_backward(y, e, st, 2, w, b)
        assert dx.shape == e.shape and not dw.any() and not db.any()


def test_offsets_past_32_bits_and_maps_past_the_abi():
    """2.4e9 values: the last image as alone (another split of its sums: one
    rounding of the output apart); more than 2^31 - 1 pixels are refused."""
    import droid_backends as nb
    one = torch.randn(1, 256, 1024, 1024, device=DEV).half().contiguous(memory_format=torch.channels_last)
    dy1 = torch.randn(1, 256, 1024, 1024, device=DEV).half().contiguous(memory_format=torch.channels_last)
    w, b = torch.rand(256, device=DEV) + 0.5, torch.randn(256, device=DEV)

    def both(x, dy):
        y, st = nb.group_norm_act(x, 8, w, b, nb.NORM_SILU, return_stats=True)
        return y[-1], nb.group_norm_act_backward(dy, x, st, 8, w, b, nb.NORM_SILU)[0][-1]

    def many(t):
        m = torch.empty((9, 256, 1024, 1024), dtype=t.dtype, device=DEV, memory_format=torch.channels_last)
        m[:8] = 0
        m[8:] = t
        return m

    for got, want in zip(both(many(one), many(dy1)), both(one, dy1)):
        for c in range(0, 256, 64):   # (in parts: bounds the memory of the comparison)
            g, e = got[c:c + 64].float(), want[c:c + 64].float()
            assert ((g - e).abs() <= 2.0 ** -10 * e.abs() + 2.0 ** -20).all()
    big = torch.empty((1, 1, 65536, 32768), dtype=torch.float16, device=DEV)
    with pytest.raises(RuntimeError, match="too large"):
        nb.group_norm_act(big.contiguous(memory_format=torch.channels_last), 1)


@pytest.mark.parametrize("mode", range(5))
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("N,C,H,W,G", [(1, 16, 64, 64, 2), (1, 16, 64, 65, 2), (1, 16, 32, 64, 2), (3, 32, 50, 101, 4),
                                       (2, 64, 97, 43, 16), (9, 8, 1, 1, 1), (40, 64, 41, 25, 8)])
def test_forward_and_backward_around_one_launch(N, C, H, W, G, dtype, mode):
    """Groups that just fit one workgroup's registers, just do not, and maps too
    large for one launch; the output in x's and in res's place."""
    import droid_backends as nb
    dt = TYPES[dtype]
    x, res, dy, w, b = _inputs(dt, N, C, H, W, seed=C + H + mode)
    y, stats = nb.group_norm_act(x, G, w, b, mode, res, return_stats=True)
    dx, dres, dw, db = nb.group_norm_act_backward(dy, x, stats, G, w, b, mode, res)
    _check(dt, x, res, dy, w, b, G, mode, y, dx, dres, dw, db)
    for place in ("x", "res"):
        xi, ri = x.clone(memory_format=torch.channels_last), res.clone(memory_format=torch.channels_last)
        out = xi if place == "x" else ri
        assert torch.equal(nb.group_norm_act(xi, G, w, b, mode, ri, out=out), y)
