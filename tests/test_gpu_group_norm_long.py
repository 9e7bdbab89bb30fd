"""Group norm's parameter gradients over many more pieces than a thread adds in fp32
(32; the rest in 64 bits), against float64 sums.

Tolerance, u = 2^-24: a thread's fp32 sums have at most 32 roundings, each within u
of a partial sum that the terms' absolute values bound: 32 u of their sum; dn xhat
has four roundings of its own (x - mean with the mean rounded, two products): 4 u of
|dn| (|xhat| + |mean| rstd).  One rounding to the parameter's type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


@pytest.mark.parametrize("dtype,H,W,mode,constant", [
    (torch.float32, 160, 240, 3, 1.750640869140625),    # 600 pieces a thread, whose fp32 sum is off by 150 u
    (torch.float32, 160, 240, 3, None), (torch.bfloat16, 160, 256, 1, None), (torch.float16, 160, 256, 0, None)])
def test_hundreds_of_pieces_a_thread(dtype, H, W, mode, constant):
    import droid_backends as nb
    N, C, G = 512, 32, 4
    g = torch.Generator(device=DEV).manual_seed(H + mode)

    def map_():
        return torch.randn((N, H, W, C), generator=g, device=DEV).to(dtype).permute(0, 3, 1, 2)

    x, dy = map_().mul_(2).add_(0.5), map_().abs_()
    if constant:
        dy.fill_(constant)
    res = map_().abs_() if mode == nb.NORM_RES_RELU else None
    w, b = 1 + 0.3 * torch.randn(C, generator=g, device=DEV), 0.3 * torch.randn(C, generator=g, device=DEV)
    y, stats = nb.group_norm_act(x, G, w, b, mode, res, return_stats=True)
    del y
    dx, dres, dw, db = nb.group_norm_act_backward(dy, x, stats, G, w, b, mode, res)
    want = torch.zeros((2, C), dtype=torch.float64, device=DEV)
    size = torch.zeros_like(want)
    for k in range(N):
        v = x[k].permute(1, 2, 0).reshape(H * W, G, C // G).double()
        var, mean = torch.var_mean(v, (0, 2), correction=0, keepdim=True)
        rstd = (var + 1e-5).rsqrt()
        xhat = ((v - mean) * rstd).reshape(H * W, C)
        n = xhat * w.double() + b.double()
        dn = dy[k].permute(1, 2, 0).reshape(H * W, C).double()
        if mode != nb.NORM_ONLY:    # (a residual >= 0 cuts nothing more, nor less: relu(res + relu(n)) > 0 where n is)
            dn = dn * (n > 0)
        want += torch.stack([(dn * xhat).sum(0), dn.sum(0)])
        far = xhat.abs() + (mean.abs() * rstd).expand(1, G, C // G).reshape(1, C)
        size += torch.stack([(dn * far).sum(0), dn.sum(0)])
    bound = U * torch.stack([36 * size[0], 32 * size[1]]) + U * want.abs()
    got = torch.stack([dw, db]).double()
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / (U * size)).max().item()
    assert dx.shape == x.shape and not dx[::97].isnan().any()
