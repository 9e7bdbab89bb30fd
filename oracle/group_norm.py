"""Group norm + activation / residual add (modules/extractor.py: nn.GroupNorm of
BasicEncoder(norm_fn='group') with the ReLUs and adds around it), forward and
backward, in float64.  Maps are (N, H, W, C)."""
import numpy as np

RELU, RES_RELU, ADD_RELU, NONE, SILU = range(5)


def _normalise(x, groups, eps):
    N, H, W, C = x.shape
    v = x.reshape(N, H * W, groups, C // groups)
    mean = v.mean((1, 3), keepdims=True)
    rstd = 1.0 / np.sqrt(((v - mean) ** 2).mean((1, 3), keepdims=True) + eps)
    return ((v - mean) * rstd).reshape(x.shape), mean.reshape(N, groups), rstd.reshape(N, groups)


def group_norm_act(x, groups, weight, bias, mode, res=None, eps=1e-5):
    """-> y, and the pre-activation n."""
    xhat, _, _ = _normalise(x, groups, eps)
    n = xhat * weight + bias
    if mode == RELU:
        return np.maximum(n, 0), n
    if mode == RES_RELU:
        return np.maximum(res + np.maximum(n, 0), 0), n
    if mode == ADD_RELU:
        return np.maximum(n + res, 0), n
    if mode == SILU:
        return n / (1 + np.exp(-n)), n
    return n, n


def group_norm_act_backward(dy, x, groups, weight, bias, mode, res=None, eps=1e-5):
    """-> dx, dres (None without a residual), dweight, dbias."""
    N, H, W, C = x.shape
    xhat, _, rstd = _normalise(x, groups, eps)
    y, n = group_norm_act(x, groups, weight, bias, mode, res, eps)
    dres = None
    if mode in (RES_RELU, ADD_RELU):
        dres = np.where(y > 0, dy, 0.0)
        dn = np.where(n > 0, dres, 0.0) if mode == RES_RELU else dres
    elif mode == RELU:
        dn = np.where(n > 0, dy, 0.0)
    elif mode == SILU:
        s = 1 / (1 + np.exp(-n))
        dn = dy * (s + n * s * (1 - s))
    else:
        dn = dy
    g = (dn * weight).reshape(N, H * W, groups, C // groups)
    xv = xhat.reshape(g.shape)
    k1 = g.mean((1, 3), keepdims=True)
    k2 = (g * xv).mean((1, 3), keepdims=True)
    dx = (rstd[:, None, :, None] * (g - k1 - xv * k2)).reshape(x.shape)
    return dx, dres, (dn * xhat).sum((0, 1, 2)), dn.sum((0, 1, 2))
