"""MotionFilter feature encoders (modules/extractor.py:1-198, droid_net.py:149-150)
on the MI355X: the same module tree (parameter names match, so the
reference's droid.pth loads), run channels-last fp16 - the convolutions on
MIOpen through torch, every InstanceNorm2d together with the ReLU / residual
add around it in one hand-written pass pair (droid_instance_norm_act_f16,
csrc/norm_kernels.hip).  `forward` keeps the reference's signature and output
(b, n, C, H/8, W/8); `forward_reference` is the module run op by op as the
reference runs it (the parity bridge for the tests).
"""
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd import forward_ad

import droid_backends

from . import tracing

DIM = 32


def _group_norm_act_plain(x, num_groups, weight, bias, mode, res, eps):
    nb = droid_backends
    f = lambda t: None if t is None else t.float()
    n = F.group_norm(x.float(), num_groups, f(weight), f(bias), eps)
    if mode == nb.NORM_RELU:
        n = torch.relu(n)
    elif mode == nb.NORM_RES_RELU:
        n = torch.relu(res.float() + torch.relu(n))
    elif mode == nb.NORM_ADD_RELU:
        n = torch.relu(n + res.float())
    elif mode == nb.NORM_SILU:
        n = F.silu(n)
    return n.to(x.dtype)


class GroupNormAct(torch.autograd.Function):
    """Group norm + activation / residual add (droid_group_norm_act and its
    backward): statistics in 64 bits, gradients of every input.  A backward pass
    that is itself differentiated (create_graph) or batched (is_grads_batched) goes
    through torch's operators."""

    @staticmethod
    def forward(ctx, x, num_groups, weight, bias, mode, res, eps):
        y, stats = droid_backends.group_norm_act(x, num_groups, weight, bias, mode, res, eps=eps, return_stats=True)
        ctx.save_for_backward(x, weight, bias, res, stats)
        ctx.num_groups, ctx.mode, ctx.eps = num_groups, mode, eps
        ctx.wdt = droid_backends._norm_params("group_norm_act", x, num_groups, weight, bias)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, weight, bias, res, stats = ctx.saved_tensors
        again = torch.is_grad_enabled()
        if again or tracing.followed(dy) or tracing.batched(dy):   # differentiated again, or a batch of dy
            with torch.enable_grad():
                # (views: x and res may be one tensor)
                ins = {i: t.view_as(t) for i, t in ((0, x), (2, weight), (3, bias), (5, res)) if t is not None}
                want = [i for i in ins if ctx.needs_input_grad[i]]
                if not again:
                    ins = {i: t.detach().requires_grad_(i in want) for i, t in ins.items()}
                y = _group_norm_act_plain(ins[0], ctx.num_groups, ins.get(2), ins.get(3), ctx.mode, ins.get(5), ctx.eps)
                grads = dict(zip(want, torch.autograd.grad(y, [ins[i] for i in want], dy, create_graph=again)))
            return tuple(grads.get(i) for i in range(7))
        # the forward call checked them; saved-tensor hooks may return another layout
        cl = torch.channels_last
        dx, dres, dw, db = droid_backends._group_norm_act_backward(
            dy.contiguous(memory_format=cl), x.contiguous(memory_format=cl), stats.contiguous(), ctx.num_groups,
            weight, bias, ctx.mode, None if res is None else res.contiguous(memory_format=cl), ctx.wdt,
            *ctx.needs_input_grad[2:4])
        return dx, None, dw, db, None, dres, None


def group_norm_act(x, num_groups, weight=None, bias=None, mode=droid_backends.NORM_RELU, res=None, eps=1e-5):
    """droid_backends.group_norm_act under autograd: x (and res) channels_last
    (N,C,H,W) fp16 / bf16 / fp32 on the GPU; gradients reach x, weight, bias and res.
    Under forward mode, function transforms and tracers: torch's operators in fp32."""
    if mode not in (droid_backends.NORM_RES_RELU, droid_backends.NORM_ADD_RELU):
        res = None
    if tracing.followed(x, weight, bias, res):
        return _group_norm_act_plain(x, num_groups, weight, bias, mode, res, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, res)):
        return GroupNormAct.apply(x, num_groups, weight, bias, mode, res, eps)
    return droid_backends.group_norm_act(x, num_groups, weight, bias, mode, res, eps=eps)


def _norm(kind, planes):
    if kind == "group":
        return nn.GroupNorm(num_groups=planes // 8, num_channels=planes)
    if kind == "batch":
        return nn.BatchNorm2d(planes)
    if kind == "instance":
        return nn.InstanceNorm2d(planes)
    return nn.Sequential()


def _norm_act(norm, x, mode, res=None):
    """nn.GroupNorm on a convolution's output, with the activation / residual add after
    it; under autocast in fp32, as torch's autocast runs group norm and what follows."""
    x = x.to(torch.float32 if torch.is_autocast_enabled("cuda") else x.dtype, memory_format=torch.channels_last)
    return group_norm_act(x, norm.num_groups, norm.weight, norm.bias, mode, res, norm.eps)


def _plain(m, kind):
    """Whether a module does what its type says and nobody listens to its calls."""
    return (type(m) is kind and not m._forward_hooks and not m._forward_pre_hooks and not m._backward_hooks
            and not m._backward_pre_hooks and "forward" not in m.__dict__)


def _plain_norm(m, dt):
    if not _plain(m, nn.GroupNorm) or m.num_channels > 512:
        return False
    kinds = {t.dtype for t in (m.weight, m.bias) if t is not None}
    return len(kinds) <= 1 and kinds <= {torch.float32, dt}


class ResidualBlock(nn.Module):
    """extractor.py:6-55 (3x3 conv - norm - ReLU twice, 1x1 strided shortcut)."""

    def __init__(self, in_planes, planes, norm_fn="group", stride=1):
        super().__init__()
        self.conv1 = nn.Conv2d(in_planes, planes, kernel_size=3, padding=1, stride=stride)
        self.conv2 = nn.Conv2d(planes, planes, kernel_size=3, padding=1)
        self.relu = nn.ReLU(inplace=True)
        self.norm_fn = norm_fn
        self.norm1 = _norm(norm_fn, planes)
        self.norm2 = _norm(norm_fn, planes)
        if stride != 1:
            self.norm3 = _norm(norm_fn, planes)
        self.downsample = None if stride == 1 else nn.Sequential(
            nn.Conv2d(in_planes, planes, kernel_size=1, stride=stride), self.norm3)

    def forward_reference(self, x):
        y = self.relu(self.norm1(self.conv1(x)))
        y = self.relu(self.norm2(self.conv2(y)))
        if self.downsample is not None:
            x = self.downsample(x)
        return self.relu(x + y)

    def forward_group(self, x):
        """channels_last in and out, group norm fused with what follows it."""
        nb = droid_backends
        y = _norm_act(self.norm1, self.conv1(x), nb.NORM_RELU)
        y2 = self.conv2(y)
        if self.downsample is None:
            return _norm_act(self.norm2, y2, nb.NORM_RES_RELU, x)          # relu(x + relu(n(y2)))
        y = _norm_act(self.norm2, y2, nb.NORM_RELU)
        return _norm_act(self.norm3, self.downsample[0](x), nb.NORM_ADD_RELU, y)

    def forward_fast(self, x):
        """channels_last fp16 in and out (instance or no norm)."""
        nb = droid_backends
        if self.norm_fn == "instance":
            y = nb.instance_norm_act_f16(_conv(self.conv1, x), nb.NORM_RELU)
            y2 = _conv(self.conv2, y)
            if self.downsample is None:
                return nb.instance_norm_act_f16(y2, nb.NORM_RES_RELU, res=x)           # relu(x + relu(n(y2)))
            y = nb.instance_norm_act_f16(y2, nb.NORM_RELU)
            return nb.instance_norm_act_f16(_conv(self.downsample[0], x), nb.NORM_ADD_RELU, res=y)
        y = torch.relu_(_conv(self.conv1, x))
        y = torch.relu_(_conv(self.conv2, y))
        if self.downsample is not None:
            x = _conv(self.downsample[0], x)
        return torch.relu_(x + y)


def _conv(conv, x):
    """nn.Conv2d on a channels_last fp16 map (MIOpen), fp16 weights as under
    autocast (cast once per parameter version)."""
    key = (conv.weight.data_ptr(), conv.weight._version,
           None if conv.bias is None else (conv.bias.data_ptr(), conv.bias._version))
    c = getattr(conv, "_f16", None)
    if c is None or c[0] != key:
        c = (key, conv.weight.detach().to(torch.float16).contiguous(memory_format=torch.channels_last),
             None if conv.bias is None else conv.bias.detach().to(torch.float16))
        conv._f16 = c
    y = F.conv2d(x, c[1], c[2], conv.stride, conv.padding)
    return y.contiguous(memory_format=torch.channels_last)


class BasicEncoder(nn.Module):
    """extractor.py:120-198 (multidim=False, as DroidNet builds it)."""

    def __init__(self, output_dim=128, norm_fn="batch", dropout=0.0, multidim=False):
        super().__init__()
        if multidim:
            raise NotImplementedError("BasicEncoder(multidim=True) is not used by DroidNet")
        self.norm_fn = norm_fn
        self.norm1 = _norm(norm_fn, DIM) if norm_fn != "group" else nn.GroupNorm(num_groups=8, num_channels=DIM)
        self.conv1 = nn.Conv2d(3, DIM, kernel_size=7, stride=2, padding=3)
        self.relu1 = nn.ReLU(inplace=True)
        self.in_planes = DIM
        self.layer1 = self._make_layer(DIM, stride=1)
        self.layer2 = self._make_layer(2 * DIM, stride=2)
        self.layer3 = self._make_layer(4 * DIM, stride=2)
        self.conv2 = nn.Conv2d(4 * DIM, output_dim, kernel_size=1)
        self.dropout = nn.Dropout2d(p=dropout) if dropout > 0 else None
        for m in self.modules():
            if isinstance(m, nn.Conv2d):
                nn.init.kaiming_normal_(m.weight, mode="fan_out", nonlinearity="relu")
            elif isinstance(m, (nn.BatchNorm2d, nn.InstanceNorm2d, nn.GroupNorm)):
                if m.weight is not None:
                    nn.init.constant_(m.weight, 1)
                if m.bias is not None:
                    nn.init.constant_(m.bias, 0)

    def _make_layer(self, dim, stride=1):
        layers = (ResidualBlock(self.in_planes, dim, self.norm_fn, stride=stride),
                  ResidualBlock(dim, dim, self.norm_fn, stride=1))
        self.in_planes = dim
        return nn.Sequential(*layers)

    def forward_reference(self, x):
        b, n, c1, h1, w1 = x.shape
        x = x.view(b * n, c1, h1, w1)
        x = self.relu1(self.norm1(self.conv1(x)))
        for layer in (self.layer1, self.layer2, self.layer3):
            for blk in layer:
                x = blk.forward_reference(x)
        x = self.conv2(x)
        _, c2, h2, w2 = x.shape
        return x.view(b, n, c2, h2, w2)

    def forward_group(self, x):
        """forward_reference with norm_fn 'group' on the GPU, for training and
        inference: channels_last throughout, every norm one operator with its
        activation and residual add.  Maps between the convolutions have x's type,
        under autocast fp32 (a module and input in half precision keep them in it)."""
        b, n, c1, h1, w1 = x.shape
        x = x.reshape(b * n, c1, h1, w1).contiguous(memory_format=torch.channels_last)
        x = _norm_act(self.norm1, self.conv1(x), droid_backends.NORM_RELU)
        for layer in (self.layer1, self.layer2, self.layer3):
            for blk in layer:
                x = blk.forward_group(x)
        x = self.conv2(x)
        _, c2, h2, w2 = x.shape
        return x.contiguous().view(b, n, c2, h2, w2)

    def _fuses_group(self, x):
        """Whether forward_group stands for forward_reference here: nothing but autograd's
        tape follows the tensors, and every module that it does not call is the plain one,
        without hooks, in a type and size of the operator."""
        if (tracing.followed(x) or forward_ad._current_level >= 0 or torch.nn.modules.module._has_any_global_hook()
                or x.dim() != 5 or x.shape[0] * x.shape[1] > 65534):
            return False
        if x.dtype not in (torch.float16, torch.bfloat16, torch.float32):
            return False
        dt = torch.float32 if torch.is_autocast_enabled("cuda") else x.dtype
        blocks = [blk for layer in (self.layer1, self.layer2, self.layer3) for blk in layer]
        return (_plain_norm(self.norm1, dt) and _plain(self.relu1, nn.ReLU)
                and all(_plain_norm(b.norm1, dt) and _plain_norm(b.norm2, dt) and _plain(b.relu, nn.ReLU)
                        and (b.downsample is None
                             or _plain(b.downsample, nn.Sequential) and len(b.downsample) == 2
                             and b.downsample[1] is b.norm3 and _plain_norm(b.norm3, dt)) for b in blocks))

    def forward(self, x):
        """(b, n, 3, H, W) -> (b, n, C, H/8, W/8) fp16: the MI355X path for the
        norms DroidNet uses (instance: fnet, none: cnet - no running statistics,
        so train and eval mode agree; the reference never applies its dropout).
        Training (gradients through the encoder) runs the reference ops, except
        with norm_fn 'group', whose norms are one operator each (forward_group)."""
        if self.norm_fn == "group" and x.is_cuda and self._fuses_group(x):
            return self.forward_group(x)
        if (self.norm_fn not in ("instance", "none") or not x.is_cuda
                or (torch.is_grad_enabled() and self.conv1.weight.requires_grad)):
            return self.forward_reference(x)
        b, n, c1, h1, w1 = x.shape
        x = x.reshape(b * n, c1, h1, w1).to(torch.float16).contiguous(memory_format=torch.channels_last)
        with torch.autocast("cuda", enabled=False):
            x = _conv(self.conv1, x)
            if self.norm_fn == "instance":
                x = droid_backends.instance_norm_act_f16(x, droid_backends.NORM_RELU)
            else:
                x = torch.relu_(x)
            for layer in (self.layer1, self.layer2, self.layer3):
                for blk in layer:
                    x = blk.forward_fast(x)
            x = _conv(self.conv2, x)
        _, c2, h2, w2 = x.shape
        return x.contiguous().view(b, n, c2, h2, w2)
