"""What follows a tensor besides autograd's tape.

The operators' kernels write their outputs through pointers: forward-mode
tangents, function transforms (vmap, jvp, grad of torch.func), tracers
(torch.jit.trace, torch.compile, export, fake tensors) and dispatch modes do not
see that.  Where there is one, operators with a form in torch's own operators run
that, and the others refuse the call."""
import torch
from torch.autograd import forward_ad


_PLAIN = {torch.Tensor, torch.nn.Parameter, type(None)}
_MODES = (torch._C._TorchDispatchModeKey.FAKE, torch._C._TorchDispatchModeKey.PROXY,
          torch._C._TorchDispatchModeKey.FUNCTIONAL)
_compiling, _tracing = torch.compiler.is_compiling, torch._C._is_tracing
_transform, _modes = torch._C._functorch.peek_interpreter_stack, torch._C._len_torch_dispatch_stack


def _carries(tensors):
    """Whether a tensor dispatches by itself or has a tangent."""
    for t in tensors:
        if type(t) not in _PLAIN and type(t).__torch_dispatch__ is not torch.Tensor.__torch_dispatch__:
            return True
    return forward_ad._current_level >= 0 and any(
        t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def followed(*tensors):
    """Whether anything but the tape follows this call, any dispatch mode included:
    what a form in torch's operators is for."""
    return _compiling() or _tracing() or _transform() is not None or _modes() > 0 or _carries(tensors)


def batched(g):
    """Whether an upstream gradient is a batch of them (autograd.grad's is_grads_batched)."""
    return torch._C._functorch.is_legacy_batchedtensor(g)


def refuse(fn, *tensors):
    """For operators without such a form.  Dispatch modes that only watch (counters,
    selective checkpointing) are let through, tracers are not; torch.compile runs the
    operator between two graphs and needs no refusal."""
    if (_tracing() or _transform() is not None or _carries(tensors)
            or _modes() > 0 and any(torch._C._get_dispatch_mode(k) is not None for k in _MODES)):
        _refused(fn)


def _refused(fn):
    raise RuntimeError("%s: forward-mode tangents, function transforms (vmap, jvp, torch.func.grad) and tracers "
                       "do not reach this operator" % fn)


def refuse_upstream(fn, g):
    """The same for a backward pass."""
    refuse(fn, g)
    if batched(g):
        _refused(fn)
