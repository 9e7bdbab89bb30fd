"""The encoder with group norm keeps the precision of torch's autocast: convolutions in
the half type, norms, ReLUs, residual stream and their gradients in fp32.

Tolerance of the comparison with the modules run one by one under the same autocast:
each of the 15 convolutions rounds a value the other way where its fp32 sums differ
across the border between two numbers of the type.  The sums differ by at most 1152
2^-24 = 7e-5 of their terms' size, such borders lie eps (2^-10 in fp16, 2^-7 in bf16)
apart: a share of 7e-5 / eps of the values, 0.07 or 0.009, by one eps each (not half:
the two results are neighbours).  A norm doubles a relative difference at most:
2-norm 2 eps sqrt(15 share) = 2.0e-3 in fp16, 5.7e-3 in bf16."""
import copy

import pytest
import torch

from test_gpu_group_encoder import DEV, _encoder, _rel

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,bound", [(torch.float16, 2.0e-3), (torch.bfloat16, 5.7e-3)])
@pytest.mark.parametrize("xdtype", [torch.float32, torch.float16])
def test_maps_and_their_gradients_stay_in_fp32(dtype, bound, xdtype):
    enc = _encoder(6, 32).to(DEV)
    x = torch.randn((1, 2, 3, 64, 80), generator=torch.Generator().manual_seed(6)).to(DEV, xdtype)
    seen = {}

    def watch(which):
        def hook(name):
            def f(m, args):
                a = args[0]
                seen[which].append((name, a.dtype))
                if a.requires_grad:
                    a.register_hook(lambda g: seen[which].append((name + ".grad", g.dtype)))
            return f
        return hook

    out = {}
    for which, run in (("fused", lambda e: e(x)), ("plain", lambda e: e.forward_reference(x))):
        e, seen[which] = copy.deepcopy(enc), []
        for name, m in e.named_modules():
            if isinstance(m, torch.nn.Conv2d):
                m.register_forward_pre_hook(watch(which)(name))
        assert e._fuses_group(x)      # (the convolutions are called as modules)
        with torch.autocast("cuda", dtype=dtype):
            out[which] = run(e)
        out[which].float().square().sum().backward()
    assert out["fused"].dtype == out["plain"].dtype == dtype
    key = lambda v: sorted((n, str(t)) for n, t in v)
    assert key(seen["fused"]) == key(seen["plain"]), (seen["fused"], seen["plain"])
    assert sum(t == torch.float32 for _, t in seen["fused"]) >= 2 * 14
    assert _rel(out["fused"].detach(), out["plain"].detach()) < bound


def test_norm_parameters_in_half_under_autocast():
    """torch's autocast casts them; the operator takes fp32 ones beside fp32 maps."""
    enc = _encoder(7, 16).to(DEV).half()
    x = torch.randn((1, 1, 3, 32, 48), device=DEV)
    with torch.no_grad(), torch.autocast("cuda"):
        assert not enc._fuses_group(x)
        assert torch.isfinite(enc(x)).all()
    assert enc._fuses_group(x.half())
