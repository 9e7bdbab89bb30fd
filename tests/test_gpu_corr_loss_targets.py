"""Target lists of the distillation loss on the MI355X as teachers write them:
keys named twice, places without weight, masks of the lowest value.  Oracle and
tolerances of test_gpu_corr_loss.py."""
import numpy as np
import pytest
import torch

from gpu_util import host
from test_gpu_corr_loss import PAIR, TYPES, _check, _problem, _run, _t

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("K,T", [(2, 1.0), (3, 1.0), (16, 2.0), (17, 1.0), (40, 2.0), (64, 1.0)])
def test_a_repeated_key_whose_first_place_has_no_weight(K, T, shared, dtype):
    """The first place and a later one (K > 16: of another lane's share) name one
    key; the first has a logit of -inf, or one so low that its weight is zero."""
    import droid_backends as nb
    dt = TYPES[dtype]
    a, b, f1, f2, idx, logits, g = _problem(40 + K, dt, K, 4, 3, 90, 3, 90, 64, shared=shared)
    if shared:
        f1[:], f2[:], g = [0, 1, 2, 2], [1, 0, 1, 2], np.abs(g)
    rng = np.random.default_rng(K)
    idx = rng.random((4, 90, 90)).argsort(-1)[..., :K].astype(np.int32)
    later = rng.integers(1, K, (4, 90))
    key = np.take_along_axis(idx, later[..., None], 2)[..., 0]
    idx[..., 0] = key
    low = rng.random((4, 90)) < 0.5
    logits[..., 0] = np.where(low, -np.inf, -400.0)          # e^-200 at T = 2: zero in fp32
    if K > 2:                                                # and a third place of the key, before or after
        idx[:, ::3, K - 1] = key[:, ::3]
    p = (a, b, f1, f2, idx, logits, g)
    loss, grads = _run(*p, shared, 1 / 16, T)
    _check(dt, *p, shared, 1 / 16, T, loss, grads, PAIR if shared else 0)
    prob = host(nb.corr_loss_forward(a, None if shared else b, _t(f1), _t(f2), _t(idx), _t(logits), 1 / 16, T)[2])
    assert not prob[..., 0].any()
    # the weights kept add up to one: K + 2 fp32 roundings of them
    np.testing.assert_allclose(prob.sum(-1), 1.0, atol=(K + 2) * 2.0 ** -24 * 4)


def test_a_list_padded_with_key_zero():
    """Short lists filled up with key 0 and a logit of -inf, key 0 itself a target of some rows."""
    dt = torch.float16
    a, b, f1, f2, idx, logits, g = _problem(50, dt, 8, 3, 2, 130, 2, 77, 128)
    n = np.random.default_rng(50).integers(0, 9, (3, 130))
    pad = np.arange(8) >= n[..., None]
    idx[idx < 0] = 5
    idx[:, ::4, 0] = 0
    idx[pad], logits[pad] = 0, -np.inf
    p = (a, b, f1, f2, idx, logits, g)
    loss, grads = _run(*p, False, 1 / 16, 1.0)
    assert not loss[torch.from_numpy(n == 0).to(loss.device)].any()
    _check(dt, *p, False, 1 / 16, 1.0, loss, grads)


@pytest.mark.parametrize("value", [np.inf, np.nan])
def test_teacher_logits_that_are_no_numbers_are_not_dropped(value):
    """+inf or NaN among a row's logits: the row's loss is NaN."""
    dt = torch.float16
    a, b, f1, f2, idx, logits, g = _problem(51, dt, 4, 2, 2, 40, 2, 50, 64)
    idx[:] = np.arange(4)
    logits[1, 7, 2] = value
    loss, grads = _run(a, b, f1, f2, idx, logits, g, False, 1 / 16, 1.0)
    bad = torch.zeros((2, 40), dtype=torch.bool)
    bad[1, 7] = True
    assert torch.equal(loss.isnan().cpu(), bad)
    assert grads[0][f1[1], 7].isnan().all()


@pytest.mark.parametrize("T", [0.5, 1.0, 2.0])
def test_logits_masked_with_the_lowest_value(T):
    """The type's lowest value is a logit like any other: a row of nothing else is
    uniform, beside an ordinary one it has no weight - at T < 1 too, where it
    overflows when divided."""
    dt = torch.bfloat16
    a, b, f1, f2, idx, logits, g = _problem(52, dt, 5, 2, 2, 70, 2, 90, 64)
    idx[:] = np.random.default_rng(52).random((2, 70, 90)).argsort(-1)[..., :5]
    logits[:, ::2, :4] = np.finfo(np.float32).min
    logits[:, ::3] = np.finfo(np.float32).min
    p = (a, b, f1, f2, idx, logits, g)
    loss, grads = _run(*p, False, 1 / 16, T)
    assert (loss[:, ::3] != 0).all()
    _check(dt, *p, False, 1 / 16, T, loss, grads)
