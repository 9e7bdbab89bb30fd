"""Targets from coordinates of any type: the row index is a whole number that half
types do not hold."""
import pytest
import torch

from droid_mi355x import bilinear_targets, nearest_targets

TYPES = [torch.float16, torch.bfloat16, torch.float32, torch.float64, torch.int64]


def _grid(ht, wd):
    yy, xx = torch.meshgrid(torch.arange(ht), torch.arange(wd), indexing="ij")
    return torch.stack([xx, yy], -1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ht,wd", [(40, 64), (80, 128), (3, 7)])
def test_whole_coordinates_name_their_own_pixel(ht, wd, dtype):
    """Coordinates up to 128 are exact in every type."""
    want = torch.arange(ht * wd, dtype=torch.int32).view(ht, wd)
    c = _grid(ht, wd).to(dtype)
    assert torch.equal(nearest_targets(c, ht, wd), want)
    idx, logw = bilinear_targets(c, ht, wd)
    assert torch.equal(idx[..., 0], want) and not logw[..., 0].any()
    assert (logw[..., 1:] == -float("inf")).all() and idx.max() == ht * wd - 1


@pytest.mark.parametrize("dtype", TYPES[:4])
def test_fractions_and_the_border(dtype):
    """Halves and quarters are exact in every type here: as in float64."""
    c = _grid(12, 30).double() * 1.25 - 1.5
    for fn in (nearest_targets, bilinear_targets):
        got, want = fn(c.to(dtype), 11, 29), fn(c, 11, 29)
        for p, q in zip(got if isinstance(got, tuple) else [got], want if isinstance(want, tuple) else [want]):
            assert p.dtype == q.dtype and torch.equal(p, q)


def test_maps_wider_than_a_half_type_counts():
    """2049 columns: the border itself is no number of the coordinates' type."""
    c = torch.tensor([[2048.0, 0.0], [2050.0, 0.0], [float("inf"), 0.0], [0.0, float("nan")]]).half()
    assert nearest_targets(c, 1, 2049).tolist() == [2048, -1, -1, -1]
    assert bilinear_targets(c, 1, 2049)[0][:, 0].tolist() == [2048, -1, -1, -1]


def test_valid_as_reproject_returns_it():
    c = _grid(4, 6).float().expand(3, 4, 6, 2)
    valid = (torch.rand(3, 4, 6, 1, generator=torch.Generator().manual_seed(0)) > 0.5).float()
    for fn in (lambda v: nearest_targets(c, 4, 6, v), lambda v: bilinear_targets(c, 4, 6, v)[0]):
        assert torch.equal(fn(valid), fn(valid[..., 0]))
        assert (fn(valid) < 0).any() and (fn(valid) >= 0).any()
        assert torch.equal(fn(torch.ones(4, 6)), fn(None))
        with pytest.raises(RuntimeError):
            fn(torch.ones(5, 3, 4, 6))
        with pytest.raises(RuntimeError):
            fn(torch.ones(3, 3, 4, 6, 1))
