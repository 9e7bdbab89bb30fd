"""Calls that the correlation losses refuse on the host, through the C ABI: pointers
are never read, each call ends at its check."""
import pytest

from test_corr_loss_cpu import OK, _backward, _forward


def _says():
    from droid_backends._lib import lib
    return lib.droid_last_error().decode()


@pytest.mark.parametrize("scale,T", [(1e-38, 10.0), (1e-30, 1e10), (1e30, 1e-10), (1e30, 1e10), (1.0, 1e20), (1e-20, 1e-20),
                                     (1e-3, 1e-19)])
def test_scales_that_leave_fp32(scale, T):
    """0 times -inf (a key past the end) is NaN, as is an infinite temperature^2 times 0."""
    for call in (_forward, _backward):
        assert call({**OK, "scale": scale, "T": T}) != 0 and "normal numbers" in _says()


def test_more_edges_than_the_gradient_searches():
    """Each edge looks for its reverse in the whole list: 10^6 edges would take
    seconds to minutes, however small the frames."""
    many = {**OK, "E": 65537, "P": 1, "Q": 1}
    assert _backward(many) != 0 and "65536 edges" in _says()
    assert _backward({**many, "E": 65536, "wsb": 3}) != 0 and "workspace" in _says()
    assert _forward({**many, "wsb": 3}) != 0 and "workspace" in _says()
