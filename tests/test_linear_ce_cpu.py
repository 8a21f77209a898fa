"""What linear_ce_loss and newton_schulz refuse before anything reaches the device."""
import pytest
import torch

from fedicra_amd import _lib as L
from fedicra_amd import ops

X, W, B, Y = torch.zeros(6, 8), torch.zeros(5, 8), torch.zeros(5), torch.zeros(6, dtype=torch.int64)


@pytest.mark.parametrize("x,w,b,y,kw", [
    (X, torch.zeros(5, 7), B, Y, {}), (X, W, torch.zeros(4), Y, {}), (X, W, B, torch.zeros(5, dtype=torch.int64), {}),
    (X, torch.zeros(5, 8, 3, 3), B, Y, {}), (X, torch.zeros(8), B, Y, {}), (torch.zeros(0, 8), W, B, torch.zeros(0, dtype=torch.int64), {}),
    (X, torch.zeros(0, 8), torch.zeros(0), Y, {}), (X, W, B, Y, {"reduction": "batchmean"}),
])
def test_linear_ce_refuses_arguments_that_do_not_go_together(x, w, b, y, kw):
    with pytest.raises(ValueError):
        ops.linear_ce_loss(x, w, b, y, **kw)


def test_linear_ce_has_no_cpu_path():
    with pytest.raises(L.FiError):
        ops.linear_ce_loss(X, W, B, Y)
    with pytest.raises(L.FiError):
        ops.linear_ce_loss(X, W, B, Y.float())
    with pytest.raises(L.FiError):
        ops.linear_ce_loss(X.bfloat16(), W.half(), B, Y)


@pytest.mark.parametrize("u,kw", [
    (torch.zeros(3), {}), (torch.zeros(2, 2, 2, 2), {}), ([torch.zeros(3)], {}), ([torch.zeros(0, 3)], {}), (torch.zeros(3, 3), {"steps": 0}),
    (torch.zeros(3, 3), {"coeffs": (1.0, 2.0)}), (torch.zeros(3, 3), {"steps": 2, "coeffs": [(1.0, 0.0, 0.0)] * 3}),
    (torch.zeros(3, 3), {"eps": -1.0}), (torch.zeros(3, 3), {"eps": float("nan")}),
])
def test_newton_schulz_refuses(u, kw):
    with pytest.raises(ValueError):
        ops.newton_schulz(u, **kw)


def test_newton_schulz_has_no_cpu_path_and_takes_nothing():
    with pytest.raises(L.FiError):
        ops.newton_schulz(torch.ones(3, 3))
    assert ops.newton_schulz([]) == []
