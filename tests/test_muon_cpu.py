"""What fi_muon_step refuses before anything reaches the device: no launch is made, so nothing has moved when it returns."""
import ctypes as C

import pytest

from fedicra_amd import _lib as L


def _step(coeffs, steps=5, rows=4, cols=6):
    """fi_muon_step on addresses that only a kernel would read."""
    mats = (L.FiMuonMat * 1)(L.FiMuonMat(256, 512, 1024, rows, cols, 1.0))
    flat = (C.c_float * (3 * max(steps, 1)))(*(list(coeffs) * max(steps, 1)))
    return L.lib().fi_muon_step(mats, 1, C.c_void_p(2048), C.c_float(0.95), 1, C.c_float(0.0), steps, flat, C.c_float(1e-7), None, C.c_void_p(4096), None)


@pytest.mark.parametrize("coeffs", [(20.0, 0.0, 0.0), (3.4445, 4.775, 2.0315), (float("nan"), 0.0, 0.0), (4.0, 0.0, 0.0)])
def test_a_polynomial_out_of_range_is_refused_before_the_momentum_moves(coeffs):
    assert _step(coeffs) == L.FI_ERR_UNSUPPORTED


def test_steps_and_sizes_are_refused_before_the_momentum_moves():
    assert _step((3.4445, -4.775, 2.0315), steps=0) == -2
    assert _step((3.4445, -4.775, 2.0315), rows=0) == -2
