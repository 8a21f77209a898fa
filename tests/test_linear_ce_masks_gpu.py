"""ops.linear_ce_loss where a row's sum runs over thousands of tiles."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fedicra_amd import ops  # noqa: E402
from test_linear_ce_gpu import BF16, F16, F32, _ce64, _head, _within  # noqa: E402


@pytest.mark.parametrize("shift", [0.0, -100.0, 300.0])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_a_row_sum_over_two_thousand_tiles(dtype, shift):
    """More than 65536 rows stream the classes in one part; 131072 classes are 2048 tiles."""
    rows, classes, width = 70000, 131072, 16
    x, w, b, lab = _head(3, rows, classes, width, dtype, 0.998)
    b = torch.full_like(b, shift)
    lab[1] = 77
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    loss = ops.linear_ce_loss(*leaves, lab, -100, "none")
    above = torch.full((rows,), 64.0, device="cuda")
    dx, dw, db = torch.autograd.grad(loss, leaves, above)
    want, tol = _ce64(x, w, b, lab, -100, "none", above)
    # the logits' own error (tol: 2 dz + 2^-20) and the row sum's: 2048 additions of a tile and 16 within, each off by 2^-25 of the sum at random
    # (zero on average: a standard deviation of sqrt(2064) 2^-25), six deviations allowed
    bound = tol[0] + 6 * math.sqrt(2064) * 2.0 ** -25
    _within(loss.detach(), want[0], bound, ("loss", F32))
    _within(dx, want[1], tol[1], ("dx", dtype))
    _within(dw, want[2], tol[2], ("dw", dtype))
    _within(db, want[3], tol[3], ("db", F32))
