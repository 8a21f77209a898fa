"""ops.linear_ce_loss where sizes differ by many orders: rows' own factors."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from fedicra_amd import ops  # noqa: E402
from test_linear_ce_gpu import BF16, F16, F32, _ce64, _gen, _head, _within  # noqa: E402


def _none(x, w, b, lab, above=None):
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    loss = ops.linear_ce_loss(*leaves, lab, -100, "none")
    return (loss.detach(), *torch.autograd.grad(loss, leaves, torch.ones_like(loss) if above is None else above))


@pytest.mark.parametrize("dtype,rows,classes,width", [(F32, 300, 400, 200), (F32, 600, 800, 72), (BF16, 600, 800, 200), (BF16, 60, 900, 300), (BF16, 100, 900, 300),
                                                      (BF16, 700, 300, 72), (F16, 1500, 1000, 200), (F16, 300, 400, 200), (BF16, 70000, 5000, 136)])
def test_a_row_of_dx_knows_its_own_factor_alone(dtype, rows, classes, width):
    """Factors over twelve orders (eight where dx is fp16): every row of dx is as good as if its factor were the only one."""
    x, w, b, lab = _head(rows + width, rows, classes, width, dtype, 0.2)
    lab[0] = 1
    e = torch.rand(rows, generator=_gen(5), device="cuda") * (8 if dtype == F16 else 12)
    above = 10.0 ** ((4 if dtype == F16 else 0) - e) * torch.where(torch.rand(rows, generator=_gen(6), device="cuda") < 0.5, 1.0, -1.0)
    loss, dx, dw, db = _none(x, w, b, lab, above)
    one = torch.ones(rows, device="cuda")
    for lo in range(0, rows, 10000):
        sl = slice(lo, lo + 10000)
        want, tol = _ce64(x[sl], w, b, lab[sl], -100, "none", one[sl])         # dx of a factor of one, and its tolerance, times the row's own
        _within(loss[sl], want[0], tol[0], ("loss", F32))
        g = above[sl, None].double()
        _within(dx[sl], want[1] * g, tol[1] * g.abs(), ("dx", dtype))
    if rows <= 10000:
        want, tol = _ce64(x, w, b, lab, -100, "none", above)
        _within(dw, want[2], tol[2], ("dw", dtype))
        _within(db, want[3], tol[3], ("db", F32))
