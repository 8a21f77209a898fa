"""ops.linear_ce_loss where classes are ruled out by a large finite bias, and where a row's sum runs over thousands of tiles."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fedicra_amd import ops  # noqa: E402
from test_linear_ce_gpu import BF16, F16, F32, _ce64, _head, _within  # noqa: E402


# rows, classes, features: up to 128 features, more, up to 64 rows; half precision above 2^28 multiply-adds, below which it takes the form of fp32
FORMS = [(BF16, 300, 700, 72), (BF16, 300, 900, 200), (BF16, 37, 900, 96), (BF16, 100, 900, 300), (F16, 3000, 1000, 100), (F16, 1500, 1000, 200),
         (F16, 60, 40000, 128), (F16, 300, 700, 72), (F32, 300, 700, 72)]


@pytest.mark.parametrize("mask", [-1e9, -1e10, -1e20, -1e30, torch.finfo(F32).min, -math.inf])
@pytest.mark.parametrize("dtype,rows,classes,width", FORMS)
def test_classes_ruled_out_by_their_bias(dtype, rows, classes, width, mask):
    """Whole tiles of them, the first and the last among them: what is left is the loss of the other classes, exactly."""
    x, w, b, lab = _head(rows + classes, rows, classes, width, dtype, 0.1)
    kept = torch.zeros(classes, dtype=torch.bool, device="cuda")
    kept[290:310] = True
    kept[classes // 2:classes // 2 + 3] = True
    which = kept.nonzero()[:, 0]
    local = torch.where(lab == -100, lab, lab % len(which))
    lab = torch.where(lab == -100, lab, which[local.clamp(min=0)])
    b = torch.where(kept, b, torch.full_like(b, mask))
    up = torch.full((), 64.0 if dtype == F16 else 1.0, device="cuda")
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    loss = ops.linear_ce_loss(*leaves, lab)
    dx, dw, db = torch.autograd.grad(loss, leaves, up)
    want, tol = _ce64(x, w[which], b[which], local, -100, "mean", up)      # (exp(-1e9) is zero in 64 bits too)
    _within(loss.detach().reshape(1), want[0].reshape(1), tol[0], ("loss", F32))
    _within(dx, want[1], tol[1], ("dx", dtype))
    _within(dw[which], want[2], tol[2], ("dw", dtype))
    _within(db[which], want[3], tol[3], ("db", F32))
    assert not dw[~kept].any() and not db[~kept].any()


@pytest.mark.parametrize("mask", [-1e10, -1e30, torch.finfo(F32).min])
@pytest.mark.parametrize("dtype,rows,classes,width", FORMS)
def test_rows_whose_classes_are_all_ruled_out_alike(dtype, rows, classes, width, mask):
    """The bias drowns every product: V equal logits."""
    x, w, b, lab = _head(rows, rows, classes, width, dtype, 0.1)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, torch.full_like(b, mask))]
    loss = ops.linear_ce_loss(*leaves, lab, -100, "none")
    grads = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
    part = loss[lab != -100].double()
    # (a sum of ones, its 1 / sum and logarithm: some roundings of fp32)
    assert float((part - math.log(classes)).abs().max()) <= 2.0 ** -20 * math.log(classes) and all(torch.isfinite(g).all() for g in grads)
    n = int((lab != -100).sum())
    want = torch.full((classes,), n / classes, dtype=torch.float64, device="cuda") - torch.bincount(lab[lab != -100], minlength=classes)
    # a label's entry is rounded to 11 bits or better, the others' n entries too
    assert float(((grads[2].double() - want).abs() - 2.0 ** -11 * (n / classes + want.abs())).max()) <= 2.0 ** -20


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
