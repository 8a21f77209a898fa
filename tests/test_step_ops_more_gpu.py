"""The tail of a training step where it meets the flat gradient buffer, differences of the loss, and matrices of unlike size in one call."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from fedicra_amd import ops  # noqa: E402
from test_linear_ce_gpu import BF16, F16, F32, _ce64, _gen, _head, _within  # noqa: E402
from test_muon_gpu import _Head  # noqa: E402
from test_newton_schulz_gpu import _ns64, _update  # noqa: E402


@pytest.mark.parametrize("dtype,rows,classes,width", [
    (BF16, 5, 3, 4), (BF16, 300, 200, 72), (BF16, 500, 90, 50), (BF16, 20000, 70, 23), (BF16, 20000, 70, 24), (BF16, 20000, 70, 126),       # in registers
    (BF16, 300, 400, 200), (BF16, 300, 400, 201), (BF16, 9000, 300, 201), (F16, 1500, 1000, 203), (F16, 3000, 1000, 99),
    (F32, 16, 1000, 256), (F32, 300, 400, 33), (F32, 4001, 900, 77), (F32, 5000, 60, 40), (F16, 300, 100, 70)])
def test_gradients_are_added_to_the_flat_buffer(dtype, rows, classes, width):
    """fp32 parameters of a flat-store model, their gradient buffer not empty: what stood there plus the gradient, nothing beside it touched."""
    x, w, b, lab = _head(rows + width, rows, classes, width, dtype, 0.1 if rows > 5 else 0.0, F32)
    head = _Head(classes, width).cuda()
    with torch.no_grad():
        head.weight.copy_(w)
        head.bias.copy_(b)
    before = torch.randn(head.flat_grads.numel(), generator=_gen(1), device="cuda") * 1e-2
    head.zero_grad()
    head.flat_grads.copy_(before)
    for p in (head.weight, head.bias):
        p.grad = p._fi_gview
    up = torch.full((), 64.0 if dtype == F16 else 1.0, device="cuda")
    ops.linear_ce_loss(x, head.weight, head.bias, lab).backward(up)
    want, tol = _ce64(x, w.to(dtype), b, lab, -100, "mean", up)
    ow, ob = head.weight._fi_off, head.bias._fi_off
    assert head.weight.grad.data_ptr() == head.flat_grads[ow:].data_ptr()
    _within(head.weight.grad, want[2] + before[ow:ow + w.numel()].double().reshape(w.shape), tol[2], ("dw", F32))
    _within(head.bias.grad, want[3] + before[ob:ob + classes].double(), tol[3], ("db", F32))
    rest = torch.ones_like(before, dtype=torch.bool)
    rest[ow:ow + w.numel()] = rest[ob:ob + classes] = False
    assert torch.equal(head.flat_grads[rest], before[rest])


@pytest.mark.parametrize("dtype,rows,classes,width", [(F32, 60, 30, 20), (F32, 300, 200, 150)])
def test_gradient_against_differences_along_itself(dtype, rows, classes, width):
    """A step of length h along the gradient itself changes the loss by h times the gradient's length."""
    args = list(_head(15, rows, classes, width, dtype, 0.2))
    lab = args.pop()
    leaves = [t.detach().requires_grad_(True) for t in args]
    grads = torch.autograd.grad(ops.linear_ce_loss(*leaves, lab), leaves)
    keep = lab != -100
    for k in range(3):
        slope = float(grads[k].double().norm())
        d = (grads[k].double() / slope).float()
        h = 0.05
        ends = []
        for s in (1, -1):
            moved = [a + s * h * d if i == k else a for i, a in enumerate(args)]
            want, tol = _ce64(*moved, lab, -100, "mean", torch.ones((), device="cuda"))
            ends.append((float(ops.linear_ce_loss(*moved, lab)), float(tol[0]) + 2.0 ** -24 * float(want[0])))
        diff = (ends[0][0] - ends[1][0]) / (2 * h)
        # the third derivative is the mean of a third central moment of the logits' change, at most the cube of its spread over the classes; the moved
        # argument is rounded (2^-24 of it, along a gradient of length `slope`), and each loss is off by its tolerance
        u = d.double() @ args[1].double().t() if k == 0 else args[0].double() @ d.double().t() if k == 1 else d.double().expand(rows, classes)
        spread = (u.amax(1) - u.amin(1))[keep]
        bound = h * h / 6 * float((spread ** 3).mean()) + (ends[0][1] + ends[1][1]) / (2 * h) + slope * 2.0 ** -24 * float(args[k].norm()) / h
        assert bound <= slope / 10                                     # (so that a gradient off by a tenth shows)
        assert abs(diff - slope) <= bound, (k, diff, slope, bound)


@pytest.mark.parametrize("m,n", [(17, 40), (20, 300), (31, 31), (48, 700), (64, 576)])
def test_small_matrices_beside_a_larger_one(m, n):
    """Whatever shares their call: off by no more than twice what an iteration in fp32 products leaves."""
    u = _update(m + n, m, n)
    want = _ns64(u)
    x = u / (u.double().square().sum().sqrt() + 1e-7).float()
    for _ in range(5):
        g = x @ x.t()
        x = 3.4445 * x + (-4.7750 * g + 2.0315 * (g @ g)) @ x
    bound = 2 * (x.double() - want).norm().item()
    for others in ([], [_update(1, 100, 200)], [_update(2, 300, 400)], [_update(3, 1000, 1537)]):
        got = ops.newton_schulz([u] + others)[0]
        err = (got.double() - want).norm().item()
        print(m, n, len(others) and tuple(others[0].shape), "%.2e of %.2e" % (err / want.norm().item(), bound / 2 / want.norm().item()))
        assert err <= bound, (err, bound)


@pytest.mark.parametrize("dtype,rows,classes,width", [(F32, 300, 20, 16), (F32, 100, 700, 72), (F32, 20, 300, 40), (F32, 600, 300, 200), (BF16, 300, 400, 200), (BF16, 40, 300, 200),
                                                      (F16, 300, 400, 200), (F16, 3000, 1000, 100), (F16, 1500, 1000, 200)])
def test_no_labelled_row(dtype, rows, classes, width):
    x, w, b, lab = _head(rows, rows, classes, width, dtype)
    lab.fill_(-100)
    for red in ("mean", "sum", "none"):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        loss = ops.linear_ce_loss(*leaves, lab, -100, red)
        assert torch.isnan(loss) if red == "mean" else (loss == 0).all()
        assert all((g == 0).all() for g in torch.autograd.grad(loss, leaves, torch.ones_like(loss)))
