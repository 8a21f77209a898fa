"""ops.linear_ce_loss where sizes differ by many orders: rows' own factors, rows, classes and features of fp32 operands."""
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


SIZES = [(300, 400, 200), (64, 2000, 40), (600, 50, 33), (100, 700, 72), (300, 100, 72)]


@pytest.mark.parametrize("big", [1e6, 1e10, 1e30, torch.finfo(F32).max])
@pytest.mark.parametrize("rows,classes,width", SIZES)
def test_a_large_value_in_one_row_leaves_the_others_alone(rows, classes, width, big):
    """A labelled row whose one feature is far larger than all else.  It is its own class for certain (no gradient): losses and dx of the other rows, dw and db
    are those of the other rows alone."""
    x, w, b, lab = _head(rows, rows, classes, width, F32, 0.1)
    x[0, 3] = big
    w[:, 3] *= 0.2
    w[7, 3] = 0.9
    lab[0], lab[1] = 7, 5
    loss, dx, dw, db = _none(x, w, b, lab)
    assert float(loss[0]) == 0.0 and not dx[0].any()
    want, tol = _ce64(x[1:], w, b, lab[1:], -100, "none", torch.ones(rows - 1, device="cuda"))
    _within(loss[1:], want[0], tol[0], ("loss", F32))
    _within(dx[1:], want[1], tol[1], ("dx", F32))
    _within(dw, want[2], tol[2], ("dw", F32))
    _within(db, want[3], tol[3], ("db", F32))


@pytest.mark.parametrize("big", [1e6, 1e10, 1e30, torch.finfo(F32).max])
@pytest.mark.parametrize("rows,classes,width", SIZES)
def test_a_large_weight_of_one_class_leaves_the_others_alone(rows, classes, width, big):
    """A class that one huge weight rules out for every row: everything else is as without it."""
    x, w, b, lab = _head(rows, rows, classes, width, F32, 0.1)
    x[:, 3] = -0.5 - 0.4 * torch.rand(rows, generator=_gen(1), device="cuda")
    lab = torch.where(lab == 7, torch.full_like(lab, 8), lab)
    w[7, 3] = big
    loss, dx, dw, db = _none(x, w, b, lab)
    kept = torch.arange(classes, device="cuda") != 7
    want, tol = _ce64(x, w[kept], b[kept], torch.where(lab > 7, lab - 1, lab), -100, "none", torch.ones(rows, device="cuda"))
    _within(loss, want[0], tol[0], ("loss", F32))
    _within(dx, want[1], tol[1], ("dx", F32))
    _within(dw[kept], want[2], tol[2], ("dw", F32))
    _within(db[kept], want[3], tol[3], ("db", F32))
    assert not dw[7].any() and float(db[7]) == 0.0


@pytest.mark.parametrize("rows,classes,width", SIZES)
def test_features_of_unlike_size(rows, classes, width):
    """Features from 1e-8 to 1e8 whose weights make up for it."""
    x, w, b, lab = _head(rows, rows, classes, width, F32, 0.1)
    s = 10.0 ** (torch.rand(width, generator=_gen(2), device="cuda") * 16 - 8)
    x, w = x * s, w / s
    above = torch.ones(rows, device="cuda")
    loss, dx, dw, db = _none(x, w, b, lab)
    want, tol = _ce64(x, w, b, lab, -100, "none", above)
    _within(loss, want[0], tol[0], ("loss", F32))
    _within(dx, want[1], tol[1], ("dx", F32))
    _within(dw, want[2], tol[2], ("dw", F32))
    _within(db, want[3], tol[3], ("db", F32))


def test_tens_of_millions_of_rows():
    """So many that the labelled ones before a workgroup's are counted by a scan; few are labelled."""
    rows, classes, width = 36_000_000, 5, 2
    g = _gen(7)
    x = torch.randn(rows, width, generator=g, device="cuda").to(BF16)
    w, b = torch.randn(classes, width, generator=g, device="cuda").to(BF16), torch.randn(classes, generator=g, device="cuda")
    lab = torch.full((rows,), 255, dtype=torch.uint8, device="cuda")
    at = torch.unique(torch.randint(0, rows, (40000,), generator=g, device="cuda"))
    at[0], at[-1] = 0, rows - 1
    lab[at] = torch.randint(0, classes, at.shape, generator=g, device="cuda").to(torch.uint8)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    loss = ops.linear_ce_loss(*leaves, lab, 255)
    dx, dw, db = torch.autograd.grad(loss, leaves)
    want, tol = _ce64(x[at], w, b, lab[at], 255, "mean", torch.ones((), device="cuda"))
    _within(loss.detach().reshape(1), want[0].reshape(1), tol[0], ("loss", F32))
    _within(dx[at], want[1], tol[1], ("dx", BF16))
    _within(dw, want[2], tol[2], ("dw", BF16))
    _within(db, want[3], tol[3], ("db", F32))
    dx[at] = 0
    assert not dx.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_lone_row_or_class_of_any_stride(dtype):
    """What a slice of a large tensor leaves: one row, its stride far beyond what several rows may have."""
    store = torch.randn(1 << 10, generator=_gen(8), device="cuda").to(dtype)
    x = store.as_strided((1, 24), (1 << 40, 1))
    w = store.as_strided((1, 24), (1 << 23, 1), 512)
    b = torch.zeros(1, device="cuda")
    loss, dx, dw, db = _none(x, w, b, torch.zeros(1, dtype=torch.int64, device="cuda"))
    assert float(loss[0]) == 0.0 and not dx.any() and not dw.any() and not db.any()
    lab = torch.zeros(50, dtype=torch.int64, device="cuda")
    loss, dx, dw, db = _none(torch.randn(50, 24, generator=_gen(9), device="cuda").to(dtype), w, b, lab)
    assert not loss.any() and not dx.any() and not dw.any() and not db.any()
    w = torch.randn(30, 24, generator=_gen(10), device="cuda").to(dtype)
    b = torch.randn(30, generator=_gen(11), device="cuda")
    loss, dx, dw, db = _none(x, w, b, lab[:1])
    want, tol = _ce64(x, w, b, lab[:1], -100, "none", torch.ones(1, device="cuda"))
    _within(loss, want[0], tol[0], ("loss", F32))
    _within(dx, want[1], tol[1], ("dx", dtype))
    _within(dw, want[2], tol[2], ("dw", dtype))
    _within(db, want[3], tol[3], ("db", F32))


@pytest.mark.parametrize("size", [1e-32, 1e30])
def test_features_next_to_the_ends_of_the_range(size):
    x, w, b, lab = _head(12, 300, 400, 72, F32, 0.1)
    x, w = (x.double() * size).float(), (w.double() / size).float()
    loss, dx, dw, db = _none(x, w, b, lab)
    want, tol = _ce64(x, w, b, lab, -100, "none", torch.ones(300, device="cuda"))
    _within(loss, want[0], tol[0], ("loss", F32))
    _within(dx, want[1], tol[1], ("dx", F32))
    _within(dw, want[2], tol[2], ("dw", F32))
    _within(db, want[3], tol[3], ("db", F32))
