"""ops.linear_ce_loss against its definition in 64 bits, at the sizes, types, masks and layouts where it can go wrong."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fedicra_amd import _lib as L  # noqa: E402
from fedicra_amd import ops  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ce64(x, w, b, labels, ignore, reduction, above):
    """loss, dx, dw, db and what each may be off by (see _ce_check)."""
    x2, w2 = x.detach().double().reshape(-1, x.shape[-1]), w.detach().double().reshape(w.shape[0], -1)
    lab = labels.reshape(-1).long()
    keep = (lab != ignore).nonzero()[:, 0]
    xs, ls = x2[keep], lab[keep]
    z = xs @ w2.t()
    if b is not None:
        z = z + b.detach().double()
    lse = torch.logsumexp(z, 1)
    rows = torch.zeros(x2.shape[0], dtype=torch.float64, device=x.device)
    rows[keep] = lse - z[torch.arange(len(ls)), ls]
    loss = rows if reduction == "none" else rows.sum() / (len(ls) if reduction == "mean" else 1)
    g = above.double().reshape(-1)[keep] if reduction == "none" else above.double() / (len(ls) if reduction == "mean" else 1)
    p = torch.exp(z - lse[:, None])
    G = p.clone()
    G[torch.arange(len(ls)), ls] -= 1.0
    G = G * (g[:, None] if reduction == "none" else g)
    dx = torch.zeros_like(x2)
    dx[keep] = G @ w2
    # a logit is off by at most its products' accumulation (D fp32 additions; pairs leave 2^-21 of each product besides)
    mag = (xs.abs() @ w2.abs().t()).amax() + (0 if b is None else b.detach().double().abs().max())
    pair = x.dtype == F32
    dz = float(mag) * ((x.shape[-1] + 2) * 2.0 ** -24 + (2.0 ** -21 if pair else 0.0)) + 2.0 ** -22 * float(z.abs().max())
    # so a probability by 2 dz of itself (its row's sum moves too); G is rounded to fp16 (half a step: 2^-12, and 2^-25 of the largest factor where
    # fp16 runs out of exponents) or kept as a pair; its product is accumulated in fp32
    rel = 2 * dz + (2.0 ** -21 if pair else 2.0 ** -11)
    gmax = float(g.abs().max()) if len(ls) else 0.0
    Gerr = rel * G.abs() + rel * p * (g.abs()[:, None] if reduction == "none" else abs(g)) + gmax * 2.0 ** -38
    n = max(w2.shape[0], len(ls), 1)
    acc = min(n, 4096) * 2.0 ** -24
    tdx = torch.zeros_like(dx)
    tdx[keep] = Gerr @ w2.abs() + acc * (G.abs() @ w2.abs()) + 2.0 ** -21 * (G.abs() @ w2.abs())
    tdw = Gerr.t() @ xs.abs() + (acc + 2.0 ** -21) * (G.abs().t() @ xs.abs())
    tdb = Gerr.sum(0) + 2.0 ** -22 * G.abs().sum(0)
    tl = (2 * dz + 2.0 ** -20) * (1 + (0 if reduction != "sum" else len(ls)))
    return (loss, dx.reshape(x.shape), G.t() @ xs, G.sum(0)), (tl, tdx.reshape(x.shape), tdw, tdb)


def _within(got, want, tol, what):
    got = got.double().reshape(want.shape)
    assert torch.isfinite(got).all(), what
    half = torch.finfo(what[1]).eps / 2
    over = (got - want).abs() - tol - half * want.abs() - torch.finfo(what[1]).tiny * half * 2
    assert float(over.max()) <= 0.0, (what, float(over.max()), float((got - want).abs().max()))


def _ce_check(x, w, b, labels, ignore=-100, reduction="mean", above=None):
    if above is None:
        above = torch.ones((), device=x.device)
    leaves = [t.detach().requires_grad_(True) for t in (x, w)] + ([] if b is None else [b.detach().requires_grad_(True)])
    loss = ops.linear_ce_loss(leaves[0], leaves[1], None if b is None else leaves[2], labels, ignore, reduction)
    assert loss.dtype == F32
    grads = torch.autograd.grad(loss, leaves, above.reshape(loss.shape).to(loss.dtype))
    want, tol = _ce64(x, w, b, labels, ignore, reduction, above)
    _within(loss.detach().reshape(-1), want[0].reshape(-1), tol[0], ("loss", F32))
    for k, (g, leaf) in enumerate(zip(grads, leaves)):
        assert g.shape == leaf.shape and g.dtype == leaf.dtype
        _within(g, want[k + 1].reshape(g.shape), tol[k + 1].reshape(g.shape), (("dx", "dw", "db")[k], g.dtype))
    return loss, grads


def _head(seed, rows, classes, width, dtype, ignored=0.0, wdtype=None):
    g = _gen(seed)
    x = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
    w = (torch.randn(classes, width, generator=g, device="cuda") * (1.5 / math.sqrt(width))).to(dtype)
    b = torch.randn(classes, generator=g, device="cuda") * 0.3
    lab = torch.randint(0, classes, (rows,), generator=g, device="cuda")
    lab[torch.rand(rows, generator=g, device="cuda") < ignored] = -100
    return x, w.to(wdtype or dtype), b, lab


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,classes,width", [(1, 1, 1), (1, 2, 8), (3, 7, 9), (16, 1000, 256), (64, 65, 64), (65, 64, 96), (63, 300, 33), (257, 257, 129),
                                                (300, 513, 64), (513, 105, 16), (2049, 33, 40), (4500, 700, 200), (100, 300, 130), (128, 1000, 190), (129, 1000, 190)])
def test_linear_ce_sizes_and_types(rows, classes, width, dtype):
    x, w, b, lab = _head(rows + classes, rows, classes, width, dtype, 0.2 if rows > 3 else 0.0)
    lab[0] = classes - 1
    up = torch.full((), 256.0 if dtype == F16 else 1.0, device="cuda")
    _ce_check(x, w, b, lab, above=up)
    _ce_check(x, w, None, lab, reduction="sum")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linear_ce_rows_of_losses_with_their_own_gradients(dtype):
    x, w, b, lab = _head(1, 700, 300, 72, dtype, 0.4)
    above = torch.randn(700, generator=_gen(2), device="cuda") * 10.0 ** torch.randint(-4, 3, (700,), generator=_gen(3), device="cuda")
    loss, grads = _ce_check(x, w, b, lab, reduction="none", above=above)
    assert (loss[lab == -100] == 0).all() and (grads[0][lab == -100] == 0).all()


def test_linear_ce_keeps_sizes_types_and_layouts():
    x, w, b, lab = _head(4, 6 * 5 * 7, 40, 24, BF16, 0.3)
    lab = torch.where(lab == -100, torch.full_like(lab, 255), lab)
    for lt in (torch.int64, torch.int32, torch.uint8):
        a = _ce_check(x.reshape(6, 5, 7, 24), w.reshape(40, 24, 1, 1), b, lab.reshape(6, 5, 7).to(lt), ignore=255)
    want = ops.linear_ce_loss(x, w, b, lab, 255)
    assert torch.equal(a[0], want)
    wide = torch.randn(100, 3, 48, generator=_gen(5), device="cuda").to(BF16)
    lab = torch.randint(0, 40, (100,), generator=_gen(6), device="cuda")
    _ce_check(wide[:, 1, :24], w, b, lab)                              # rows far apart
    _ce_check(wide[:, 1, ::2], w, b, lab)                              # features far apart
    _ce_check(wide[:, 2, 1:25], w.t().contiguous().t(), b, lab)        # unaligned rows, a transposed weight
    row = torch.randn(24, generator=_gen(9), device="cuda").to(BF16)
    _ce_check(row.expand(100, 24), w, b, lab)                          # every row the same memory
    _ce_check(torch.randn(123, generator=_gen(10), device="cuda").to(BF16).as_strided((100, 24), (1, 1)), w, b, lab)     # overlapping rows
    _ce_check(wide[:, 0, :24], w[:1].expand(40, 24), b, lab)
    _ce_check(wide[:1, 0, :24], w, b, lab[:1])
    big = torch.randn(70, 200, generator=_gen(7), device="cuda").to(F16)
    _ce_check(big[:, 4:132], (torch.randn(50, 300, generator=_gen(8), device="cuda") * 0.1).to(F16)[:, 3:131], None, lab[:70], above=torch.full((), 64.0, device="cuda"))


def test_linear_ce_parameter_in_fp32_under_16_bit_features():
    x, w, b, lab = _head(9, 500, 90, 48, BF16, 0.1)
    w32 = (w.float() * 1.001).requires_grad_(True)                    # not a bf16 value
    loss = ops.linear_ce_loss(x, w32, b, lab)
    loss.backward()
    xr, wr = x.detach().requires_grad_(True), w32.detach().to(BF16)
    want, tol = _ce64(xr, wr, b, lab, -100, "mean", torch.ones((), device="cuda"))
    _within(loss.detach().reshape(1), want[0].reshape(1), tol[0], ("loss", F32))
    assert w32.grad.dtype == F32
    _within(w32.grad, want[2], tol[2], ("dw", F32))


@pytest.mark.parametrize("dtype,rows,classes,width", [(F16, 300, 200, 72), (F16, 4000, 700, 100), (BF16, 300, 200, 72), (BF16, 300, 200, 200)])
def test_linear_ce_fp32_weights_meet_16_bit_features_rounded(dtype, rows, classes, width):
    """fp32 weights are the 16-bit type's in the product and in dx, whatever form the sizes choose."""
    x, w, b, lab = _head(31, rows, classes, width, dtype, 0.1, F32)
    w = w + 1e-4 * torch.randn(w.shape, generator=_gen(32), device="cuda")          # (no longer the type's own values)
    got = []
    for v in (w, w.to(dtype).float()):
        leaves = [x.detach().requires_grad_(True), v.detach().requires_grad_(True)]
        loss = ops.linear_ce_loss(*leaves, b, lab)
        got.append([loss.detach(), *torch.autograd.grad(loss, leaves)])
    assert all(torch.equal(p, q) for p, q in zip(*got))


def test_linear_ce_everything_ignored_and_nothing_ignored():
    x, w, b, lab = _head(10, 300, 20, 16, BF16)
    none = torch.full_like(lab, -100)
    for red in ("mean", "sum", "none"):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        loss = ops.linear_ce_loss(*leaves, none, -100, red)
        assert torch.isnan(loss) if red == "mean" else (loss == 0).all()
        grads = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
        assert all((g == 0).all() for g in grads)
    only = none.clone()
    only[137] = 3
    _ce_check(x, w, b, only)


def test_linear_ce_what_stands_in_ignored_rows_does_not_matter():
    x, w, b, lab = _head(11, 400, 33, 24, F32, 0.5)
    want = _ce_check(x, w, b, lab)
    y = x.clone()
    bad = (lab == -100).nonzero()[:, 0]
    y[bad[0::3]], y[bad[1::3]], y[bad[2::3]] = math.nan, math.inf, torch.finfo(F32).min
    leaves = [t.detach().requires_grad_(True) for t in (y, w, b)]
    loss = ops.linear_ce_loss(*leaves, lab)
    grads = torch.autograd.grad(loss, leaves)
    assert torch.equal(loss, want[0]) and all(torch.equal(a, c) for a, c in zip(grads, want[1]))


def test_linear_ce_labels_that_are_no_class_and_values_that_are_no_numbers():
    for at in (-1, 20, 2 ** 40):
        x, w, b, lab = _head(12, 300, 20, 16, BF16)
        lab[7] = at
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        rows = ops.linear_ce_loss(*leaves, lab, -100, "none")
        assert torch.isnan(rows[7]) and torch.isfinite(rows[:7]).all() and torch.isfinite(rows[8:]).all()
        dx, dw, db = torch.autograd.grad(rows, leaves, torch.ones_like(rows))
        assert torch.isnan(dx[7]).all() and torch.isfinite(dx[8:]).all() and torch.isnan(dw).all() and torch.isnan(db).all()
    x, w, b, lab = _head(13, 300, 20, 16, F32)
    x[5, 3] = math.inf
    rows = ops.linear_ce_loss(x, w, b, lab, -100, "none")
    assert not torch.isfinite(rows[5]) and torch.isfinite(rows[:5]).all() and torch.isfinite(rows[6:]).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_linear_ce_logits_far_apart(dtype):
    x, w, b, lab = _head(14, 200, 90, 32, dtype)
    b = b * 1000.0                                                     # all but one class underflow
    rows = ops.linear_ce_loss(x, w, b, lab, -100, "none")
    want, tol = _ce64(x, w, b, lab, -100, "none", torch.ones(200, device="cuda"))
    _within(rows, want[0], tol[0], ("loss", F32))
    b = torch.full_like(b, -math.inf)                                  # classes that are ruled out
    b[:3] = 0.0
    loss = ops.linear_ce_loss(x, w, b, lab % 3)
    assert torch.allclose(loss.double(), _ce64(x, w[:3], b[:3], lab % 3, -100, "mean", torch.ones((), device="cuda"))[0][0], atol=1e-4)


def test_linear_ce_gradient_against_differences():
    x, w, b, lab = _head(15, 60, 30, 20, F32, 0.2)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(ops.linear_ce_loss(*leaves, lab), leaves)
    for k, t in enumerate((x, w, b)):
        step = torch.randn(t.shape, generator=_gen(16 + k), device="cuda")
        h = 1e-2
        hi, lo = [[a + s * h * step if i == k else a for i, a in enumerate((x, w, b))] for s in (1, -1)]
        diff = (ops.linear_ce_loss(*hi, lab).double() - ops.linear_ce_loss(*lo, lab).double()) / (2 * h)
        slope = (grads[k].double() * step.double()).sum()
        # the difference quotient: h^2 / 6 of the third derivative (|x step|^3 at most), and the losses' own 2^-20 over h
        size = float(step.norm()) * (1.0 if k else 1.0)
        assert abs(float(diff - slope)) <= h * h * size ** 2 + 2.0 ** -19 / h, (k, float(diff), float(slope))


def test_linear_ce_needs_only_some_gradients():
    x, w, b, lab = _head(17, 300, 70, 40, BF16, 0.1)
    _, full = _ce_check(x, w, b, lab)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1)):
        leaves = [t.detach().requires_grad_(bool(n)) for t, n in zip((x, w, b), need)]
        loss = ops.linear_ce_loss(*leaves, lab)
        got = torch.autograd.grad(loss, [t for t, n in zip(leaves, need) if n])
        assert all(torch.equal(a, c) for a, c in zip(got, [f for f, n in zip(full, need) if n]))


def test_linear_ce_in_pieces_equals_the_definition():
    """More rows x classes than one piece holds: class pieces, row pieces, and both."""
    for rows, classes, width, dtype in ((70000, 5000, 136, BF16), (1100000, 300, 132, F16), (1200, 230000, 24, F32), (70000, 5000, 16, BF16)):
        x, w, b, lab = _head(rows, rows, classes, width, dtype, 0.05)
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        loss = ops.linear_ce_loss(*leaves, lab)
        dx, dw, db = torch.autograd.grad(loss, leaves)
        # against the definition, accumulated over chunks of rows in 64 bits
        n = int((lab != -100).sum())
        one = torch.ones((), device="cuda")
        tot, gw, gb, tw, tb = 0.0, 0.0, 0.0, 0.0, 0.0
        for lo in range(0, rows, 40000 if classes < 10000 else 300):
            sl = slice(lo, min(rows, lo + (40000 if classes < 10000 else 300)))
            k = int((lab[sl] != -100).sum())
            want, tol = _ce64(x[sl], w, b, lab[sl], -100, "mean", one * (k / n))
            tot, gw, gb, tw, tb = tot + float(want[0]) * k / n, gw + want[2], gb + want[3], tw + tol[2], tb + tol[3]
            _within(dx[sl], want[1], tol[1], ("dx", dtype))
        assert abs(float(loss) - tot) <= 1e-5 * tot
        _within(dw, gw, tw, ("dw", dtype))
        _within(db, gb, tb, ("db", F32))


def test_linear_ce_is_repeatable_and_runs_on_any_stream():
    x, w, b, lab = _head(18, 5000, 900, 96, BF16, 0.3)
    first = _ce_check(x, w, b, lab)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        loss = ops.linear_ce_loss(*leaves, lab)
        grads = torch.autograd.grad(loss, leaves)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(loss, first[0]) and all(torch.equal(a, c) for a, c in zip(grads, first[1]))


def test_linear_ce_graph_replays_with_another_number_of_labelled_rows():
    x, w, b, lab = _head(19, 3000, 400, 64, BF16, 0.5)
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]

    def step():
        loss = ops.linear_ce_loss(*leaves, lab)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for k in range(4):
        lab.copy_(_head(20 + k, 3000, 400, 64, BF16, (0.9, 0.0, 0.5, 0.999)[k])[3])
        with torch.no_grad():
            leaves[0].copy_(_head(30 + k, 3000, 400, 64, BF16)[0])
        g.replay()
        torch.cuda.synchronize()
        for a, c in zip(got, step()):
            assert torch.equal(a.nan_to_num(), c.nan_to_num())
        assert bool(torch.isnan(got[0])) == (not (lab != -100).any()) and all(torch.isfinite(t).all() for t in got[1:])


def test_linear_ce_agrees_with_ce_loss_on_its_logits():
    """The operator beside it: the fp32 logits and uint8 labels of ce_loss, four classes."""
    x, w, b, lab = _head(40, 2 * 12 * 12, 4, 16, F32, 0.5)
    lab = torch.where(lab == -100, torch.full_like(lab, 4), lab).to(torch.uint8)
    z = (x.double() @ w.double().t() + b.double()).float().reshape(2, 12, 12, 4).requires_grad_(True)
    want = ops.ce_loss(z, lab.reshape(2, 12, 12), 4)
    xr = x.detach().requires_grad_(True)
    got = ops.linear_ce_loss(xr, w, b, lab, 4)
    assert abs(float(got) - float(want)) <= 2.0 ** -20 * (1 + float(z.abs().max()))
    want.backward()
    got.backward()
    assert (xr.grad - z.grad.reshape(-1, 4) @ w).abs().max() <= 1e-6


def test_refusals_on_the_device():
    x, w, b, lab = _head(50, 20, 10, 8, BF16)
    with pytest.raises(L.FiError):
        ops.linear_ce_loss(x, w.half(), b, lab)
    with pytest.raises(L.FiError):
        ops.linear_ce_loss(x, w, b, lab.float())
    with pytest.raises(L.FiError):
        ops.linear_ce_loss(x.double(), w.double(), b, lab)
    with pytest.raises(L.FiError):
        ops.linear_ce_loss(x, w, b, lab.cpu())
    xr = x.detach().requires_grad_(True)
    (g,) = torch.autograd.grad(ops.linear_ce_loss(xr, w, b, lab), xr, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("rows,classes,width", [(5, 3, 4), (64, 64, 64), (65, 129, 65), (1000, 63, 12), (130, 4000, 128), (20000, 70, 24), (900, 20000, 100)])
def test_linear_ce_narrow_features_keep_the_gradient_in_registers(dtype, rows, classes, width):
    """Up to 128 features: either side streamed in tiles of 64, split or whole, tails on both sides, four or eight values to a vector or none."""
    x, w, b, lab = _head(rows * 3 + classes, rows, classes, width, dtype, 0.1 if rows > 5 else 0.0)
    lab[-1] = classes - 1
    up = torch.full((), 64.0 if dtype == F16 else 1.0, device="cuda")
    _, full = _ce_check(x, w, b, lab, above=up)
    b2 = b.clone()
    b2[0] = 90.0                                                      # a class whose exponential overflows without its row's maximum
    _ce_check(x, w, b2, lab, above=up)
    w32 = w.float().requires_grad_(True)                              # fp32 parameter: the gradient is added to, not rounded
    ops.linear_ce_loss(x, w32, b, lab).backward()
    assert w32.grad.dtype == F32 and torch.isfinite(w32.grad).all()
