"""ops.newton_schulz against its definition in 64 bits, at the sizes, types and layouts where it can go wrong."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from fedicra_amd import _lib as L  # noqa: E402
from fedicra_amd import ops  # noqa: E402

COEFFS = (3.4445, -4.7750, 2.0315)
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ns64(u, steps=5, coeffs=COEFFS, eps=1e-7):
    x = u.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.square().sum().sqrt() + eps)
    per = [coeffs] * steps if not hasattr(coeffs[0], "__len__") else coeffs
    for a, b, c in per:
        g = x @ x.t()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.t() if tall else x


def _ns_check(got, u, steps=5, coeffs=COEFFS):
    """What the products may leave: X, A, S and their product are each off by 2^-22 of a matrix of norm <= 1 (pairs of fp16), which the remaining steps
    grow at most a-fold each: 4 * a^steps * 2^-22 in the 2-norm over all entries; and the result's own rounding, half a step of its type per entry."""
    want = _ns64(u, steps, coeffs)
    a = 1.0
    for abc in ([coeffs] * steps if not hasattr(coeffs[0], "__len__") else coeffs):
        a *= max(1.0, abs(abc[0]))
    tol = 4 * a * 2.0 ** -22 + torch.finfo(u.dtype).eps / 2 * want.norm().item()
    assert got.shape == u.shape and got.dtype == u.dtype
    err = (got.double() - want).norm().item()
    assert err <= tol, (tuple(u.shape), u.dtype, err, tol)


def _update(seed, m, n, dtype=F32, scale=1e-3):
    g = _gen(seed)
    r = max(1, min(m, n) // 8)
    u = torch.randn(m, r, generator=g, device="cuda") @ torch.randn(r, n, generator=g, device="cuda")
    return (scale * (u + 0.5 * torch.randn(m, n, generator=g, device="cuda"))).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 77), (33, 1), (2, 144), (16, 9), (31, 33), (64, 64), (65, 129), (256, 2304), (257, 300), (1153, 130),
                                 (700, 700), (1030, 1100)])
def test_newton_schulz_sizes_and_types(m, n, dtype):
    u = _update(m * 1000 + n, m, n, dtype, 1.0 if dtype == F16 else 1e-3)
    _ns_check(ops.newton_schulz(u), u)


def test_newton_schulz_of_many_matrices_in_one_call_equals_each_alone():
    shapes = [(3 + 7 * i, 5 + 11 * (i % 9)) for i in range(30)] + [(300, 400), (1100, 1050)]     # more than one launch takes, three tile sizes
    us = [_update(i, m, n) for i, (m, n) in enumerate(shapes)]
    got = ops.newton_schulz(us)
    for u, o in zip(us, got):
        _ns_check(o, u)
    again = ops.newton_schulz(us)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_newton_schulz_short_matrices_keep_their_accuracy_beside_large_ones():
    """A matrix of up to 16 rows is taken through all its steps in 64 bits, whatever it is called with."""
    short = [_update(3, 4, 7), _update(4, 2, 50), _update(5, 900, 16), _update(6, 1, 1)]
    alone = ops.newton_schulz(short)
    large = _update(7, 300, 520)
    mixed = ops.newton_schulz([short[0], large, *short[1:], large])
    for a, b in zip(alone, [mixed[0], *mixed[2:5]]):
        assert torch.equal(a, b)
    assert torch.equal(mixed[1], mixed[5])
    _ns_check(mixed[1], large)
    for u, got in zip(short, alone):
        # X0 and the coefficients as the definition has them up to fp32's half step, 2^-24, each (5 steps of 3 coefficients, eps, the result's own
        # rounding), every one of which moves a value of at most 1.2 by no more than its growth, 3.4445, times itself
        assert (got.double() - _ns64(u)).abs().max().item() <= 17 * 1.2 * 3.4445 * 2.0 ** -24


@pytest.mark.parametrize("shape,dtype", [((5, 70000), F32), ((40000, 16), BF16), ((16, 257), F16), ((255, 3), F32), ((1, 33000), F32)])
def test_newton_schulz_few_rows_over_long_ones(shape, dtype):
    u = _update(70, *shape, dtype, 1.0)
    _ns_check(ops.newton_schulz(u), u)
    _ns_check(ops.newton_schulz(u, steps=33, coeffs=(1.0, 0.0, 0.0)), u, steps=33, coeffs=(1.0, 0.0, 0.0))      # more steps than one launch takes


def test_newton_schulz_batch_strides_and_mixed_types():
    b = torch.stack([_update(i, 24, 50) for i in range(3)])
    for u, o in zip(b, ops.newton_schulz(b)):
        _ns_check(o, u)
    wide = _update(9, 40, 200)
    for u in (wide.t(), wide[:, ::3], wide[5:17, 3:100]):
        _ns_check(ops.newton_schulz(u), u)
    mixed = [_update(1, 20, 30), _update(2, 30, 20, BF16), _update(3, 9, 70, F16, 1.0)]
    for u, o in zip(mixed, ops.newton_schulz(mixed)):
        _ns_check(o, u)


def test_newton_schulz_steps_and_coefficients():
    u = _update(4, 60, 90)
    _ns_check(ops.newton_schulz(u, steps=1), u, steps=1)
    _ns_check(ops.newton_schulz(u, steps=7), u, steps=7)
    per = [(4.0, -6.0, 2.5), (3.0, -4.0, 1.8), (1.5, -0.5, 0.0)]
    _ns_check(ops.newton_schulz(u, steps=3, coeffs=per), u, steps=3, coeffs=per)


def test_newton_schulz_leaves_its_argument_alone_and_takes_unaligned_ones():
    flat = torch.randn(1 + 33 * 70, generator=_gen(60), device="cuda")
    for t in (flat[1:].view(33, 70), flat[1:].half()[:33 * 70].view(33, 70), flat.half()[1:].view(33, 70)):
        keep = t.clone()
        _ns_check(ops.newton_schulz(t), t)
        assert torch.equal(t, keep)


def test_newton_schulz_extreme_values():
    u = torch.zeros(20, 30, device="cuda")
    assert torch.equal(ops.newton_schulz(u), u)                       # nothing to orthogonalise
    for scale in (1e-30, 1e-6, 1e15):                                 # the norm is taken in 64 bits; eps as the definition says
        v = _update(5, 20, 30, scale=scale)
        _ns_check(ops.newton_schulz(v), v)
    one = torch.zeros(70, 90, device="cuda")
    one[13, 17] = -3.0                                                # rank one
    _ns_check(ops.newton_schulz(one), one)
    for bad in (math.nan, math.inf):
        w = _update(6, 20, 30)
        good = _update(7, 33, 10)
        w[3, 4] = bad
        got = ops.newton_schulz([w, good])
        assert torch.isnan(got[0]).all()
        _ns_check(got[1], good)                                       # its neighbour in the launch is not touched


@pytest.mark.parametrize("shape", [(1, 1), (4, 5), (20, 30), (70, 90), (300, 270)])
def test_newton_schulz_of_zeros_without_eps(shape):
    u = torch.zeros(shape, device="cuda")
    assert torch.equal(ops.newton_schulz(u, eps=0.0), u)
    tiny = torch.full(shape, 2.0 ** -130, device="cuda")              # rank one: every entry 1 / sqrt(m n) of the polynomial of 1
    s = 1.0
    for _ in range(5):
        s = COEFFS[0] * s + COEFFS[1] * s ** 3 + COEFFS[2] * s ** 5
    want = s / math.sqrt(u.numel())
    assert (ops.newton_schulz(tiny, eps=0.0).double() - want).norm().item() <= 4 * COEFFS[0] ** 5 * 2.0 ** -22


def test_newton_schulz_graph_replays():
    us = [_update(i, 40 + i, 300, BF16) for i in range(3)]
    eager = ops.newton_schulz(us)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.newton_schulz(us)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.newton_schulz(us)
    keep = [u.clone() for u in us]
    for k in range(3):
        for u, v in zip(us, keep):
            u.copy_(v * (k + 1) if k < 2 else v.flip(0))
        g.replay()
        torch.cuda.synchronize()
        eager = ops.newton_schulz(us)
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


def test_refusals_on_the_device():
    with pytest.raises(L.FiError):
        ops.newton_schulz(torch.randn(4, 4, device="cuda"), steps=5, coeffs=(9.0, 1.0, 1.0))     # grows without bound
    with pytest.raises(L.FiError):
        ops.newton_schulz(torch.randn(4, 4, device="cuda").double())
    with pytest.raises(L.FiError):
        ops.newton_schulz([torch.randn(4, 4, device="cuda"), torch.randn(4, 4, device="cuda").int()])
