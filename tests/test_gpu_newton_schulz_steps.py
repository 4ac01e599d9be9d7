"""Newton-Schulz in up to 100 steps on matrices of up to 16 rows or columns, of full rank and of less.

x q(x^2) = 3.4445 x - 4.775 x^3 + 2.0315 x^5 is at most 1.2024 for x in [0, 1.2024] (at 0.5545) and at least 0.6818 for x
from 0.5545 on (at 1.050), and larger than x below 0.5545: after a dozen steps the singular values of a matrix lie between
the two whatever is rounded on the way, and those that were zero, where roundings grow as any value does, between 0 and
1.2024.  1.5 x - 0.5 x^3 takes all of (0, 1] to one.

Slack: a step rounds X (norm up to 4.81), S (5.8, which the polynomial multiplies by up to 10.7) and P: less than 100
roundings of 2^-22, of 2^-12 in bfloat16; and the result's own rounding.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NS = (3.4445, -4.7750, 2.0315)
NEWTON = (1.5, -0.5, 0.0)
TYPES = [torch.float32, torch.float16, torch.bfloat16]
SHAPES = [(16, 27), (2, 3), (16, 16), (100, 10), (1, 40), (16, 1000), (5000, 12)]


def _slack(dtype):
    return 100 * 2.0 ** (-12 if dtype == torch.bfloat16 else -22) + 4.81 * torch.finfo(dtype).eps / 2


def _matrix(kind, shape, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    if kind == "full":
        return torch.randn(*shape, generator=g).to(dtype).to(DEV)
    if kind == "rank one":   # rounded: in 16 bits the rest is small, not zero
        return (torch.randn(shape[0], 1, generator=g) @ torch.randn(1, shape[1], generator=g)).to(dtype).to(DEV)
    one = torch.randn(1, max(shape), generator=g).expand(min(shape), -1)   # the same row or column again and again
    return (one if shape[0] <= shape[1] else one.t()).to(dtype).to(DEV).contiguous()


def _values(x):
    return torch.linalg.svdvals(x.double().cpu())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("steps", [7, 12, 14, 20, 30, 100])
@pytest.mark.parametrize("kind", ["full", "rank one", "equal"])
def test_singular_values_stay_in_their_interval(kind, steps, dtype):
    from spherical_distortion import functional as F
    for shape in SHAPES:
        got = F.orthogonalize(_matrix(kind, shape, dtype), steps)
        assert bool(got.isfinite().all()), shape
        s = _values(got)
        assert float(s.max()) <= 1.2024 + _slack(dtype), shape
        if kind == "full" and steps >= 12 or steps == 100:
            assert float(s.max()) >= 0.6818 - _slack(dtype), shape
        if kind == "full" and steps >= 12:
            assert float(s.min()) >= 0.6818 - _slack(dtype), shape


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("steps", [50, 100])
def test_steps_that_converge(steps, dtype):
    """The polar factor, which a matrix moves by at most sqrt(2) / (its smallest singular value) of a change of its own; the
    smallest singular value grows by 1.5 a step, so the steps' roundings count three times: 5 in all."""
    from spherical_distortion import functional as F
    for shape in ((16, 27), (2, 3), (100, 10), (16, 1000), (5000, 12)):
        x = _matrix("full", shape, dtype)
        u, s, vt = torch.linalg.svd(x.double().cpu(), full_matrices=False)
        got = F.orthogonalize(x, steps, NEWTON)
        off = float((got.double().cpu() - u @ vt).norm())
        assert off <= 5 * _slack(dtype) * float(s.norm() / s.min()), shape
    for kind in ("rank one", "equal"):
        for shape in SHAPES:
            got = F.orthogonalize(_matrix(kind, shape, dtype), steps, NEWTON)
            assert float(_values(got).max()) <= 1 + _slack(dtype), (kind, shape)


@pytest.mark.parametrize("steps", [1, 2, 5, 6])
@pytest.mark.parametrize("shape", [(16, 27), (2, 3), (10, 100), (16, 1000), (16, 16), (900, 7)])
def test_few_steps_round_once(shape, steps):
    """64 bits up to six steps, and of them 2^-25 lost at most: the result's rounding."""
    from spherical_distortion import functional as F
    for kind in ("full", "rank one", "equal"):
        x = _matrix(kind, shape, torch.float32)
        y = x.double().cpu()
        y = y.t() if shape[0] > shape[1] else y
        y = y / (y.norm() + 1e-7)
        for _ in range(steps):
            s = y @ y.t()
            y = NS[0] * y + (NS[1] * s + NS[2] * (s @ s)) @ y
        y = y.t() if shape[0] > shape[1] else y
        off = float((F.orthogonalize(x, steps).double().cpu() - y).norm())
        assert off <= (2.0 ** -24 + 2.0 ** -25) * float(y.norm()), kind


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("steps", [5, 30])
def test_matrices_of_few_rows_beside_others(steps, dtype):
    """A Muon step over both: the bits of each alone."""
    from spherical_distortion import functional as F
    shapes = [(16, 27), (16, 1000), (40, 50), (1, 7), (130, 200), (3000, 9)]
    lists = [[_matrix("full", s, kind) for s in shapes] for kind in (dtype, dtype, torch.float32)]
    alone = [[t.clone() for t in ts] for ts in lists]
    F.muon_step(*lists, lr=0.1, steps=steps)
    for i in range(len(shapes)):
        F.muon_step(*(ts[i:i + 1] for ts in alone), lr=0.1, steps=steps)
    for ts, us in zip(lists, alone):
        assert all(torch.equal(t, u) and bool(t.isfinite().all()) for t, u in zip(ts, us))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(12, 40), (60, 60), (200, 90)])
def test_singular_values_go_where_the_polynomial_takes_them(shape, dtype):
    """Spread over 0.001 to 0.7 of the norm, so that some end near its maximum of 1.2024.  Of the slack each value takes what the
    slope of five steps makes of it (the product of their slopes, at most 3.4445^5 for the smallest): bounded over the matrix
    as the largest slope times the rounding of the matrix and a step, 2^-22 or 2^-12, and the slack itself."""
    from spherical_distortion import functional as F
    g = torch.Generator().manual_seed(sum(shape))
    k = min(shape)
    u, v = (torch.linalg.qr(torch.randn(n, k, generator=g, dtype=torch.float64))[0] for n in shape)
    x = ((u * torch.logspace(0, -2.5, k, dtype=torch.float64)) @ v.t()).to(dtype).to(DEV)
    s = _values(x)
    s = s / s.norm()
    slope = torch.ones_like(s)
    for _ in range(5):
        slope = slope * (NS[0] + 3 * NS[1] * s ** 2 + 5 * NS[2] * s ** 4).abs()
        s = NS[0] * s + NS[1] * s ** 3 + NS[2] * s ** 5
    got = _values(F.orthogonalize(x))
    assert float(s.max()) > 1.19
    unit = 2.0 ** (-12 if dtype == torch.bfloat16 else -22)
    off = (got - s.sort(descending=True).values).abs().max()
    assert float(off) <= _slack(dtype) + float(slope.max()) * unit
    assert float(got.max()) <= 1.2024 + _slack(dtype)


def test_gradients_are_refused_or_not_wanted():
    from spherical_distortion import functional as F
    x = torch.randn(20, 30, device=DEV)
    leaf = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradients"):
        F.orthogonalize(leaf)
    want = F.orthogonalize(x)
    assert not want.requires_grad and torch.equal(F.orthogonalize(leaf.detach()), want)
    with torch.no_grad():
        assert torch.equal(F.orthogonalize(leaf), want)


def test_coefficients_that_are_taken_stay_in_range():
    """Whatever the coefficients, what is not refused ends finite, with singular values that pass 3.8 by roundings alone (2^-10 a
    step, and the slack): of one singular value, which takes the extremes, and of many."""
    from spherical_distortion import functional as F
    g = torch.Generator().manual_seed(9)
    taken = 0
    for i in range(120):
        c = ((torch.rand(3, generator=g) * 2 - 1) * torch.tensor([4.0, 6.0, 4.0 * (i % 3 > 0)])).tolist()
        c = [(3.0, -1.0, 0.0), NS, NEWTON, (2.6, -1.0, 0.0)][i] if i < 4 else c
        steps = 1 + i % 12
        for dtype in TYPES:
            for kind, shape in (("rank one", (8, 50)), ("equal", (40, 30)), ("rank one", (100, 130)), ("full", (70, 70))):
                try:
                    got = F.orthogonalize(_matrix(kind, shape, dtype), steps, c)
                except RuntimeError as e:
                    assert "grow too far" in str(e)
                    continue
                taken += 1
                assert bool(got.isfinite().all()), (c, steps, kind, shape, dtype)
                assert float(_values(got)[0]) <= 3.8 * (1 + 2.0 ** -10) + _slack(dtype), (c, steps, kind, shape, dtype)
    assert taken >= 100   # of 1440 the most are refused


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(16, 1000), (50, 60), (300, 200)])
def test_norms_beyond_float32(shape, dtype):
    """Values of up to 2^127, whose norm float32 does not hold: the bits of the same matrix times 2^-100, as powers of two
    change nothing but eps' share (2^-122 beside 1)."""
    from spherical_distortion import functional as F
    x = _matrix("full", shape, dtype).float()
    x = (x / x.abs().max()).to(dtype)
    big = (x.double() * 2.0 ** 127).to(dtype)
    assert bool(big.isfinite().all()) and float(big.double().norm()) > torch.finfo(torch.float32).max
    assert torch.equal(F.orthogonalize(big), F.orthogonalize((big.double() * 2.0 ** -100).to(dtype)))
    p, m = torch.zeros_like(x), big.float().clone()
    F.muon_step([p], [big], [m], lr=1.0, momentum=0.5)
    assert torch.equal(m, big.float()) and bool(p.isfinite().all()) and float(p.double().norm()) > 0.5
