"""Residual addition with layer norm and its gradients, against float64.

u: half a step of the type (2^-24, 2^-8, 2^-11).  A result is rounded once, u of its size; before that the float32 sums
of a row (at most 16 values a thread in order, ten levels of a tree) and the operations on them are off by less than
32 * 2^-24 of the sizes of their terms (float32 sums, which the backward reads as they were written, by 2^-24 of theirs).
dw and db: sums over rows, of which a thread adds rows / 256 in order, 128 levels above them.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SHAPES = [(1, 1), (3, 2), (3, 7), (5, 64), (70, 65), (2, 3, 100), (301, 129), (17, 1024), (9, 1025), (40, 2048), (3, 4096),
          (2, 5000), (33, 8193), (2, 16384), (3, 16383), (5000, 48), (2049, 96)]
F32 = 2.0 ** -24


def _inputs(shape, dtype, seed, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    x, r, dy, ds = ((torch.randn(*shape, generator=g) + o).to(dtype).to(DEV) for o in (offset, 0, 0, 0))
    w, b = ((o + 0.3 * torch.randn(shape[-1], generator=g)).to(DEV) for o in (1, 0))
    return x, r, w, b, dy, ds


def _d(t):
    return None if t is None else t.detach().double()


def _forward(x, r, w, b, eps):
    """Values in 64 bits, and the size of what each is formed from."""
    h = _d(x) if r is None else _d(x) + _d(r)
    mean = h.mean(-1, keepdim=True)
    inv = 1 / torch.sqrt((h - mean).square().mean(-1, keepdim=True) + eps)
    y = (h - mean) * inv * _d(w) + (0 if b is None else _d(b))
    size = (h.abs() + mean.abs() + h.abs().mean(-1, keepdim=True)) * inv * _d(w).abs() + y.abs()
    return y, h, mean, inv, size


def _within(got, want, size, u, factor=32):
    """|got - want| <= u |want| + factor 2^-24 of the largest size in the row (size of the last axis, or a vector)."""
    assert got.shape == want.shape
    bound = u * want.abs() + factor * F32 * size
    assert bool(((_d(got) - want).abs() <= bound).all()), float(((_d(got) - want).abs() / bound.clamp(min=1e-300)).max())


def _check(x, r, w, b, dy, ds, eps=1e-5, leaves=None):
    from spherical_distortion import functional as F
    u = U[x.dtype]
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, r, w, b)]
    y, total = F.add_layer_norm(*leaves, eps=eps)
    want, h, mean, inv, size = _forward(x, r, w, b, eps)
    _within(y, want, size.amax(-1, keepdim=True), u)
    _within(total, h, h.abs(), 0 if r is None else u, factor=1)
    given = [t for t in leaves if t is not None]
    if r is None:
        grads = torch.autograd.grad(y, given, dy)
    else:
        grads = torch.autograd.grad([y, total], given, [dy, ds])
    z, g = (h - mean) * inv, _d(dy)
    q = g * _d(w)
    flat, along = q.mean(-1, keepdim=True), (q * z).mean(-1, keepdim=True)
    dh = inv * (q - flat - z * along) + (0 if r is None else _d(ds))
    rough = z.abs() + (h.abs() + mean.abs()) * inv         # what z is formed from
    sizes = inv * (q.abs() + q.abs().mean(-1, keepdim=True) + rough * (q * rough).abs().mean(-1, keepdim=True)
                   + rough * along.abs()) + (0 if r is None else _d(ds).abs())
    _within(grads[0], dh, sizes.amax(-1, keepdim=True), u)
    if r is not None:
        assert torch.equal(grads[0], grads[1])
    flatten = lambda t: t.reshape(-1, t.shape[-1])
    terms, uw = 160 + flatten(g).shape[0] / 256, U[w.dtype]
    at = 1 if r is None else 2
    _within(grads[at], flatten(g * z).sum(0), flatten(g.abs() * rough).sum(0), uw, factor=terms)
    if b is not None:
        _within(grads[at + 1], flatten(g).sum(0), flatten(g.abs()).sum(0), uw, factor=terms)
    return y, total, grads


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_and_gradients(shape, dtype):
    x, r, w, b, dy, ds = _inputs(shape, dtype, seed=sum(shape))
    first = _check(x, r, w, b, dy, ds)
    _check(x, None, w.to(dtype), b.to(dtype), dy, ds)
    _check(x, r, w, None, dy, ds)
    again = _check(x, r, w, b, dy, ds)
    assert all(torch.equal(a, c) for a, c in zip(first[2], again[2]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_rows_far_from_zero(dtype):
    """A mean of 100 deviations: squares of the distances from it, not a difference of sums of squares."""
    _check(*_inputs((50, 300), dtype, seed=3, offset=100.0))


def test_rows_without_spread():
    from spherical_distortion import functional as F
    x = torch.full((3, 40), 7.25, device=DEV)
    w, b = torch.ones(40, device=DEV), torch.arange(40.0, device=DEV)
    y, _ = F.add_layer_norm(x, None, w, b)
    assert torch.equal(y, b.expand(3, 40))


@pytest.mark.parametrize("width", [96, 97])
def test_memory_at_odd_addresses(width):
    g = torch.Generator().manual_seed(5)
    for dtype in (torch.float32, torch.bfloat16):
        def odd():
            return torch.randn(20 * width + 1, generator=g).to(dtype).to(DEV)[1:].view(20, width)
        x, r, dy, ds = odd(), odd(), odd(), odd()
        w, b = (torch.randn(width + 1, generator=g).to(DEV)[1:] for _ in range(2))
        _check(x, r, w, b, dy, ds)


def test_parts_of_the_gradients():
    from spherical_distortion import functional as F
    x, r, w, b, dy, ds = _inputs((50, 200), torch.float32, seed=4)
    whole = _check(x, r, w, b, dy, ds)[2]
    for wanted in ((1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (0, 1, 0, 1)):
        leaves = [t.detach().requires_grad_(bool(n)) for t, n in zip((x, r, w, b), wanted)]
        y, h = F.add_layer_norm(*leaves)
        needed = [t for t in leaves if t.requires_grad]
        uses_h = wanted[0] or wanted[1]
        grads = torch.autograd.grad([y, h] if uses_h else y, needed, [dy, ds] if uses_h else dy)
        assert all(torch.equal(a, c) for a, c in zip(grads, [v for v, n in zip(whole, wanted) if n]))
    leaves = [t.detach().requires_grad_() for t in (x, r, w, b)]
    y, h = F.add_layer_norm(*leaves)
    only = torch.autograd.grad(h, leaves, ds, allow_unused=True)
    assert torch.equal(only[0], ds) and torch.equal(only[1], ds)
    assert all(t is None or not bool(t.any()) for t in only[2:])
    with torch.no_grad():
        again, total = F.add_layer_norm(x, r, w, b)
    assert torch.equal(again, y) and torch.equal(total, h)


def test_gradients_against_differences():
    """A weighted sum of about 30 terms of order one: quotients with a step of 2^-5 are off by about 30 * 2^-23 / 2^-5 =
    1e-4 from rounding and 2^-10 / 6 of a third derivative of order ten: 4e-3."""
    from spherical_distortion import functional as F
    x, r, w, b, dy, ds = _inputs((3, 10), torch.float32, seed=9)
    leaves = [t.requires_grad_() for t in (x, r, w, b)]
    grads = torch.autograd.grad(F.add_layer_norm(*leaves), leaves, [dy, ds])
    for i, grad in enumerate(grads):
        for at in ((0, 1), (2, 9)) if i < 2 else ((0,), (7,)):
            sides = []
            for sign in (1, -1):
                moved = [t.detach().clone() for t in leaves]
                moved[i][at] += sign * 2.0 ** -5
                y, h = F.add_layer_norm(*moved)
                sides.append(float((y.double() * dy).sum() + (h.double() * ds).sum()))
            want = (sides[0] - sides[1]) * 16
            assert abs(float(grad[at]) - want) <= 4e-3 * max(1.0, abs(want))


def test_no_rows_and_values_that_are_not_finite():
    from spherical_distortion import functional as F
    w = torch.ones(8, device=DEV, requires_grad=True)
    x = torch.zeros(0, 8, device=DEV, requires_grad=True)
    y, h = F.add_layer_norm(x, None, w, w)
    grads = torch.autograd.grad(y, [x, w], torch.zeros_like(y))
    assert y.shape == (0, 8) and grads[0].shape == (0, 8) and not bool(grads[1].any())
    rows = torch.randn(4, 300, device=DEV)
    clean = F.add_layer_norm(rows, None, torch.ones(300, device=DEV))[0]
    rows[1, 7], rows[2, 299] = float("nan"), float("inf")
    y = F.add_layer_norm(rows, None, torch.ones(300, device=DEV))[0]
    assert bool(y[1:3].isnan().all()) and torch.equal(y[[0, 3]], clean[[0, 3]])


def test_refusals():
    from spherical_distortion import functional as F
    x, w = torch.randn(4, 16, device=DEV), torch.ones(16, device=DEV)
    bad = [(x, x[:2], w, None), (x, x.half(), w, None), (x, None, w[:8], None), (x, None, w.half(), None),
           (x, None, w, w[:8]), (x, None, w, w.half()), (x, None, w, w.cpu()), (x.t(), None, w[:4], None),
           (x.double(), None, w, None), (x, None, w.expand(2, 16), None), (torch.randn(2, 16385, device=DEV), None,
                                                                           torch.ones(16385, device=DEV), None)]
    for args in bad:
        with pytest.raises(RuntimeError):
            F.add_layer_norm(*args)
    with pytest.raises(RuntimeError):
        F.add_layer_norm(x, None, w, eps=-1.0)
    leaf = x.clone().requires_grad_()
    y, _ = F.add_layer_norm(leaf, None, w)
    first, = torch.autograd.grad(y.square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        first.sum().backward()
