"""The gated recurrence and its gradients, against float64, token by token.

u: half a step of the type (2^-24, 2^-8, 2^-11); M: the largest input or state.  A step's own operations are off by less
than 8 * 2^-24 of what it adds, which adds up to 8 * 2^-24 M as the weights of a state add up to one; the state's rounding
(2^-24 M a step) stays for as many tokens as the channel remembers, at most n = min(tokens, 1 / (1 - f)), and so do those
of the products of spans: 2^-24 M (16 + 3 n), and u |h| for the result's rounding.  Gradients alike, with the size of the
accumulated gradient; they are compared with the formula on h as the forward wrote it, which is what the backward reads.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32 = 2.0 ** -24


def _inputs(B, L, D, dtype, seed, state=True, ragged=False):
    g = torch.Generator().manual_seed(seed)
    both = torch.randn(B, L, 2, D, generator=g)
    both[:, :, 1] += 5 * torch.rand(D, generator=g)
    both = both.to(dtype).to(DEV)
    first = torch.randn(B, D, generator=g).to(DEV) if state else None
    lengths = None
    if ragged:
        lengths = torch.randint(0, L + 1, (B,), generator=g, dtype=torch.int32)
        lengths[0] = L
        if B > 1:
            lengths[1] = 0
        lengths = lengths.to(DEV)
    dy, dl = torch.randn(B, L, D, generator=g).to(dtype).to(DEV), torch.randn(B, D, generator=g).to(DEV)
    return both[:, :, 0], both[:, :, 1], first, lengths, dy, dl


def _exact(x, gate, state, lengths, reverse, written=None, dy=None, dl=None):
    """On the CPU in 64 bits: h, last; and with gradients those of x, gate, state and the largest accumulated one."""
    x, gate = x.detach().double().cpu(), gate.detach().double().cpu()
    B, L, D = x.shape
    f = torch.sigmoid(gate)
    h = torch.zeros(B, D, dtype=torch.float64) if state is None else state.detach().double().cpu()
    first = h
    n = torch.full((B,), L) if lengths is None else lengths.cpu().long()
    order = list(range(L - 1, -1, -1) if reverse else range(L))
    out = torch.zeros_like(x)
    for t in order:
        on = (t < n)[:, None]
        new = f[:, t] * h + (1 - f[:, t]) * x[:, t]
        h = torch.where(on, new, h)
        out[:, t] = torch.where(on, new, 0.0)
    if dy is None:
        return out, h
    written = written.double().cpu()
    e = torch.zeros(B, D, dtype=torch.float64) if dl is None else dl.double().cpu()
    dy = torch.zeros_like(x) if dy is False else dy.double().cpu()
    dx, dg, largest = torch.zeros_like(x), torch.zeros_like(x), e.abs().max()
    for t in reversed(order):
        on = (t < n)[:, None]
        before = t + 1 if reverse else t - 1
        inside = ((torch.full((B,), before) < n) & (0 <= before < L))[:, None]
        prev = torch.where(inside, written[:, min(max(before, 0), L - 1)], first)
        total = e + dy[:, t]
        largest = torch.maximum(largest, total.abs().max())
        dx[:, t] = torch.where(on, total * (1 - f[:, t]), 0.0)
        dg[:, t] = torch.where(on, total * (prev - x[:, t]) * f[:, t] * (1 - f[:, t]), 0.0)
        e = torch.where(on, f[:, t] * total, e)
    return out, h, dx, dg, e, largest


def _check(x, gate, state, lengths, reverse, dy, dl):
    from spherical_distortion import functional as F
    u, L = U[x.dtype], x.shape[1]
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, gate, state)]
    out, last = F.gated_scan(*leaves, lengths=lengths, reverse=reverse)
    assert out.is_contiguous() and last.dtype == torch.float32
    given = [t for t in leaves if t is not None]
    grads = torch.autograd.grad([out, last], given, [dy, dl])
    want = _exact(x, gate, state, lengths, reverse, out.detach(), dy, dl)
    n = min(L, float(1 + gate.float().max().exp())) if x.numel() else 0
    largest = max(float(x.abs().max()), float(state.abs().max()) if state is not None else 0.0) if x.numel() else 0
    def close(got, exact, own, slack):
        got = got.detach().double().cpu()
        assert got.shape == exact.shape
        assert bool(((got - exact).abs() <= own * exact.abs() + slack).all()), float((got - exact).abs().max())
    close(out, want[0], u, F32 * largest * (16 + 3 * n))
    close(last, want[1], F32, F32 * largest * (16 + 3 * n))
    slack = F32 * float(want[5]) * (16 + 3 * n)
    close(grads[0], want[2], u, slack)
    close(grads[1], want[3], u, slack * 2 * largest)
    if state is not None:
        close(grads[2], want[4], F32, slack)
    return out.detach(), last.detach(), grads


# one tile, parts of tiles, several tiles in segments, widths of no vector, of one lane, of many blocks
SIZES = [(1, 1, 1), (2, 3, 8), (3, 129, 5), (2, 128, 64), (1, 1000, 16), (2, 515, 17), (4, 300, 72), (1, 2050, 130),
         (2, 640, 200), (300, 5, 33), (1, 4096, 64)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,L,D", SIZES)
def test_scan_and_gradients(B, L, D, dtype):
    for reverse in (False, True):
        x, gate, state, lengths, dy, dl = _inputs(B, L, D, dtype, seed=B + L + D, state=not reverse, ragged=reverse)
        first = _check(x, gate, state, lengths, reverse, dy, dl)
        again = _check(x, gate, state, lengths, reverse, dy, dl)
        assert all(torch.equal(a, b) for a, b in zip(first[:2] + tuple(first[2]), again[:2] + tuple(again[2])))


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("B,L,D", [(5, 700, 40), (1, 900, 8), (3, 130, 256)])
def test_ragged_sequences_with_states(B, L, D, reverse):
    """Lengths of zero, of all and between; what lies behind them is not read."""
    from spherical_distortion import functional as F
    x, gate, state, lengths, dy, dl = _inputs(B, L, D, torch.float32, seed=L, ragged=True)
    first = _check(x, gate, state, lengths, reverse, dy, dl)
    behind = (torch.arange(L, device=DEV)[None] >= lengths[:, None])[:, :, None].expand(B, L, D)
    dirty = [torch.where(behind, float("nan"), t) for t in (x, gate, dy)]
    out, last = F.gated_scan(dirty[0].requires_grad_(), dirty[1].requires_grad_(), state, lengths, reverse)
    grads = torch.autograd.grad([out, last], dirty[:2], [dirty[2], dl])
    assert torch.equal(out, first[0]) and torch.equal(last, first[1])
    assert all(torch.equal(a, b) for a, b in zip(grads, first[2]))
    assert not bool(out[behind].any())
    # lengths outside the sequence count as none and all
    wild = lengths.clone()
    wild[0], wild[-1] = L + 7, -3
    tame = wild.clamp(0, L)
    assert all(torch.equal(a, b) for a, b in zip(F.gated_scan(x, gate, state, wild, reverse),
                                                 F.gated_scan(x, gate, state, tame, reverse)))


def test_parts_follow_each_other():
    """A sequence in two calls, the state handed on, and token by token: within the bound of two roundings of h."""
    from spherical_distortion import functional as F
    x, gate, state, _, _, _ = _inputs(3, 400, 48, torch.float32, seed=1)
    whole, last = F.gated_scan(x, gate, state)
    a, middle = F.gated_scan(x[:, :150], gate[:, :150], state)
    b, end = F.gated_scan(x[:, 150:], gate[:, 150:], middle)
    bound = F32 * float(x.abs().max()) * 2 * (16 + 3 * 400)
    assert float((torch.cat([a, b], 1) - whole).abs().max()) <= bound and float((end - last).abs().max()) <= bound
    held = state.clone()
    for t in range(400):
        assert float((F.gated_scan_step(x[:, t], gate[:, t], held) - whole[:, t]).abs().max()) <= bound
    assert float((held - last).abs().max()) <= bound


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,D", [(1, 1), (64, 1024), (7, 33), (200, 24)])
def test_steps(B, D, dtype):
    from spherical_distortion import functional as F
    x, gate, state, _, _, _ = _inputs(B, 1, D, dtype, seed=B * D)
    pool = torch.full((B, D + 3), 9.0, device=DEV)
    held = pool[:, :D]
    held.copy_(state)
    version = held._version
    out = F.gated_scan_step(x[:, 0], gate[:, 0], held)
    want = _exact(x, gate, state, None, False)[1]
    assert float((held.double().cpu() - want).abs().max()) <= 16 * F32 * 5
    assert torch.equal(out, held.to(dtype)) and bool((pool[:, D:] == 9).all()) and held._version > version
    # strided and transposed inputs
    wide = x[:, 0].t().contiguous().t()
    again = state.clone()
    assert torch.equal(F.gated_scan_step(wide, gate[:, 0], again), out) and torch.equal(again, held)


def test_layouts():
    """Views of one projection, tokens outside the batch, expanded gates, dense tensors at odd addresses."""
    from spherical_distortion import functional as F
    g = torch.Generator().manual_seed(2)
    for dtype in (torch.float32, torch.bfloat16):
        base = torch.randn(2, 130, 64, generator=g).to(dtype).to(DEV)
        gate = torch.randn(130, 64, generator=g).to(dtype).to(DEV)
        want = F.gated_scan(base, gate.expand(2, 130, 64).contiguous())
        outside = base.transpose(0, 1).contiguous().transpose(0, 1)
        wide = torch.cat([base, base], -1)[..., :64]
        odd = torch.empty(base.numel() + 1, dtype=dtype, device=DEV)[1:].view_as(base).copy_(base)
        turned = base.transpose(1, 2).contiguous().transpose(1, 2)
        for x in (base, outside, wide, odd, turned):
            got = F.gated_scan(x, gate.expand(2, 130, 64))
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        leaf = gate.clone().requires_grad_()
        out, _ = F.gated_scan(base, leaf.expand(2, 130, 64))
        out.sum().backward()        # a gradient without strides
        parts = [gate.clone().requires_grad_() for _ in range(2)]
        for b, part in enumerate(parts):
            F.gated_scan(base[b:b + 1], part[None])[0].sum().backward()
        # the sum of two gradients, rounded once more
        both = parts[0].grad.double() + parts[1].grad.double()
        assert float((leaf.grad.double() - both).abs().max()) <= 2 * U[dtype] * float(both.abs().max()) + 1e-6


def test_parts_of_the_gradients():
    from spherical_distortion import functional as F
    x, gate, state, lengths, dy, dl = _inputs(2, 300, 40, torch.float32, seed=11, ragged=False)
    whole = _check(x, gate, state, None, False, dy, dl)[2]
    for wanted in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        leaves = [t.detach().requires_grad_(bool(n)) for t, n in zip((x, gate, state), wanted)]
        out = F.gated_scan(*leaves)
        grads = torch.autograd.grad(out, [t for t in leaves if t.requires_grad], [dy, dl])
        assert all(torch.equal(a, b) for a, b in zip(grads, [v for v, n in zip(whole, wanted) if n]))
    leaves = [t.detach().requires_grad_() for t in (x, gate, state)]
    out, last = F.gated_scan(*leaves)
    only_out = torch.autograd.grad(out, leaves, dy, retain_graph=True)
    only_last = torch.autograd.grad(last, leaves, dl)
    zero = torch.zeros_like(dl)
    assert all(torch.equal(a, b) for a, b in zip(only_out, _check(x, gate, state, None, False, dy, zero)[2]))
    assert all(torch.equal(a, b) for a, b in zip(only_last, _check(x, gate, state, None, False, torch.zeros_like(dy), dl)[2]))


def test_gradients_against_differences():
    """A weighted sum of about 60 terms of order one: quotients with a step of 2^-5 are off by about 60 * 2^-23 / 2^-5 =
    2.3e-4 from rounding and 2^-10 / 6 of a third derivative of order one: 2e-3."""
    from spherical_distortion import functional as F
    x, gate, state, _, dy, dl = _inputs(2, 9, 3, torch.float32, seed=5)
    leaves = [t.detach().requires_grad_() for t in (x, gate, state)]
    grads = torch.autograd.grad(F.gated_scan(*leaves), leaves, [dy, dl])
    for i, grad in enumerate(grads):
        for at in ((0, 1, 2), (1, 8, 0), (1, 0, 1)) if i < 2 else ((0, 1), (1, 2)):
            sides = []
            for sign in (1, -1):
                moved = [t.detach().clone() for t in leaves]
                moved[i][at] += sign * 2.0 ** -5
                out, last = F.gated_scan(*moved)
                sides.append(float((out.double() * dy).sum() + (last.double() * dl).sum()))
            want = (sides[0] - sides[1]) * 16
            assert abs(float(grad[at]) - want) <= 2e-3 * max(1.0, abs(want))


def test_gates_of_any_size():
    """Gates far beyond where a sigmoid is one or zero, infinite ones among them: the state is kept or replaced."""
    from spherical_distortion import functional as F
    sizes = torch.tensor([-float("inf"), -1e4, -200.0, -90.0, -20.0, 0.0, 20.0, 90.0, 200.0, 1e4, float("inf")], device=DEV)
    gate = sizes[None, None].expand(1, 3, 11).contiguous().requires_grad_()
    x = torch.full((1, 3, 11), 2.0, device=DEV).requires_grad_()
    out, last = F.gated_scan(x, gate, torch.full((1, 11), 5.0, device=DEV))
    f = torch.sigmoid(sizes.double())
    want = torch.stack([5 * f ** t + 2 * (1 - f ** t) for t in (1, 2, 3)])
    assert float((out[0].double() - want).abs().max()) <= 64 * F32 * 5
    grads = torch.autograd.grad(out.sum(), [x, gate])
    assert all(bool(t.isfinite().all()) for t in grads)
    bad = torch.zeros(1, 4, 2, device=DEV)
    bad[0, 1, 0] = float("nan")
    out, _ = F.gated_scan(torch.ones(1, 4, 2, device=DEV), bad)
    assert out.isnan()[0].tolist() == [[False, False], [True, False], [True, False], [True, False]]


def test_nothing_to_scan():
    from spherical_distortion import functional as F
    state = torch.randn(2, 8, device=DEV).requires_grad_()
    x = torch.zeros(2, 0, 8, device=DEV, dtype=torch.bfloat16).requires_grad_()
    out, last = F.gated_scan(x, x, state)
    assert out.shape == (2, 0, 8) and torch.equal(last, state)
    dl = torch.randn(2, 8, device=DEV)
    assert torch.equal(torch.autograd.grad(last, state, dl)[0], dl)
    out, last = F.gated_scan(x, x)
    assert not bool(last.any())
    for shape in ((0, 5, 8), (2, 5, 0)):
        out, last = F.gated_scan(torch.zeros(shape, device=DEV), torch.zeros(shape, device=DEV))
        assert out.shape == shape and last.shape == (shape[0], shape[2])


def test_refusals():
    from spherical_distortion import functional as F
    x, s = torch.randn(2, 5, 8, device=DEV), torch.zeros(2, 8, device=DEV)
    n = torch.ones(2, dtype=torch.int32, device=DEV)
    bad = [(x, x[:1]), (x, x.half()), (x[0], x[0]), (x.double(), x.double()), (x, x.cpu()), (x, x, s[:1]), (x, x, s.half()),
           (x, x, s.cpu()), (x, x, s, n.long()), (x, x, s, n[:1]), (x, x, s, n.cpu())]
    for args in bad:
        with pytest.raises(RuntimeError):
            F.gated_scan(*args)
    t = x[:, 0]
    steps = [(t, t, s[:1]), (t, t, s.half()), (t, t.half(), s), (x, x, s), (t, t, torch.zeros(8, 2, device=DEV).t()),
             (t, t, torch.zeros(1, 8, device=DEV).expand(2, 8)), (t, t, s.cpu())]
    for args in steps:
        with pytest.raises(RuntimeError):
            F.gated_scan_step(*args)
    with pytest.raises(RuntimeError, match="no gradients"):
        F.gated_scan_step(t.clone().requires_grad_(), t, s)
    leaf = x.clone().requires_grad_()
    first, = torch.autograd.grad(F.gated_scan(leaf, x)[0].square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        first.sum().backward()
