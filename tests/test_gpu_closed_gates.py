"""Gates that close: the state is replaced, and what is left of it is small but known to its last digits.

Everything is positive, so nothing cancels but h - x in the gates' gradient, and errors are relative to each value: a token
costs less than 16 roundings of 2^-24 (16-bit gates 48: their power's argument is rounded, 43 * 2^-24 at a gate of 30), an
earlier error goes on in the share that the state before has, and gates between -30 and 3 forget within 64 tokens.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
F32 = 2.0 ** -24


def _rounding(dtype):
    return F32 * (16 if dtype == torch.float32 else 48)


def _positive(g, lo, hi, *shape):
    """Spread over their logarithm."""
    return torch.exp(torch.rand(*shape, generator=g) * (torch.tensor(hi / lo).log()) + torch.tensor(lo).log())


def _inputs(B, L, D, dtype, seed, lowest=-30.0):
    g = torch.Generator().manual_seed(seed)
    x = _positive(g, 1e-3, 1e4, B, L, D).to(dtype).to(DEV)
    gate = (lowest + (3 - lowest) * torch.rand(B, L, D, generator=g)).to(dtype).to(DEV)
    state = _positive(g, 1.0, 1e5, B, D).to(DEV)
    dy = _positive(g, 1e-2, 1.0, B, L, D).to(dtype).to(DEV)
    dl = _positive(g, 1e-2, 1.0, B, D).to(DEV)
    return x, gate, state, dy, dl


def _exact(x, gate, state, written, dy, dl):
    x, gate, h, written, dy, e = (t.detach().double().cpu() for t in (x, gate, state, written, dy, dl))
    f, u = torch.sigmoid(gate), torch.sigmoid(-gate)
    out, dx, dg, size = (torch.zeros_like(x) for _ in range(4))
    first = h
    for t in range(x.shape[1]):
        h = out[:, t] = f[:, t] * h + u[:, t] * x[:, t]
    for t in reversed(range(x.shape[1])):
        before = written[:, t - 1] if t else first
        total = e + dy[:, t]
        dx[:, t] = total * u[:, t]
        dg[:, t] = total * f[:, t] * u[:, t] * (before - x[:, t])
        size[:, t] = total * f[:, t] * u[:, t] * (before + x[:, t])
        e = f[:, t] * total
    return out, h, dx, dg, e, size


def _close(got, want, own, slack, size=None):
    """float16 has no finite values beyond 65504: half a step further, 65520, and what is off by less than `slack` of it, may
    be infinite, and everything beyond has to be, as have gradients that read such a state (`want` is infinite itself)."""
    got = got.detach().double().cpu()
    size = want.abs() if size is None else size
    smallest = 2.0 ** -25 if own == 2.0 ** -11 else 1e-36    # of float16 below 2^-14
    off = (got - want).abs() - own * want.abs() - slack * size - smallest
    fine = (off <= 0) | (got == want)
    if own == 2.0 ** -11:
        fine |= (want.abs() >= 65520 * (1 - slack)) & (got == want.sign() * float("inf"))
    assert bool(fine.all()), off[~fine]


# threads alone, a tile of one workgroup, tiles that hand on, widths of no vector, many sequences
SIZES = [(3, 1, 8), (5, 7, 33), (2, 100, 64), (1, 3000, 64), (2, 1500, 201), (140, 300, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,L,D", SIZES)
@pytest.mark.parametrize("reverse", [False, True])
def test_values_and_gradients(B, L, D, dtype, reverse):
    from spherical_distortion import functional as F
    x, gate, state, dy, dl = _inputs(B, L, D, dtype, seed=B + L + D)
    leaves = [t.detach().requires_grad_() for t in (x, gate, state)]
    out, last = F.gated_scan(*leaves, reverse=reverse)
    grads = torch.autograd.grad([out, last], leaves, [dy, dl])
    turned = (lambda t: t.flip(1)) if reverse else (lambda t: t)
    want = _exact(turned(x), turned(gate), state, turned(out), turned(dy), dl)
    own, slack = torch.finfo(dtype).eps / 2, _rounding(dtype) * min(L, 64)
    _close(turned(out), want[0], own, slack)
    _close(last, want[1], F32, slack)
    _close(turned(grads[0]), want[2], own, slack)
    _close(turned(grads[1]), want[3], own, slack, want[5])
    _close(grads[2], want[4], F32, slack)


@pytest.mark.parametrize("dtype", TYPES)
def test_single_tokens(dtype):
    from spherical_distortion import functional as F
    x, gate, state, _, _ = _inputs(300, 1, 72, dtype, seed=3)
    state *= 100
    held = state.clone()
    out = F.gated_scan_step(x[:, 0], gate[:, 0], held)
    f, u = torch.sigmoid(gate[:, 0].double()), torch.sigmoid(-gate[:, 0].double())
    want = (f * state.double() + u * x[:, 0].double()).cpu()
    _close(held, want, 0, _rounding(dtype))
    assert torch.equal(out, held.to(dtype))


def test_resets():
    """Of a state of 1000 a gate of -20 leaves 2e-6 beside 1e-3; of one of 1e4 a gate of -30 leaves 1e-9 beside 1e-4; a gate of
    minus infinity leaves nothing, and the gradients of gates of -8 to -30 have all their digits."""
    from spherical_distortion import functional as F
    for h, x, g in ((1000.0, 1e-3, -20.0), (1e4, 1e-4, -30.0), (1e30, 1.0, -float("inf")), (1e4, 0.0, -60.0)):
        for tokens in (1, 40):
            one = torch.full((1, tokens, 4), x, device=DEV)
            gates = torch.full((1, tokens, 4), 0.0, device=DEV)
            gates[:, 0] = g
            out, _ = F.gated_scan(one, gates, torch.full((1, 4), h, device=DEV))
            f, u = torch.sigmoid(torch.tensor(g).double()), torch.sigmoid(-torch.tensor(g).double())
            want = float(f * h + u * x)
            assert bool(((out[0, 0].double() - want).abs() <= 16 * F32 * want).all()), (h, x, g)
    gate = torch.arange(-30.0, -7.5, 0.5, device=DEV).view(1, 1, -1).requires_grad_()
    x, state = torch.full_like(gate, 2.0), torch.full((1, gate.shape[2]), 5.0, device=DEV).requires_grad_()
    out, _ = F.gated_scan(x.detach(), gate, state)
    dg, ds = torch.autograd.grad(out.sum(), [gate, state])
    f, u = torch.sigmoid(gate[0, 0].double()), torch.sigmoid(-gate[0, 0].double())
    assert bool(((dg[0, 0] - 3 * f * u).abs() <= 16 * F32 * 3 * f * u).all())
    assert bool(((ds[0] - f).abs() <= 16 * F32 * f).all())
