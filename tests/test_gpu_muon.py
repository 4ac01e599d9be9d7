"""Matrices made orthogonal by products and the Muon step, against float64.

Errors, of the result's norm: a step rounds X, S and P (pieces of 22 bits, or 11 in bfloat16, and float32 sums): six
roundings at random, which the steps after it multiply by the polynomial's slope, at most 2 where singular values end
(smaller ones grow by as much as their errors).  sqrt(6 (1 + 4 + 16 + 64 + 256)) = 45 roundings of 2^-22 and, in
bfloat16, 2^-12: 1.1e-5 and 1.1e-2; and the result's own rounding, 2^-11 in float16 and 2^-8 in bfloat16.
"""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = {torch.float32: 1.1e-5, torch.float16: 1.1e-5 + 2.0 ** -11, torch.bfloat16: 1.1e-2 + 2.0 ** -8}
SHAPES = [(1, 1), (1, 9), (7, 3), (16, 27), (64, 64), (65, 130), (200, 64), (129, 128), (300, 257), (90, 1000), (1000, 40)]
COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _exact(x, steps=5, c=COEFFICIENTS, eps=1e-7):
    x = x.detach().double().cpu()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-1, -2)
    x = x / (x.square().sum((-1, -2), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        s = x @ x.transpose(-1, -2)
        x = c[0] * x + (c[1] * s + c[2] * (s @ s)) @ x
    return x.transpose(-1, -2) if tall else x


def _off(got, want):
    return float((got.detach().double().cpu() - want).norm() / want.norm().clamp(min=1e-300))


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(shape, dtype):
    from spherical_distortion import functional as F
    g = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(3, *shape, generator=g) * torch.tensor([1.0, 1e-3, 50.0])[:, None, None]).to(dtype).to(DEV)
    got = F.orthogonalize(x)
    assert got.shape == x.shape and got.dtype == dtype
    want = _exact(x)
    for i in range(3):
        assert _off(got[i], want[i]) <= TOL[dtype], i
        assert torch.equal(F.orthogonalize(x[i]), got[i])
    assert torch.equal(F.orthogonalize(x.transpose(-1, -2).contiguous().transpose(-1, -2)), got)


@pytest.mark.parametrize("shape", [(1100, 1300), (2048, 1025)])
def test_large_matrices(shape):
    """Tiles of 128, of which the last reach over the sides."""
    from spherical_distortion import functional as F
    g = torch.Generator().manual_seed(1)
    for dtype in TOL:
        x = torch.randn(*shape, generator=g).to(dtype).to(DEV)
        want = _exact(x.to(DEV))
        assert _off(F.orthogonalize(x), want) <= TOL[dtype]


def test_singular_values_and_other_settings():
    """Well conditioned matrices: singular values between 0.68 and 1.14 after five steps, and other coefficients and
    numbers of steps as given."""
    from spherical_distortion import functional as F
    g = torch.Generator().manual_seed(2)
    x = torch.randn(100, 300, generator=g).to(DEV)
    s = torch.linalg.svdvals(F.orthogonalize(x).double().cpu())
    assert 0.68 <= float(s.min()) and float(s.max()) <= 1.14
    for steps, c in ((1, COEFFICIENTS), (12, (1.875, -1.25, 0.375)), (3, (1.5, -0.5, 0.0))):
        assert _off(F.orthogonalize(x, steps, c), _exact(x, steps, c)) <= TOL[torch.float32]


def test_zeros_tiny_and_infinite_matrices():
    from spherical_distortion import functional as F
    x = torch.zeros(3, 20, 30, device=DEV)
    x[1] = torch.randn(20, 30, device=DEV) * 1e-25     # squares vanish in 32 bits; eps outweighs the norm
    x[2, 3, 4] = float("inf")
    got = F.orthogonalize(x)
    assert not bool(got[0].any()) and bool(got[2].isnan().any())
    assert _off(F.orthogonalize(x[1] * 1e20, eps=1e-30), _exact(x[1] * 1e20, eps=1e-30)) <= TOL[torch.float32]
    assert _off(F.orthogonalize(x[1], eps=2.0 ** -100), _exact(x[1], eps=2.0 ** -100)) <= TOL[torch.float32]
    assert F.orthogonalize(torch.zeros(0, 4, 5, device=DEV)).shape == (0, 4, 5)
    assert F.orthogonalize(torch.zeros(2, 0, 5, device=DEV)).shape == (2, 0, 5)


def test_more_matrices_than_a_launch_holds():
    from spherical_distortion import functional as F
    x = torch.randn(150, 10, 14, device=DEV)
    got, want = F.orthogonalize(x), _exact(x)
    for i in (0, 63, 64, 127, 128, 149):
        assert _off(got[i], want[i]) <= TOL[torch.float32]


def _lists(shapes, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    params, grads, momenta = ([(torch.randn(*s, generator=g) * scale).to(kind).to(DEV) for s in shapes]
                              for scale, kind in ((0.05, dtype), (1e-3, dtype), (1e-3, torch.float32)))
    return params, grads, momenta


@pytest.mark.parametrize("dtype", list(TOL))
@pytest.mark.parametrize("nesterov", [True, False])
def test_steps(dtype, nesterov):
    from spherical_distortion import functional as F
    shapes = [(16, 3, 9), (40, 16, 9), (65, 7), (7, 65), (128, 300), (5, 1)] + [(9, 9)] * 70
    params, grads, momenta = _lists(shapes, dtype, seed=3)
    before = copy.deepcopy((params, grads, momenta))
    F.muon_step(params, grads, momenta, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.2)
    for p, g, m, p0, g0, m0 in zip(params, grads, momenta, *before):
        assert torch.equal(g, g0)
        gd = g0.double().cpu()
        want_m = 0.9 * m0.double().cpu() + 0.1 * gd
        # three roundings of values of which the sum may be smaller
        assert float((m.double().cpu() - want_m).abs().max()) <= 4 * 2.0 ** -24 * 1e-2
        u = 0.9 * want_m + 0.1 * gd if nesterov else want_m
        flat = u.reshape(u.shape[0], -1)
        rate = 0.1 * math.sqrt(max(1.0, flat.shape[0] / flat.shape[1]))
        update = rate * _exact(flat).reshape(u.shape)
        want = p0.double().cpu() * (1 - 0.1 * 0.2) - update
        own = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
        bound = (TOL[dtype] * float(update.norm()) + own * float(want.norm()) + 1e-12)
        assert float((p.double().cpu() - want).norm()) <= bound


def test_steps_are_reproducible_and_counted():
    from spherical_distortion import functional as F
    a = _lists([(130, 70), (33, 200)], torch.float32, seed=4)
    b = copy.deepcopy(a)
    versions = [t._version for t in a[0] + a[2]]
    F.muon_step(*a)
    F.muon_step(*b)
    assert all(torch.equal(x, y) for x, y in zip(a[0] + a[2], b[0] + b[2]))
    assert all(t._version > v for t, v in zip(a[0] + a[2], versions))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optimizer(dtype):
    """A network's matrices by Muon and its vectors by AdamW; a checkpoint goes on bit for bit."""
    from spherical_distortion.optim import AdamW, Muon
    torch.manual_seed(0)

    def net():
        return torch.nn.Sequential(torch.nn.Linear(24, 50), torch.nn.GELU(), torch.nn.Linear(50, 6)).to(DEV).to(dtype)

    def optimizers(model):
        return (Muon([p for p in model.parameters() if p.dim() > 1], lr=0.01, weight_decay=0.1),
                AdamW([p for p in model.parameters() if p.dim() < 2]))

    def train(model, steps, opts, seed):
        g = torch.Generator().manual_seed(seed)
        for _ in range(steps):
            x = torch.randn(32, 24, generator=g).to(dtype).to(DEV)
            loss = (model(x) - x[:, :6]).float().square().mean()
            for o in opts:
                o.zero_grad()
            loss.backward()
            for o in opts:
                o.step()

    model = net()
    opts = optimizers(model)
    train(model, 3, opts, 1)
    assert all(opts[0].state[p]["momentum"].dtype == torch.float32 for p in opts[0].param_groups[0]["params"])
    other = copy.deepcopy(model)
    resumed = optimizers(other)
    for o, r in zip(opts, resumed):
        r.load_state_dict(copy.deepcopy(o.state_dict()))
    train(model, 2, opts, 2)
    train(other, 2, resumed, 2)
    assert all(torch.equal(a, b) for a, b in zip(model.parameters(), other.parameters()))


def test_refusals():
    from spherical_distortion import functional as F
    x = torch.randn(4, 5, device=DEV)
    for bad in (x[0], x.double(), x.int()):
        with pytest.raises(RuntimeError):
            F.orthogonalize(bad)
    for settings in (dict(steps=0), dict(steps=101), dict(coefficients=(1.0, 2.0)), dict(eps=0.0), dict(eps=float("nan")),
                     dict(coefficients=(1.0, float("nan"), 0.0)), dict(coefficients=(1.0, 1e3, 0.0))):
        with pytest.raises(RuntimeError):
            F.orthogonalize(x, **settings)
    m = torch.zeros_like(x)
    bad = [([x], [x], []), ([x], [x.half()], [m]), ([x], [x], [m.half()]), ([x[0]], [x[0]], [m[0]]), ([x], [x[:2]], [m]),
           ([x.t()], [x.t()], [m.t()]), ([], [x], [])]
    for lists in bad:
        with pytest.raises(RuntimeError):
            F.muon_step(*lists)
    for settings in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(steps=0)):
        before = x.clone()
        with pytest.raises(RuntimeError):
            F.muon_step([x], [x.clone()], [m], **settings)
        assert torch.equal(x, before) and not bool(m.any())
