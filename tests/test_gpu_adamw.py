"""AdamW over lists of tensors, moments in 32 bits and in 8, against float64 on the CPU.

Tolerances: each value is formed by about ten float32 roundings: 1e-6 of the value for moments, and for a
parameter 1e-6 of the larger of itself and the step; a first moment's two terms may cancel: 1e-6 of both.  A
parameter of 16 bits is rounded once, to half a unit in its last place: float16's smallest is 2^-24.  Codes: the float32 value before rounding is off by 1e-6
of itself, so a code differs from the nearest one of the float64 value only beside a tie: by one, where the
exact position is within 2e-4 of the tie (127 or 255 times a few float32 roundings of the root).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SETTINGS = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
SIZES = [(1,), (3, 5), (256,), (257,), (4, 64), (1000, 3), (0,), (4099,), (16384,), (70, 71)]


def _tensors(sizes, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    p = [torch.randn(*s, generator=g) for s in sizes]
    gr = [0.1 * torch.randn(*s, generator=g) * torch.exp(torch.randn(*s, generator=g)) for s in sizes]
    return [t.to(dtype).to(DEV) for t in p], [t.to(dtype).to(DEV) for t in gr]


def _exact(p, g, m, v, step, lr, betas, eps, weight_decay):
    p, g, m, v = (t.detach().double().cpu() for t in (p, g, m, v))
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    move = lr * (m / (1 - betas[0] ** step)) / (torch.sqrt(v / (1 - betas[1] ** step)) + eps)
    return p * (1 - lr * weight_decay) - move, m, v, move


def _near(got, want, allowed):
    assert bool(((got.detach().double().cpu() - want).abs() <= allowed).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("count", [1, 10, 200])
def test_steps_of_32_bits(dtype, count):
    from spherical_distortion import functional as F
    sizes = [SIZES[i % len(SIZES)] for i in range(count)]
    p, _ = _tensors(sizes, dtype, seed=count)
    m, v = [[torch.zeros_like(t, dtype=torch.float32) for t in p] for _ in range(2)]
    ulp = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    least = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    for step in (1, 2, 7):
        _, g = _tensors(sizes, dtype, seed=step)
        want = [_exact(*t, step, **SETTINGS) for t in zip(p, g, m, v)]
        terms = [0.9 * a.double().cpu().abs() + 0.1 * b.double().cpu().abs() for a, b in zip(m, g)]
        F.adamw_step(p, g, m, v, step=step, **SETTINGS)
        for got_p, got_m, got_v, (wp, wm, wv, move), size in zip(p, m, v, want, terms):
            _near(got_p, wp, 1e-6 * (wp.abs() + move.abs()) + ulp * wp.abs() + least)
            _near(got_m, wm, 1e-6 * size)
            _near(got_v, wv, 1e-6 * wv + 1e-30)


def _values(codes, scales, second):
    """What codes stand for, in float64."""
    c = codes.reshape(-1).double().cpu()
    s = scales.double().cpu().repeat_interleave(256)[:c.numel()]
    x = (c / 255) ** 4 * s if second else c * c.abs() / 127 ** 2 * s
    return x.reshape(codes.shape)


def _check_codes(codes, scales, want, second):
    flat = want.reshape(-1)
    n = flat.numel()
    padded = torch.zeros(-(-n // 256) * 256, dtype=torch.float64)
    padded[:n] = flat
    s = padded.view(-1, 256).abs().amax(1)
    _near(scales, s, 1e-6 * s)
    s = s.repeat_interleave(256)[:n]
    at = torch.where(s > 0, flat.abs() / s, 0.0)
    at = 255 * at ** 0.25 if second else 127 * at.sqrt()
    got = codes.reshape(-1).double().cpu()
    if not second:
        assert bool(((got == 0) | (got.sign() == flat.sign())).all())
    off = (got.abs() - at).abs()
    assert bool((off <= torch.where((at < 1) & second, 1.0, 0.5) + 2e-4).all())
    if second:
        assert bool((got[flat > 0] >= 1).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("count", [1, 10, 130])
def test_steps_of_8_bits(dtype, count):
    from spherical_distortion import functional as F
    sizes = [SIZES[i % len(SIZES)] for i in range(count)]
    p, _ = _tensors(sizes, dtype, seed=count)
    blocks = [(-(-t.numel() // 256),) for t in p]
    mc, vc = ([torch.zeros(t.shape, dtype=d, device=DEV) for t in p] for d in (torch.int8, torch.uint8))
    ms, vs = ([torch.zeros(b, device=DEV) for b in blocks] for _ in range(2))
    ulp = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    least = 2.0 ** -25 if dtype == torch.float16 else 1e-30
    for step in (1, 2, 7):
        _, g = _tensors(sizes, dtype, seed=step)
        m, v = ([_values(*t, second) for t in zip(c, s)] for c, s, second in ((mc, ms, False), (vc, vs, True)))
        want = [_exact(*t, step, **SETTINGS) for t in zip(p, g, m, v)]
        F.adamw_step_8bit(p, g, mc, ms, vc, vs, step=step, **SETTINGS)
        for i, (wp, wm, wv, move) in enumerate(want):
            # values of the codes: five roundings more
            _near(p[i], wp, 2e-6 * (wp.abs() + move.abs()) + ulp * wp.abs() + least)
            _check_codes(mc[i], ms[i], wm, False)
            _check_codes(vc[i], vs[i], wv, True)
    for c, s, second in ((mc, ms, False), (vc, vs, True)):
        for codes, scales in zip(c, s):
            exact = _values(codes, scales, second)
            _near(F.adamw_moment_values(codes, scales), exact, 1e-6 * exact.abs())
            rounded = F.adamw_moment_values(codes, scales, dtype=torch.bfloat16)
            assert rounded.dtype == torch.bfloat16
            _near(rounded, exact, 2.0 ** -8 * exact.abs())


def test_views_at_any_address():
    from spherical_distortion import functional as F
    flat = [torch.randn(3000, device=DEV).abs() for _ in range(4)]
    views = [[t[1:1001], t[1003:2800]] for t in flat]
    want = [[t.clone() for t in v] for v in views]
    F.adamw_step(*views, step=3, **SETTINGS)
    F.adamw_step(*want, step=3, **SETTINGS)
    for a, b in zip(views, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_small_zero_and_broken_blocks():
    """Blocks of zeros and of values whose squares vanish stay finite; a NaN stays in its block."""
    from spherical_distortion import functional as F
    p = [torch.ones(1024, device=DEV)]
    g = [torch.zeros(1024, device=DEV)]
    g[0][256:512] = 1e-25      # squares below the smallest normal number
    g[0][512 + 7] = math.nan
    g[0][768:] = 1e-3
    mc, vc = [torch.zeros(1024, dtype=torch.int8, device=DEV)], [torch.zeros(1024, dtype=torch.uint8, device=DEV)]
    ms, vs = [torch.zeros(4, device=DEV)], [torch.zeros(4, device=DEV)]
    F.adamw_step_8bit(p, g, mc, ms, vc, vs, step=1, lr=1e-3, weight_decay=0.0)
    assert bool(torch.isfinite(p[0][:512]).all()) and bool(torch.isfinite(p[0][768:]).all())
    assert torch.equal(p[0][:256], torch.ones(256, device=DEV))
    assert ms[0].isnan().tolist() == [False, False, True, False]
    assert float(vs[0][0]) == 0 and float(vs[0][1]) == 0
    assert int(p[0].isnan().sum()) == 1
    values = F.adamw_moment_values(mc[0], ms[0])
    assert bool(values[512:768].isnan().all()) and bool(torch.isfinite(values[768:]).all())


def test_refusals():
    from spherical_distortion import functional as F
    p, g = _tensors([(4, 5), (6,)], torch.float32, seed=1)
    m, v = [torch.zeros_like(t) for t in p], [torch.zeros_like(t) for t in p]
    F.adamw_step([], [], [], [], step=1)
    for bad in ((p, g[:1], m, v), (p, g, m[::-1], v), (p, [t.half() for t in g], m, v), (p, g, [t.half() for t in m], v),
                ([t.double() for t in p], g, m, v), (p, g, [t.cpu() for t in m], v), ([p[0].t(), p[1]], [g[0].t(), g[1]],
                                                                                    [m[0].t(), m[1]], v)):
        with pytest.raises(RuntimeError):
            F.adamw_step(*bad, step=1)
    for settings in (dict(step=0), dict(step=1, lr=-1.0), dict(step=1, betas=(1.0, 0.9)), dict(step=1, eps=-1.0)):
        with pytest.raises(RuntimeError):
            F.adamw_step(p, g, m, v, **settings)
    codes, scales = [torch.zeros(t.shape, dtype=torch.int8, device=DEV) for t in p], [torch.zeros(1, device=DEV)] * 2
    with pytest.raises(RuntimeError):
        F.adamw_step_8bit(p, g, codes, scales, codes, scales, step=1)   # the second moment's codes are uint8
    with pytest.raises(RuntimeError):
        F.adamw_moment_values(codes[0], torch.zeros(2, device=DEV))
    with pytest.raises(RuntimeError):
        F.adamw_moment_values(codes[0].int(), scales[0])
