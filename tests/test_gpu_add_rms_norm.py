"""Residual addition with root-mean-square norm, its gradients and its 8-bit rows, against float64 on the CPU.

Tolerances, of the largest value of an output: float32: the sum of squares of n values is off by less than
sqrt(n) 2^-24 / 2 of itself in the kernels' order, the reciprocal root by half of that, and three roundings
follow: 1e-6.  bfloat16 and float16: one rounding of the result, and in the backward one of the saved sum, both
2^-9 and 2^-12 of the value: 8e-3 and 1e-3.  dw sums rows products each off by 2^-9 or 2^-12 at random and is
rounded once: the same bound.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = {torch.float32: 1e-6, torch.bfloat16: 8e-3, torch.float16: 1e-3}
SHAPES = [(1, 1), (3, 7), (5, 64), (2, 3, 100), (300, 129), (17, 1024), (9, 1025), (70, 1000), (40, 2048), (3, 4096),
          (2, 5000), (33, 4097), (2, 16384), (3, 16383), (1500, 48)]


def _inputs(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x, r, dy, ds = (torch.randn(*shape, generator=g).to(dtype).to(DEV) for _ in range(4))
    w = (1 + 0.3 * torch.randn(shape[-1], generator=g)).to(DEV)
    return x, r, w, dy, ds


def _exact(x, r, w, eps=1e-6, dy=None, ds=None):
    x, w = x.detach().double().cpu(), w.detach().double().cpu()
    h = x if r is None else x + r.detach().double().cpu()
    inv = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    y = h * inv * w
    if dy is None:
        return y, h
    dy = dy.double().cpu()
    g = dy * w
    dh = inv * (g - h * inv ** 2 * (g * h).mean(-1, keepdim=True)) + (0 if ds is None else ds.double().cpu())
    return y, h, dh, (dy * h * inv).reshape(-1, h.shape[-1]).sum(0)


def _close(got, want, tol):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    assert float((got - want).abs().max()) <= tol * max(float(want.abs().max()), 1e-30)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_and_gradients(shape, dtype):
    from spherical_distortion import functional as F
    x, r, w, dy, ds = _inputs(shape, dtype, seed=sum(shape))
    for weight in (w, w.to(dtype)):
        leaves = [t.detach().requires_grad_() for t in (x, r, weight)]
        y, h = F.add_rms_norm(*leaves)
        grads = torch.autograd.grad([y, h], leaves, [dy, ds])
        ref = _exact(x, r, weight, dy=dy, ds=ds)
        for got, want in zip((y, h, grads[0], grads[1], grads[2]), (ref[0], ref[1], ref[2], ref[2], ref[3])):
            _close(got, want, TOL[dtype])
        assert grads[2].dtype == weight.dtype
        again = torch.autograd.grad(F.add_rms_norm(*leaves), leaves, [dy, ds])
        assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_without_residual_and_parts_of_the_gradients(dtype):
    from spherical_distortion import functional as F
    x, r, w, dy, ds = _inputs((50, 200), dtype, seed=4)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    y, h = F.add_rms_norm(leaves[0], None, leaves[1])
    assert torch.equal(h, x)
    ref = _exact(x, None, w, dy=dy)
    for got, want in zip((y, *torch.autograd.grad(y, leaves, dy)), (ref[0], ref[2], ref[3])):
        _close(got, want, TOL[dtype])
    y, h = F.add_rms_norm(x, r, w)
    got = torch.autograd.grad(h, [x, w], ds, allow_unused=True)
    assert torch.equal(got[0], ds) and (got[1] is None or not bool(got[1].any()))
    r.requires_grad_()
    y, h = F.add_rms_norm(x.detach(), r, w.detach())
    only, = torch.autograd.grad(y, [r], dy)
    _close(only, _exact(x, r, w, dy=dy)[2], TOL[dtype])


def test_gradients_against_differences():
    """A weighted sum of about 30 terms of order one: quotients with a step of 2^-5 are off by about 30 * 2^-23 /
    2^-5 = 1e-4 from rounding and 2^-10 / 6 of a third derivative of order one: 2e-3."""
    from spherical_distortion import functional as F
    x, r, w, dy, ds = _inputs((3, 10), torch.float32, seed=9)
    leaves = [t.requires_grad_() for t in (x, r, w)]
    grads = torch.autograd.grad(F.add_rms_norm(*leaves), leaves, [dy, ds])
    for i, grad in enumerate(grads):
        for at in ((0, 1), (2, 9)) if i < 2 else ((0,), (7,)):
            sides = []
            for sign in (1, -1):
                moved = [t.detach().clone() for t in leaves]
                moved[i][at] += sign * 2.0 ** -5
                y, h = F.add_rms_norm(*moved)
                sides.append(float((y.double() * dy).sum() + (h.double() * ds).sum()))
            want = (sides[0] - sides[1]) * 16
            assert abs(float(grad[at]) - want) <= 2e-3 * max(1.0, abs(want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("codes", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("shape", [(1, 1), (4, 33), (16, 4096), (7, 1003), (100, 264), (2, 16384)])
def test_rows_in_8_bits(shape, codes, dtype):
    """A code is the nearest: off by half a step (of the scale for int8; of 2^-3 of the value, or of the
    smallest step 2^-9, for float8), and where the float32 value lies beside a tie by 1e-6 more."""
    from spherical_distortion import functional as F
    x, r, w, _, _ = _inputs(shape, dtype, seed=sum(shape))
    got, scales, h = F.add_rms_norm_quantized(x, r, w, dtype=codes)
    y, sums = _exact(x, r, w)
    _close(h, sums, TOL[dtype])
    most = 127 if codes == torch.int8 else 448
    assert got.dtype == codes and scales.shape == x.shape[:-1]
    _close(scales, y.abs().amax(-1) / most, 1e-6)
    scale = scales.double().cpu()[..., None]
    value = got.float().double().cpu()
    want = y / scale
    half = torch.full_like(want, 0.5) if codes == torch.int8 else (want.abs() * 2.0 ** -4).clamp(min=2.0 ** -10)
    assert bool(((value - want).abs() <= half + 2e-6 * most).all())
    for out in (torch.float32, torch.bfloat16):
        back = F.dequantize_rows(got, scales, dtype=out)
        assert back.dtype == out and torch.equal(back, (got.float() * scales[..., None]).to(out))


def test_rows_of_zeros_and_of_nan():
    from spherical_distortion import functional as F
    x = torch.randn(4, 40, device=DEV)
    x[1] = 0
    x[2, 3] = math.nan
    x[3] *= 1e-30
    w = torch.ones(40, device=DEV)
    for codes in (torch.int8, torch.float8_e4m3fn):
        got, scales, h = F.add_rms_norm_quantized(x, None, w, dtype=codes)
        assert h is x or torch.equal(h[0], x[0])
        assert float(scales[1]) == 0 and not bool(got.float()[1].any())
        assert math.isnan(float(scales[2]))
        back = F.dequantize_rows(got, scales)
        assert bool(back[2].isnan().all()) and bool(torch.isfinite(back[[0, 1, 3]]).all())
    y, _ = F.add_rms_norm(x, None, w)
    assert bool(y[2].isnan().all()) and bool(torch.isfinite(y[[0, 1, 3]]).all()) and not bool(y[1].any())


def test_unaligned_rows_and_no_rows():
    from spherical_distortion import functional as F
    flat = torch.randn(1 + 8 * 64, device=DEV)
    x = flat[1:].view(8, 64)
    w = torch.rand(64, device=DEV)
    _close(F.add_rms_norm(x, None, w)[0], _exact(x, None, w)[0], 1e-6)
    none = torch.empty(0, 64, device=DEV, requires_grad=True)
    wr = w.clone().requires_grad_()
    y, h = F.add_rms_norm(none, none, wr)
    assert y.shape == (0, 64)
    grads = torch.autograd.grad(y.sum(), [none, wr])
    assert grads[0].shape == (0, 64) and not bool(grads[1].any())


def test_refusals():
    from spherical_distortion import functional as F
    x, w = torch.randn(4, 16, device=DEV), torch.ones(16, device=DEV)
    for bad in ((x.double(), None, w.double()), (x, x[:2], w), (x, x.half(), w), (x, None, w[:8]), (x, None, w.half()),
                (x.t(), None, w[:4]), (x, None, w.cpu()), (torch.empty(2, 16392, device=DEV), None,
                                                          torch.ones(16392, device=DEV))):
        with pytest.raises(RuntimeError):
            F.add_rms_norm(*bad)
        with pytest.raises(RuntimeError):
            F.add_rms_norm_quantized(*bad)
    with pytest.raises(RuntimeError):
        F.add_rms_norm_quantized(x, None, w, dtype=torch.uint8)
    codes, scales, _ = F.add_rms_norm_quantized(x, None, w)
    for bad in ((codes.float(), scales), (codes, scales[:2]), (codes, scales.half()), (codes, scales.cpu())):
        with pytest.raises(RuntimeError):
            F.dequantize_rows(*bad)
    with pytest.raises(RuntimeError):
        F.dequantize_rows(codes, scales, dtype=torch.float64)
