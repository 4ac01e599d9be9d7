"""The layers above the operators on token sequences: the compiled and the Python implementation of each operator
against each other (bit for bit: every sum has one order), modules, optimizer, bucket maps, and the example that runs
them together."""
import copy
import math
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _both(name, *args):
    from _spherical_distortion_ext import _token_ops
    assert name in _token_ops.NATIVE_OPS
    a, b = getattr(_token_ops.ops, name)(*args), _token_ops.PYTHON_IMPL[name](*args)
    one = not isinstance(a, (tuple, list))
    for x, y in zip([a] if one else a, [b] if one else b):
        assert x.shape == y.shape and x.dtype == y.dtype and x.stride() == y.stride()
        assert torch.equal(x.view(torch.uint8) if x.element_size() == 1 else x,
                           y.view(torch.uint8) if y.element_size() == 1 else y)
    return a


def test_compiled_and_python_operators_agree():
    from _spherical_distortion_ext import _token_ops
    torch.manual_seed(0)
    q = torch.randn(2, 70, 4, 32, device=DEV).transpose(1, 2)
    k, v = (torch.randn(2, 2, 90, 32, device=DEV) for _ in range(2))
    table = torch.randn(4, 9, device=DEV)
    bmap = torch.randint(0, 10, (70, 90), device=DEV).to(torch.uint8)
    n = torch.tensor([90, 41], dtype=torch.int32, device=DEV)
    out, rest, lse = _both("bucket_attention_forward", q, k, v, table, bmap, n, True, 0.2)
    do = torch.randn_like(q)
    for needs in ((True, True, True), (False, True, False), (True, False, False), (False, False, True)):
        _both("bucket_attention_backward", do, q, k, v, table, bmap, n, out, rest, lse, True, 0.2, *needs)
    x, r, w = torch.randn(20, 100, device=DEV), torch.randn(20, 100, device=DEV), torch.rand(100, device=DEV)
    for residual in (r, None):
        y, s, inv = _both("add_rms_norm", x, residual, w, 1e-6)
        for fp8 in (False, True):
            codes, scales, _ = _both("add_rms_norm_quantized", x, residual, w, 1e-6, fp8)
            _both("dequantize_rows", codes, scales, torch.bfloat16)
    y, s, inv = _both("add_rms_norm", x, r, w, 1e-6)
    _both("add_rms_norm_backward", y, x, s, w, inv, True, True)
    _both("add_rms_norm_backward", y, None, s, w, inv, True, False)
    _both("add_rms_norm_backward", y, None, s, w, inv, False, True)
    p, g = [torch.randn(300, device=DEV), torch.randn(7, 5, device=DEV)], [torch.randn(300, device=DEV),
                                                                          torch.randn(7, 5, device=DEV)]
    m32, v32 = [torch.zeros_like(t) for t in p], [torch.zeros_like(t) for t in p]
    lists = [p, g, m32, v32]
    other = copy.deepcopy(lists)
    settings = (1e-3, 0.9, 0.99, 1e-8, 0.1, 3)
    _token_ops.ops.adamw_step(*lists, *settings)
    _token_ops.PYTHON_IMPL["adamw_step"](*other, *settings)
    assert all(torch.equal(a, b) for x, y in zip(lists, other) for a, b in zip(x, y))
    mc, vc = ([torch.zeros(t.shape, dtype=d, device=DEV) for t in p] for d in (torch.int8, torch.uint8))
    ms, vs = ([torch.zeros(-(-t.numel() // 256), device=DEV) for t in p] for _ in range(2))
    lists = [p, g, mc, ms, vc, vs]
    other = copy.deepcopy(lists)
    _token_ops.ops.adamw_step_8bit(*lists, *settings)
    _token_ops.PYTHON_IMPL["adamw_step_8bit"](*other, *settings)
    assert all(torch.equal(a, b) for x, y in zip(lists, other) for a, b in zip(x, y))
    _both("adamw_moment_values", mc[0], ms[0], torch.float32)
    _both("adamw_moment_values", vc[1], vs[1], torch.float16)


def test_compiled_and_python_gradients_agree():
    """The compiled autograd functions and the Python ones: the same bits, and gradients only where wanted."""
    from _spherical_distortion_ext import _token_ops
    from spherical_distortion import functional as F
    torch.manual_seed(4)
    q = torch.randn(2, 4, 40, 16, device=DEV)
    k, v = (torch.randn(2, 2, 50, 16, device=DEV) for _ in range(2))
    table = torch.randn(4, 6, device=DEV)
    bmap = torch.randint(0, 7, (40, 50), device=DEV).to(torch.uint8)
    do = torch.randn_like(q)
    for wanted in ((1, 1, 1, 1), (1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 1), (0, 0, 0, 1)):
        results = []
        for fn in (_token_ops.ops.bucket_attention, F.BucketAttentionFunction.apply):
            leaves = [t.detach().requires_grad_(bool(w)) for t, w in zip((q, k, v, table), wanted)]
            out = fn(*leaves, bmap, None, True, 0.3)
            out.backward(do)
            results.append([out.detach()] + [t.grad for t in leaves])
        for a, b, w in zip(*results, (1,) + wanted):
            assert (a is None and b is None) if not w else torch.equal(a, b)
    x, r, dy, ds = (torch.randn(30, 70, device=DEV) for _ in range(4))
    w = torch.rand(70, device=DEV)
    for use in ((dy, ds), (dy, None), (None, ds)):
        for residual in (r, None):
            results = []
            for fn in (_token_ops.ops.rms_norm_pair, F.AddRMSNormFunction.apply):
                leaves = [t.detach().requires_grad_() for t in ((x, w) if residual is None else (x, residual, w))]
                both = fn(leaves[0], None if residual is None else leaves[1], leaves[-1], 1e-6)
                both = list(both)[:1 if residual is None else 2]
                pairs = [(o, g) for o, g in zip(both, use) if g is not None]
                if not pairs:
                    continue
                grads = torch.autograd.grad([o for o, _ in pairs], leaves, [g for _, g in pairs], allow_unused=True)
                results.append([o.detach() for o in both] + [torch.zeros(()) if g is None else g for g in grads])
            if results:
                assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(*results))


def test_python_operators_refuse_what_the_compiled_ones_refuse():
    from _spherical_distortion_ext import _token_ops
    q = torch.randn(1, 2, 4, 16, device=DEV)
    table, bmap = torch.zeros(2, 3, device=DEV), torch.zeros(4, 4, dtype=torch.uint8, device=DEV)
    x, w = torch.randn(3, 8, device=DEV), torch.ones(8, device=DEV)
    bad = [("bucket_attention_forward", (q, q[:, :, :, :8], q, table, bmap, None, False, 1.0)),
           ("bucket_attention_forward", (q, q, q, table, bmap.int(), None, False, 1.0)),
           ("bucket_attention_forward", (q, q, q, table[:1], bmap, None, False, 1.0)),
           ("bucket_attention_forward", (q, q, q, table, bmap, None, False, 0.0)),
           ("add_rms_norm", (x, x[:2], w, 1e-6)), ("add_rms_norm", (x, None, w[:4], 1e-6)),
           ("add_rms_norm", (x.t(), None, w[:3], 1e-6)),
           ("dequantize_rows", (x, w, torch.float32)),
           ("adamw_step", ([x], [x.half()], [x], [x], 1e-3, 0.9, 0.9, 1e-8, 0.0, 1)),
           ("adamw_step", ([x], [x], [x], [x], 1e-3, 0.9, 0.9, 1e-8, 0.0, 0)),
           ("adamw_moment_values", (x, w, torch.float32))]
    for name, args in bad:
        for fn in (getattr(_token_ops.ops, name), _token_ops.PYTHON_IMPL[name]):
            with pytest.raises(RuntimeError):
                fn(*args)


def test_modules_train():
    from spherical_distortion import nn as snn
    torch.manual_seed(1)
    layer, norm = snn.BucketAttention(64, 4, 9, num_key_heads=2).to(DEV), snn.AddRMSNorm(64).to(DEV)
    x = torch.randn(2, 30, 64, device=DEV)
    bmap = torch.randint(0, 9, (30, 30), device=DEV).to(torch.uint8)
    y, s = norm(layer(x, bmap), x)
    (y.square().mean() + s.mean()).backward()
    for p in list(layer.parameters()) + list(norm.parameters()):
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()) and bool(p.grad.any())
    with torch.no_grad():
        whole = layer(x, bmap)
        kept = layer.keys_and_values(x)
        one = layer(x[:, 7:8], bmap[7:8], keys_and_values=kept)
        # float32 sums in another order: 1e-5 of values of order one
        assert float((one[:, 0] - whole[:, 7]).abs().max()) <= 1e-5
        codes, scales, total = norm.quantized(x, x)
        assert codes.dtype == torch.int8 and torch.equal(total, x + x)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_optimizer_states_and_checkpoints(bits, dtype):
    """Steps against the operator itself; a state saved and loaded continues bit for bit."""
    from spherical_distortion import functional as F
    from spherical_distortion.optim import AdamW
    torch.manual_seed(2)
    params = [torch.nn.Parameter(torch.randn(*s, device=DEV).to(dtype)) for s in ((70, 100), (33,), (5000,))]
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    make = lambda ps: AdamW([{"params": ps[:2]}, {"params": ps[2:], "lr": 1e-2}], lr=1e-3, moment_bits=bits)  # noqa: E731
    optimizer, other = make(params), make(copies)
    grads = [[torch.randn_like(p) for p in params] for _ in range(4)]
    for i in range(4):
        for p, g in zip(params, grads[i]):
            p.grad = g.clone()
        if i == 1:
            params[1].grad = None   # this parameter makes a step less
        optimizer.step()
        if i == 1:
            saved = copy.deepcopy(optimizer.state_dict())
            for c, p in zip(copies, params):
                c.data.copy_(p)
            other.load_state_dict(saved)
    for i in (2, 3):
        for c, g in zip(copies, grads[i]):
            c.grad = g.clone()
        other.step()
    for p, c in zip(params, copies):
        assert torch.equal(p, c)
        assert optimizer.state[p].keys() == other.state[c].keys()
        for name, value in optimizer.state[p].items():
            assert type(value) is type(other.state[c][name])
            if torch.is_tensor(value):
                assert value.dtype == other.state[c][name].dtype and torch.equal(value, other.state[c][name])
    assert [optimizer.state[p]["step"] for p in params] == [4, 3, 4]
    eight = ["avg_codes" in optimizer.state[p] for p in params]
    assert eight == [bits == 8, False, bits == 8]
    if not eight[0]:
        m, v = torch.zeros(70, 100, device=DEV), torch.zeros(70, 100, device=DEV)
        torch.manual_seed(2)
        p = torch.randn(70, 100, device=DEV).to(dtype)
        for i in range(4):
            F.adamw_step([p], [grads[i][0]], [m], [v], step=i + 1, lr=1e-3)
        assert torch.equal(p, params[0])


def test_optimizer_refusals():
    from spherical_distortion.optim import AdamW
    p = [torch.nn.Parameter(torch.zeros(3, device=DEV))]
    for bad in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(moment_bits=4), dict(eps=-1.0), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            AdamW(p, **bad)


def test_bucket_maps():
    from spherical_distortion import util
    torch.manual_seed(3)
    lonlat = torch.stack([torch.rand(60) * 2 * math.pi - math.pi, torch.asin(2 * torch.rand(60) - 1)], -1).to(DEV)
    got = util.great_circle_bucket_map(lonlat, num_buckets=20).cpu()
    assert got.shape == (60, 60) and got.dtype == torch.uint8 and not bool(got.diagonal().any())
    d = lonlat.double().cpu()
    cos = (d[:, None, 1].sin() * d[None, :, 1].sin()
           + d[:, None, 1].cos() * d[None, :, 1].cos() * (d[:, None, 0] - d[None, :, 0]).cos())
    angle = cos.clamp(-1, 1).acos()
    at = 20 * (angle / math.pi).sqrt()
    assert bool(((got.double() <= at + 1e-5) & (got.double() > at - 1 - 1e-5)).all())
    near = util.great_circle_bucket_map(lonlat, lonlat[:7], num_buckets=20, reach=1.0).cpu()
    assert near.shape == (60, 7)
    clear = (angle[:, :7] - 1).abs() > 1e-6
    assert torch.equal((near == 255)[clear], (angle[:, :7] > 1)[clear])
    line = util.sequence_bucket_map(3, 50, 10, farthest=40).cpu()
    assert line.shape == (3, 50) and int(line[2, 49]) == 0 and int(line[0, 47]) == 0 and int(line[2, 45]) == 4
    assert int(line.max()) == 9 and bool((line[2].flip(0).diff().int() >= 0).all())
    for n in (0, 256):
        with pytest.raises(ValueError):
            util.sequence_bucket_map(2, 4, n)


def test_the_example_learns_and_serves():
    """The loss falls to less than half; a token asked alone gives the grid's answer within the 8-bit norm's step
    (1 / 127 of the largest of 128 values, at random) and bfloat16: 0.05 of outputs of order one."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import panorama_tokens
    losses, off = panorama_tokens.main(steps=30)
    assert sum(losses[-3:]) / 3 < 0.5 * losses[0]
    assert off <= 0.05
