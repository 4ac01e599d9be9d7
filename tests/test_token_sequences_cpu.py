"""Layer norm, the gated scan, Newton-Schulz and Muon without a GPU: argument checks of the C entries (all of them before
anything touches the device), workspace sizes, and what modules and the optimizer refuse."""
import ctypes

import pytest
import torch

ONE = ctypes.c_void_p(256)   # aligned, never dereferenced
NS = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope="module")
def lib():
    from _spherical_distortion_ext import _capi
    handle = _capi.load()
    handle.sdk_last_error.restype = ctypes.c_char_p
    return handle


def test_layer_norm_refuses(lib):
    def run(x=ONE, weight=ONE, out=ONE, rows=4, width=64, eps=1e-5, dtype=0, weight_dtype=0):
        return lib.sdk_add_layer_norm(x, None, weight, None, out, None, None, None, rows, width, eps, dtype, weight_dtype, None)
    for bad in (dict(x=None), dict(weight=None), dict(out=None), dict(rows=-1), dict(rows=1 << 31), dict(width=0),
                dict(width=16385), dict(eps=-1.0), dict(eps=float("nan")), dict(dtype=1), dict(weight_dtype=2),
                dict(dtype=2, weight_dtype=3)):
        assert run(**bad) == -1, bad
    assert run(rows=0, x=None) == 0

    def back(grad=ONE, x=ONE, weight=ONE, mean=ONE, gx=ONE, gw=ONE, gb=None, ws=ONE, bytes_=1 << 30, rows=4, width=64):
        return lib.sdk_add_layer_norm_backward(grad, None, x, None, weight, mean, ONE, gx, gw, gb, ws, bytes_, rows, width, 0, 0,
                                               None)
    for bad in (dict(grad=None), dict(x=None), dict(weight=None), dict(mean=None), dict(gx=None, gw=None), dict(rows=-2),
                dict(width=20000)):
        assert back(**bad) == -1, bad
    need = lib.sdk_add_layer_norm_backward_workspace_bytes(4, 64)
    # 4 threads a row: 64 rows share a workgroup; dw and db
    assert need == 2 * 64 * 4
    assert lib.sdk_add_layer_norm_backward_workspace_bytes(1 << 20, 64) == 1024 * 2 * 64 * 4
    assert lib.sdk_add_layer_norm_backward_workspace_bytes(4, 20000) == 0
    assert back(bytes_=need - 1) == -3 and back(ws=None) == -3


def _scan(**changes):
    from _spherical_distortion_ext import _capi
    a = _capi.GatedScan()
    for name in ("x", "gate", "output", "last", "grad_x"):
        setattr(a, name, 256)
    a.batch, a.tokens, a.width = 2, 4096, 1024
    for name in ("x_strides", "gate_strides", "grad_output_strides"):
        setattr(a, name, (ctypes.c_int64 * 2)(4096 * 1024, 1024))
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes", [dict(dtype=1), dict(dtype=9), dict(batch=-1), dict(tokens=-1), dict(width=-1),
                                     dict(width=(1 << 20) + 1), dict(tokens=1 << 31), dict(batch=1 << 31), dict(x=None),
                                     dict(gate=None), dict(output=None)])
def test_scan_refuses(lib, changes):
    a = _scan(**changes)
    for entry in (lib.sdk_gated_scan_forward, lib.sdk_gated_scan_backward):
        assert entry(ctypes.byref(a), ONE, 1 << 40, None) == -1
    assert lib.sdk_gated_scan_forward(ctypes.byref(_scan(last=None)), ONE, 1 << 40, None) == -1
    assert lib.sdk_gated_scan_backward(ctypes.byref(_scan(grad_x=None)), ONE, 1 << 40, None) == -1
    assert lib.sdk_gated_scan_forward(None, ONE, 0, None) == -1
    assert lib.sdk_gated_scan_workspace_bytes(None, 0) == 0


def test_scan_workspaces(lib):
    size = lib.sdk_gated_scan_workspace_bytes
    need = size(ctypes.byref(_scan()), 0)
    # 32 channels of float32 a block: 64 groups; at least a word each of A and H for every tile of 512 tokens and channel
    assert need >= 2 * 8 * 2 * 1024 * 8
    for bad in ((None, need), (ONE, need - 1), (ctypes.c_void_p(260), need)):
        assert lib.sdk_gated_scan_forward(ctypes.byref(_scan()), *bad, None) == -3
    assert lib.sdk_gated_scan_backward(ctypes.byref(_scan()), ONE, size(ctypes.byref(_scan()), 1) - 1, None) == -3
    # sequences of one tile, and enough of them to fill the GPU, hand nothing on
    assert size(ctypes.byref(_scan(tokens=100)), 1) == 0 and size(ctypes.byref(_scan(batch=64)), 1) == 0
    # nor do more tiles than a launch has workgroups
    assert size(ctypes.byref(_scan(batch=1000, tokens=1 << 27, width=1)), 0) == 0
    for nothing in (dict(batch=0, x=None), dict(width=0, x=None)):
        for entry in (lib.sdk_gated_scan_forward, lib.sdk_gated_scan_backward):
            assert entry(ctypes.byref(_scan(**nothing)), None, 0, None) == 0
    assert lib.sdk_gated_scan_backward(ctypes.byref(_scan(tokens=0)), None, 0, None) == 0   # no gradient of a state wanted


def test_scan_step_refuses(lib):
    def run(x=ONE, gate=ONE, state=ONE, out=ONE, stride=8, batch=2, width=8, dtype=0):
        return lib.sdk_gated_scan_step(x, 8, gate, 8, state, stride, out, batch, width, dtype, None)
    for bad in (dict(x=None), dict(gate=None), dict(state=None), dict(out=None), dict(stride=7), dict(stride=0), dict(batch=-1),
                dict(batch=1 << 31), dict(width=-1), dict(width=(1 << 20) + 1), dict(dtype=1)):
        assert run(**bad) == -1, bad
    assert run(batch=0, x=None) == 0 and run(width=0, x=None) == 0


def _three(c):
    return (ctypes.c_double * 3)(*c)


def test_orthogonalize_refuses(lib):
    def run(x=ONE, out=ONE, rows=100, columns=100, count=1, steps=5, c=_three(NS), eps=1e-7, ws=ONE, bytes_=1 << 40, dtype=0):
        return lib.sdk_orthogonalize(x, out, rows, columns, count, steps, c, eps, ws, bytes_, dtype, None)
    for bad in (dict(x=None), dict(out=None), dict(rows=-1), dict(columns=(1 << 17) + 1), dict(rows=1 << 17, columns=(1 << 14) + 1),
                dict(count=-1), dict(steps=0), dict(steps=101), dict(c=None), dict(eps=0.0), dict(eps=2.0), dict(dtype=1),
                dict(eps=float("nan")), dict(c=_three((1.0, float("inf"), 0.0)))):
        assert run(**bad) == -1, bad
    need = lib.sdk_orthogonalize_workspace_bytes(100, 100, 1, 0)
    # X twice, S and P, 4 bytes a value of sides padded to 128, and the norm's parts
    assert need == 4 * 128 * 128 * 4 + 128
    assert run(bytes_=need - 1) == -3 and run(ws=None) == -3 and run(ws=ctypes.c_void_p(320)) == -3
    assert lib.sdk_orthogonalize_workspace_bytes(100, 100, 100, 0) == 64 * need   # as many as a launch takes
    assert lib.sdk_orthogonalize_workspace_bytes(60, 60, 9, 0) == 0               # small ones need none
    assert lib.sdk_orthogonalize_workspace_bytes(-1, 60, 9, 0) == 0
    for nothing in (dict(count=0, x=None), dict(rows=0, x=None), dict(columns=0, x=None)):
        assert run(**nothing) == 0


def test_coefficients_that_would_leave_float16_are_refused():
    """Those with which entries stay below 16 pass, whatever the steps: against the polynomial at many points."""
    from _spherical_distortion_ext import _token_ops

    def allowed(steps, c):
        try:
            _token_ops.check_newton_schulz(steps, c, 1e-7)
        except RuntimeError as e:
            assert "grow too far" in str(e)
            return False
        return True
    for steps, c in ((100, NS), (12, (1.875, -1.25, 0.375)), (30, (1.5, -0.5, 0.0)), (1, (3.0, 0.0, 0.0)), (4, (0.0, 0.0, 0.0))):
        assert allowed(steps, c)
    for steps, c in ((1, (16.0, 0.0, 0.0)), (2, (3.0, 0.0, 0.0)), (1, (1.0, -70.0, 70.0)), (3, (2.0, 1.0, 0.0))):   # q(1/2) = -16.5
        assert not allowed(steps, c)
    g = torch.Generator().manual_seed(0)
    seen = set()
    for i in range(300):
        c = ((torch.rand(3, generator=g, dtype=torch.float64) * 2 - 1) * torch.tensor([5.0, 8.0, 5.0 * (i % 4 > 0)])).tolist()
        most, good = 1.0, True
        for _ in range(3):
            x = torch.linspace(0, most, 20001, dtype=torch.float64)
            q = (c[0] + c[1] * x ** 2 + c[2] * x ** 4).abs()
            good = good and float(q.max()) <= 15 and float((x * q).max()) <= 3.8
            most = float((x * q).max())
        assert allowed(3, c) == good, c
        seen.add(good)
    assert seen == {True, False}


def test_muon_step_refuses(lib):
    def lists(*addresses):
        return (ctypes.c_void_p * len(addresses))(*addresses)

    def sizes(*n):
        return (ctypes.c_int64 * len(n))(*n)

    def run(p=lists(256, 512), g=lists(1024, 2048), m=lists(4096, 8192), rows=sizes(100, 3), columns=sizes(100, 3), count=2, lr=0.1,
            momentum=0.9, wd=0.0, steps=5, c=_three(NS), eps=1e-7, ws=None, bytes_=0, dtype=0):
        return lib.sdk_muon_step(p, g, m, rows, columns, count, lr, momentum, 1, wd, steps, c, eps, ws, bytes_, dtype, None)
    none = (ctypes.c_void_p * 2)()
    for bad in (dict(p=None), dict(g=None), dict(m=None), dict(rows=None), dict(columns=None), dict(p=none), dict(g=none),
                dict(m=none), dict(rows=sizes(-1, 3)), dict(columns=sizes(100, 1 << 18)), dict(count=-1), dict(lr=-0.1),
                dict(lr=float("nan")), dict(momentum=1.0), dict(wd=-1.0), dict(steps=0), dict(c=_three((20.0, 0.0, 0.0))),
                dict(eps=0.0), dict(dtype=1),
                # the same memory twice
                dict(p=lists(256, 256)), dict(m=lists(4096, 4096)), dict(m=lists(4096, 256)), dict(g=lists(1024, 256)),
                dict(g=lists(8192, 2048))):
        assert run(**bad) == -1, bad
    assert "twice" in (run(p=lists(256, 256)), lib.sdk_last_error().decode())[1]
    assert run() == -3   # the matrix of 100 x 100 needs a workspace
    assert lib.sdk_muon_step_workspace_bytes(sizes(100, 3), sizes(100, 3), 2, 0) == 4 * 128 * 128 * 4 + 128
    assert lib.sdk_muon_step_workspace_bytes(sizes(100, -3), sizes(100, 3), 2, 0) == 0
    assert run(count=0) == 0
    assert run(p=none, g=none, m=none, rows=sizes(0, 3), columns=sizes(5, 0)) == 0   # empty matrices have no memory


def test_cpu_tensors_are_refused():
    from spherical_distortion import functional as F
    x, w, s = torch.zeros(2, 3, 8), torch.ones(8), torch.zeros(2, 8)
    calls = [lambda: F.add_layer_norm(x, None, w), lambda: F.add_layer_norm(x, x, w, w),
             lambda: F.add_layer_norm(x.clone().requires_grad_(), None, w), lambda: F.gated_scan(x, x),
             lambda: F.gated_scan(x.clone().requires_grad_(), x, s), lambda: F.gated_scan_step(s, s, s),
             lambda: F.orthogonalize(s), lambda: F.muon_step([s], [s], [s])]
    for call in calls:
        with pytest.raises((NotImplementedError, RuntimeError)):
            call()
    F.muon_step([], [], [])   # nothing to step


@pytest.mark.parametrize("width", [0, -3, 16385])
def test_norm_modules_refuse_at_once_what_no_call_takes(width):
    from spherical_distortion import nn as snn
    with pytest.raises(ValueError):
        snn.AddLayerNorm(width)


@pytest.mark.parametrize("settings", [dict(width=0), dict(width=8, channels=0), dict(width=8, channels=(1 << 20) + 1),
                                      dict(width=8, channels=7, both_ways=True)])
def test_scan_modules_refuse_at_once_what_no_call_takes(settings):
    from spherical_distortion import nn as snn
    with pytest.raises(ValueError):
        snn.GatedScan(**settings)


def test_scans_both_ways_refuse_states_and_single_tokens():
    from spherical_distortion import nn as snn
    layer = snn.GatedScan(6, 8, both_ways=True)
    with pytest.raises(ValueError):
        layer(torch.zeros(1, 2, 6), torch.zeros(1, 8))
    with pytest.raises(ValueError):
        layer.step(torch.zeros(1, 6), torch.zeros(1, 8))


# --------------------------------------------------------------------------- the optimizer
def _params():
    torch.manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(*s)) for s in ((5, 7), (50, 3, 9))]
    for p in params:
        p.grad = torch.ones_like(p)
    return params


@pytest.mark.parametrize("settings", [dict(lr=-1.0), dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-1.0), dict(steps=0),
                                      dict(steps=101), dict(eps=0.0), dict(coefficients=(1.0, 2.0)), dict(coefficients=(20.0, 0, 0))])
def test_muon_refuses_settings_at_once(settings):
    from spherical_distortion.optim import Muon
    with pytest.raises(ValueError):
        Muon(_params(), **settings)
    optimizer = Muon(_params())
    with pytest.raises(ValueError):
        optimizer.add_param_group(dict(params=_params(), **settings))
    assert len(optimizer.param_groups) == 1


def test_muon_refuses_vectors():
    from spherical_distortion.optim import Muon
    with pytest.raises(ValueError, match="two axes"):
        Muon([torch.nn.Parameter(torch.zeros(3))])


@pytest.fixture
def steps_on_the_cpu(monkeypatch):
    """The step in plain tensor operations, so that the optimizer runs here; raises on demand."""
    from spherical_distortion.optim import adamw, muon
    calls = []

    class fail:
        now = False

    def step(params, grads, momenta, **settings):
        if fail.now:
            raise RuntimeError("no")
        calls.append((len(params), settings))
        for p, g, m in zip(params, grads, momenta):
            m.add_(g)
            p.sub_(m)
    monkeypatch.setattr(muon.F, "muon_step", step)
    monkeypatch.setattr(adamw, "_on_gpu", lambda p: True)
    return fail, calls


def test_muon_keeps_no_state_of_a_step_that_raised(steps_on_the_cpu):
    from spherical_distortion.optim import Muon
    fail, calls = steps_on_the_cpu
    params = _params()
    optimizer = Muon([dict(params=params[:1]), dict(params=params[1:], lr=1.0, nesterov=False)])
    fail.now = True
    with pytest.raises(RuntimeError, match="no"):
        optimizer.step()
    assert not optimizer.state
    fail.now = False
    params[0].grad = None   # left as it is
    optimizer.step()
    assert list(optimizer.state) == params[1:] and len(calls) == 1
    assert calls[0][1]["lr"] == 1.0 and calls[0][1]["nesterov"] is False
    params[0].grad = torch.ones_like(params[0])
    assert optimizer.step(lambda: 7) == 7
    assert len(calls) == 3


def test_a_parameter_that_cannot_be_stepped_stops_all_before_any(steps_on_the_cpu):
    from spherical_distortion.optim import Muon
    for make in (lambda: torch.nn.Parameter(torch.randn(4, 4).double()),
                 lambda: torch.nn.Parameter(torch.randn(2, 3, 4, 4).to(memory_format=torch.channels_last))):
        params, bad = _params(), make()
        bad.grad = torch.ones_like(bad)
        values = [p.detach().clone() for p in params]
        optimizer = Muon([{"params": params}, {"params": [bad]}])
        with pytest.raises(RuntimeError):
            optimizer.step()
        assert all(torch.equal(p, v) for p, v in zip(params, values)) and not optimizer.state


def test_parameters_on_the_cpu_are_refused_before_any_state():
    from spherical_distortion.optim import Muon
    optimizer = Muon(_params())
    with pytest.raises(RuntimeError, match="GPU"):
        optimizer.step()
    assert not optimizer.state
