"""The optimizer and the modules of the token operators without a GPU: what they refuse, and what a refusal leaves."""
import copy

import pytest
import torch


@pytest.fixture
def steps_on_the_cpu(monkeypatch):
    """The operators' steps in plain tensor operations, so that the optimizer runs here; raises on demand."""
    from spherical_distortion.optim import adamw
    calls = []

    class fail:
        now = False

    def step(params, grads, *state, step, lr, betas, eps, weight_decay):
        if fail.now:
            raise RuntimeError("no")
        calls.append((len(params), step))
        for p, g in zip(params, grads):
            p -= lr * g
    monkeypatch.setattr(adamw.F, "adamw_step", step)
    monkeypatch.setattr(adamw.F, "adamw_step_8bit", step)
    monkeypatch.setattr(adamw, "_on_gpu", lambda p: True, raising=False)
    return fail, calls


def _params():
    torch.manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(*s)) for s in ((5, 7), (5000,), (3,))]
    for p in params:
        p.grad = torch.ones_like(p)
    return params


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_that_raises_is_not_counted(steps_on_the_cpu, bits):
    from spherical_distortion.optim import AdamW
    fail, calls = steps_on_the_cpu
    params = _params()
    optimizer = AdamW([{"params": params[:2]}, {"params": params[2:]}], moment_bits=bits)
    optimizer.step()
    before = copy.deepcopy(optimizer.state_dict())
    fail.now = True
    for _ in range(2):
        with pytest.raises(RuntimeError, match="no"):
            optimizer.step()
    assert optimizer.state_dict()["state"].keys() == before["state"].keys()
    assert [optimizer.state[p]["step"] for p in params] == [1, 1, 1]
    fail.now = False
    optimizer.step()
    assert [optimizer.state[p]["step"] for p in params] == [2, 2, 2] and calls[-1][1] == 2


BAD = {
    "type": lambda: torch.nn.Parameter(torch.randn(4, 4).double()),
    "layout": lambda: torch.nn.Parameter(torch.randn(2, 3, 4, 4).to(memory_format=torch.channels_last)),
    "sparse": lambda: torch.nn.Parameter(torch.randn(4, 4)),
}


@pytest.mark.parametrize("what", BAD)
def test_a_parameter_that_cannot_be_stepped_stops_all_before_any(steps_on_the_cpu, what):
    from spherical_distortion.optim import AdamW
    params = _params()
    bad = BAD[what]()
    bad.grad = torch.ones_like(bad).to_sparse() if what == "sparse" else torch.ones_like(bad)
    values = [p.detach().clone() for p in params]
    optimizer = AdamW([{"params": params}, {"params": [bad]}])
    with pytest.raises(RuntimeError):
        optimizer.step()
    assert all(torch.equal(p, v) for p, v in zip(params, values))
    assert not optimizer.state and not steps_on_the_cpu[1]


def test_parameters_on_the_cpu_are_refused_before_any_state():
    from spherical_distortion.optim import AdamW
    p = _params()[0]
    optimizer = AdamW([p])
    with pytest.raises(RuntimeError, match="GPU"):
        optimizer.step()
    assert not optimizer.state


@pytest.mark.parametrize("width,heads,buckets", [(96, 8, 9), (20, 5, 9), (1040, 8, 9), (64, 4, 0), (64, 4, 257)])
def test_attention_modules_refuse_at_once_what_no_call_takes(width, heads, buckets):
    """Heads of 12, 4 and 130 values, tables of 0 and 257 buckets."""
    from spherical_distortion import nn as snn
    with pytest.raises(ValueError):
        snn.BucketAttention(width, heads, buckets)


def test_attention_modules_take_every_size_of_a_call():
    from spherical_distortion import nn as snn
    for width, heads, buckets in ((8, 1, 1), (128, 1, 256), (1024, 8, 255)):
        assert snn.BucketAttention(width, heads, buckets).bias_table.shape == (heads, buckets)


@pytest.mark.parametrize("width", [0, -1, 16385])
def test_norm_modules_refuse_at_once_what_no_call_takes(width):
    from spherical_distortion import nn as snn
    with pytest.raises(ValueError):
        snn.AddRMSNorm(width)
    assert snn.AddRMSNorm(16384).weight.shape == (16384,)
