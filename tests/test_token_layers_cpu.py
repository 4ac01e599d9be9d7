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
