"""What a step of Muon refuses, before it changes a parameter of any group."""
import pytest
import torch


@pytest.fixture
def steps(monkeypatch):
    """The step in plain tensor operations, so that the optimizer runs here."""
    from spherical_distortion.optim import adamw, muon
    calls = []

    def step(params, grads, momenta, **settings):
        calls.append(len(params))
        for p, g, m in zip(params, grads, momenta):
            m.add_(g)
            p.sub_(m)
    monkeypatch.setattr(muon.F, "muon_step", step)
    monkeypatch.setattr(adamw, "_on_gpu", lambda p: True)
    return calls


def _param(*shape):
    p = torch.nn.Parameter(torch.randn(*shape))
    p.grad = torch.ones_like(p)
    return p


def _refused(optimizer, calls):
    held = [p for g in optimizer.param_groups for p in g["params"]]
    values = [p.detach().clone() for p in held]
    with pytest.raises((RuntimeError, ValueError)):
        optimizer.step()
    assert not calls and not optimizer.state
    assert all(torch.equal(p, v) for p, v in zip(held, values))


@pytest.mark.parametrize("change", [dict(lr=-0.1), dict(lr=float("nan")), dict(lr=float("inf")), dict(weight_decay=1e31), dict(momentum=1.0), dict(weight_decay=-1.0), dict(steps=0),
                                    dict(coefficients=(20.0, 0.0, 0.0)), dict(eps=0.0)])
def test_settings_that_were_changed_since(steps, change):
    from spherical_distortion.optim import Muon
    optimizer = Muon([dict(params=[_param(4, 5)]), dict(params=[_param(6, 5)])])
    optimizer.param_groups[1].update(change)
    _refused(optimizer, steps)
    optimizer.param_groups[1]["params"][0].grad = None   # a group that is not stepped
    optimizer.step()
    assert steps == [1]


@pytest.mark.filterwarnings("ignore:optimizer contains a parameter group with duplicate parameters")
def test_memory_that_is_listed_twice(steps):
    from spherical_distortion.optim import Muon
    first, twice = _param(4, 5), _param(6, 5)
    _refused(Muon([dict(params=[first]), dict(params=[twice, twice])]), steps)
    tied = torch.nn.Parameter(twice.data)   # another parameter of the same memory
    tied.grad = torch.ones_like(tied)
    _refused(Muon([dict(params=[first]), dict(params=[twice]), dict(params=[tied])]), steps)
    tied = _param(4, 5)
    tied.grad = first.detach()              # a gradient that is a parameter
    _refused(Muon([dict(params=[first]), dict(params=[tied])]), steps)
    empty = [_param(0, 5), _param(0, 7)]    # which share an address, or have none
    Muon([dict(params=empty), dict(params=[first])]).step()
    assert steps


def test_momenta_of_another_model(steps):
    from spherical_distortion.optim import Muon
    old = Muon([_param(4, 5), _param(7, 5)])
    old.step()
    new = Muon([dict(params=[_param(4, 5)]), dict(params=[_param(6, 5)])])
    state = old.state_dict()
    state["param_groups"] = new.state_dict()["param_groups"]
    new.load_state_dict(state)
    steps.clear()
    values = [p.detach().clone() for g in new.param_groups for p in g["params"]]
    with pytest.raises(RuntimeError, match="momentum"):
        new.step()
    assert not steps and all(torch.equal(p, v) for p, v in zip([p for g in new.param_groups for p in g["params"]], values))


def test_sides_that_no_call_takes(steps):
    """Refused with a gradient; one without is left as it is."""
    from spherical_distortion.optim import Muon
    for shape in (((1 << 17) + 1, 2), (1 << 20, 0), (2, (1 << 17) + 1), (3, 1 << 9, 1 << 9)):
        big = _param(*shape)
        optimizer = Muon([dict(params=[_param(4, 5)]), dict(params=[big])])
        _refused(optimizer, steps)
        big.grad = None
        optimizer.step()
        assert steps == [1]
        steps.clear()
    for shape in ((1 << 17, (1 << 14) + 1), (1 << 16, 1 << 16)):
        with pytest.raises(RuntimeError, match="131072"):
            Muon._check_sides(torch.empty(shape, device="meta"))
    for shape in ((1 << 17, 1 << 14), (0, 1 << 20), (1 << 17, 0)):
        Muon._check_sides(torch.empty(shape, device="meta"))


@pytest.mark.parametrize("default", [torch.float64, torch.bfloat16])
def test_momenta_are_float32_whatever_the_default_type(steps, default):
    from spherical_distortion.optim import Muon
    p = _param(4, 5)
    optimizer = Muon([p])
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        optimizer.step()
    finally:
        torch.set_default_dtype(before)
    assert optimizer.state[p]["momentum"].dtype == torch.float32


def test_a_state_that_was_only_looked_at(steps):
    """optimizer.state makes an entry for whoever is looked up."""
    from spherical_distortion.optim import Muon
    p = _param(4, 5)
    optimizer = Muon([p])
    assert not optimizer.state[p]
    optimizer.step()
    assert torch.equal(optimizer.state[p]["momentum"], p.grad)
