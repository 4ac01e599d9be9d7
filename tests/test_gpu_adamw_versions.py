"""A step counts as a change in place of the parameters and moments: autograd refuses a backward through values that it
replaced."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SETTINGS = (1e-2, 0.9, 0.99, 1e-8, 0.1, 1)


def _lists(bits):
    params = [torch.randn(300, device=DEV), torch.randn(7, 5, device=DEV)]
    grads = [torch.randn_like(p) for p in params]
    if bits == 32:
        return [params, grads, [torch.zeros_like(p) for p in params], [torch.zeros_like(p) for p in params]]
    scales = [[torch.zeros(-(-p.numel() // 256), device=DEV) for p in params] for _ in range(2)]
    codes = [[torch.zeros(p.shape, dtype=t, device=DEV) for p in params] for t in (torch.int8, torch.uint8)]
    return [params, grads, codes[0], scales[0], codes[1], scales[1]]


def _step(bits, python):
    from _spherical_distortion_ext import _token_ops
    name = "adamw_step" if bits == 32 else "adamw_step_8bit"
    return _token_ops.PYTHON_IMPL[name] if python else getattr(_token_ops.ops, name)


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_versions_grow(bits, python):
    lists = _lists(bits)
    before = [[t._version for t in tensors] for tensors in lists]
    values = [p.clone() for p in lists[0]]
    _step(bits, python)(*lists, *SETTINGS)
    assert all(not torch.equal(p, v) for p, v in zip(lists[0], values))
    for i, (tensors, versions) in enumerate(zip(lists, before)):
        for t, version in zip(tensors, versions):
            assert t._version == version if i == 1 else t._version > version   # gradients are read alone


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_view_and_its_base_count_together(bits, python):
    lists = [tensors[:1] for tensors in _lists(bits)]
    whole = torch.zeros(400, device=DEV)
    lists[0] = [whole[60:360]]
    _step(bits, python)(*lists, *SETTINGS)
    assert whole._version > 0 and bool(whole[60:360].any())


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_backward_through_replaced_weights_raises(bits, python):
    lists = _lists(bits)
    weight = lists[0][0].requires_grad_()
    x = torch.randn(300, device=DEV, requires_grad=True)
    kept = (weight * x).sum()
    with torch.no_grad():
        _step(bits, python)(*lists, *SETTINGS)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()


def test_the_optimizer_counts_its_steps_as_changes():
    from spherical_distortion.optim import AdamW
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.randn(5000, device=DEV))
        optimizer = AdamW([p], moment_bits=bits)
        x = torch.randn(5000, device=DEV, requires_grad=True)
        kept = (p * x).sum()
        p.grad = torch.randn_like(p)
        optimizer.step()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.backward()


@pytest.mark.parametrize("python", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_of_inference_mode_have_no_version(bits, python):
    with torch.inference_mode():
        lists = _lists(bits)
        values = lists[0][0].clone()
        _step(bits, python)(*lists, *SETTINGS)
        assert not torch.equal(lists[0][0], values)
