"""Muon's steps in captured graphs: as eager ones, each of them, once a parameter has a momentum."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _params(dtype):
    g = torch.Generator().manual_seed(0)
    params = [torch.nn.Parameter(torch.randn(*s, generator=g).to(dtype).to(DEV)) for s in ((16, 3, 9), (70, 40), (130, 200))]
    for p in params:
        p.grad = torch.randn(*p.shape, generator=g).to(dtype).to(DEV)
    return params


def test_a_first_step_is_not_captured():
    """Its momentum would begin as zeros again in every replay."""
    from spherical_distortion.optim import Muon
    params = _params(torch.float32)
    before = [p.detach().clone() for p in params]
    optimizer = Muon(params)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            optimizer.step()
    torch.cuda.synchronize()
    assert not optimizer.state and all(torch.equal(p, q) for p, q in zip(params, before))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_replays_are_steps(dtype):
    from spherical_distortion.optim import Muon
    params, twins = _params(dtype), _params(dtype)
    optimizer, twin = Muon(params, weight_decay=0.1), Muon(twins, weight_decay=0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        optimizer.step()
    torch.cuda.current_stream().wait_stream(side)
    twin.step()
    graph = torch.cuda.CUDAGraph()
    held = copy.deepcopy([p.detach() for p in params])
    with torch.cuda.graph(graph):
        optimizer.step()
    assert all(torch.equal(p, q) for p, q in zip(params, held))   # captured, not run
    for i in range(4):
        for p, q in zip(params, twins):
            new = torch.randn(*p.shape, generator=torch.Generator().manual_seed(i)).to(dtype).to(DEV)
            p.grad.copy_(new), q.grad.copy_(new)
        graph.replay()
        twin.step()
        torch.cuda.synchronize()
        for p, q in zip(params, twins):
            assert torch.equal(p, q) and torch.equal(optimizer.state[p]["momentum"], twin.state[q]["momentum"])
