"""Rows that the kernels cannot read where they lie are copied: dense tensors at addresses that are no multiple of 16
bytes, tokens too far apart.  The bits of the same values laid out afresh."""
import pytest
import torch

from test_gpu_bucket_attention import DEV, _inputs

pytestmark = pytest.mark.gpu


def _at_odd_address(t):
    memory = torch.empty(t.numel() + 8, dtype=t.dtype, device=DEV)
    view = memory[1:1 + t.numel()].view(t.shape)
    view.copy_(t)
    assert view.is_contiguous() and view.data_ptr() % 16
    return view


def _run(q, k, v, table, bmap, do):
    from spherical_distortion import functional as F
    leaves = [t.detach().requires_grad_() for t in (q, k, v, table)]
    out = F.bucket_attention(*leaves, bmap)
    with torch.no_grad():
        assert torch.equal(F.bucket_attention(*leaves, bmap), out)
    return (out, *torch.autograd.grad(out, leaves, do))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lq", [2, 90])
def test_dense_tensors_at_odd_addresses(lq, dtype):
    tensors = _inputs(2, 4, 2, lq, 100, 40, 7, dtype, seed=70 + lq)
    want = _run(*tensors)
    for i in range(6):
        moved = [_at_odd_address(t) if j == i else t for j, t in enumerate(tensors)]
        for a, b in zip(_run(*moved), want):
            assert torch.equal(a, b)
    for a, b in zip(_run(*(_at_odd_address(t) for t in tensors)), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("python", [False, True])
def test_an_output_and_its_rest_laid_out_differently(python):
    """The backward reads both by the same strides, wherever each of them lies."""
    from _spherical_distortion_ext import _token_ops
    q, k, v, table, bmap, do = _inputs(2, 4, 2, 30, 50, 32, 7, torch.bfloat16, seed=73)
    q = q.transpose(1, 2).contiguous().transpose(1, 2)   # the output is laid out as it is
    settings = (False, 0.2, True, True, True)
    out, rest, lse = _token_ops.ops.bucket_attention_forward(q, k, v, table, bmap, None, False, 0.2)
    assert out.stride() == q.stride()
    backward = (_token_ops.PYTHON_IMPL["bucket_attention_backward"] if python
                else _token_ops.ops.bucket_attention_backward)
    want = backward(do, q, k, v, table, bmap, None, out, rest, lse, *settings)

    def moved(t):
        return _at_odd_address(t.transpose(1, 2).contiguous()).transpose(1, 2)
    for o, r in ((moved(out), rest), (out, moved(rest)), (moved(out), moved(rest))):
        assert o.stride() == r.stride()
        for a, b in zip(backward(do, q, k, v, table, bmap, None, o, r, lse, *settings), want):
            assert torch.equal(a, b)


def test_tokens_too_far_apart_are_copied():
    """Keys 2^25 elements apart in 4.3 GB: 64 of them span more than 2^31 bytes."""
    q, k, v, table, bmap, do = _inputs(1, 2, 1, 9, 64, 16, 5, torch.bfloat16, seed=74)
    want = _run(q, k, v, table, bmap, do)
    memory = torch.empty(64 << 25, dtype=torch.bfloat16, device=DEV)
    far = []
    for i, t in enumerate((k, v)):
        view = memory.as_strided((1, 1, 64, 16), (1 << 25, 1 << 25, 1 << 25, 1), storage_offset=16 * i)
        view.copy_(t)
        far.append(view)
    for a, b in zip(_run(q, *far, table, bmap, do), want):
        assert torch.equal(a, b)
