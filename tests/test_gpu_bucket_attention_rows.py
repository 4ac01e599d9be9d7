"""Rows that stand apart in the backward of attention with a bias for each bucket: those whose level lies beyond what a
sum can be added to.  Inputs, definition and bounds are those of test_gpu_bucket_attention."""
import math

import pytest
import torch

from test_gpu_bucket_attention import DEV, TOL, _close, _exact, _inputs, _terms

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("queries", [1, 33, 65, 70])
def test_a_masked_last_row_reads_nothing_behind_it(queries, dtype):
    """The last query of the last head has nothing but the lowest bias, and its tile ends behind it: what lies behind
    the rows' sums in memory (here NaN, in memory of this test) plays no part."""
    from _spherical_distortion_ext._token_ops import ops
    q, k, v, table, bmap, do = _inputs(2, 4, 2, queries, 90, 64, 6, dtype, seed=40 + queries)
    table[-1, 2] = torch.finfo(torch.float32).min
    bmap[-1] = 2
    scale = 64 ** -0.5
    out, rest, lse = ops.bucket_attention_forward(q, k, v, table, bmap, None, False, scale)
    memory = torch.full((lse.numel() + 256,), math.nan, device=DEV)
    held = memory[:lse.numel()].view(lse.shape)
    held.copy_(lse)
    grads = ops.bucket_attention_backward(do, q, k, v, table, bmap, None, out, rest, held, False, scale, True, True, True)
    want = _exact(q, k, v, table, bmap, grad=do)
    for got, ref, terms in zip((out, *grads), want, _terms(q, k, v, do)):
        _close(got, ref, TOL[dtype], terms)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [104, 128])
@pytest.mark.parametrize("heads,queries", [(32, 1), (8, 4)])
def test_few_queries_of_wide_heads(heads, queries, dim, dtype):
    """32 rows to one key head, the most that the kernel of few queries takes: in float32 its tiles, joined states and 32
    tables are the largest LDS of all calls (137 KB)."""
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(2, heads, 1, queries, 700, dim, 200, dtype, seed=80 + dim + heads)
    lengths = torch.tensor([700, 333], dtype=torch.int32)
    out = F.bucket_attention(q, k, v, table, bmap, key_lengths=lengths.to(DEV))
    _close(out, _exact(q, k, v, table, bmap, lengths), TOL[dtype])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("buckets", [20, 200])
@pytest.mark.parametrize("lq,lk", [(70, 90), (150, 700), (3, 700)])
def test_rows_of_large_scores(lq, lk, buckets, dtype):
    """A scale of 150: most rows' largest score lies beyond 1024 powers of two, some rows' below, with weights that differ.
    A score of magnitude S is off by up to 2^-20 S (the order of its 64 float32 terms, exponent and level), and its weight
    by as much of itself, twice in a gradient, whose terms have the scale as a factor."""
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(1, 4, 2, lq, lk, 64, buckets, dtype, seed=90 + lk + buckets)
    q[:, :, ::3] /= 64
    scale = 150.0
    size = scale * float((q.double().abs() @ k.double().abs().repeat_interleave(2, 1).transpose(2, 3).contiguous()).max())
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    out = F.bucket_attention(*leaves, bmap, scale=scale)
    grads = torch.autograd.grad(out, leaves, do)
    want = _exact(q, k, v, table, bmap, scale=scale, grad=do)
    assert size > 5000
    for got, ref, terms, factor in zip((out, *grads), want, _terms(q, k, v, do), (1, scale, scale, 1, 1)):
        _close(got, ref, TOL[dtype] + 2.0 ** -19 * size, terms * factor)
