"""Attention with a bias for each bucket of relative positions, against its definition in float64 on the
CPU: forward, the gradients of queries, keys, values and bias table, and the forms of serving.

Tolerances, of the largest value of an output (norm-relative): a sum of products of values rounded to a type
with unit roundoff u is off by a few u where the weights p and ds are rounded once before the second product and
the result once more; 4 u covers both and the order of float32 sums: 2^-7 / 2 = 1.6e-2 for bfloat16, 2e-3 for
float16.  float32: the exponent of exp2 is off by 2^-24 of its magnitude (up to 2^5 here), so p by 2^-24 * 32 * ln 2
= 1.3e-6; sums over at most 700 terms of either sign add less than as much again: 4e-6.
ds is the difference of two float32 sums over the head's values, which cancel where a row has one key: an absolute
term of 2^-22 of the sum's terms comes on top of the relative one.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = {torch.float32: 4e-6, torch.bfloat16: 1.6e-2, torch.float16: 2e-3}


def _exact(q, k, v, table, bmap, lengths=None, causal=False, scale=None, grad=None):
    """Definition in float64 on the CPU; with grad also the gradients of q, k, v and table."""
    q, k, v, table = (t.detach().double().cpu() for t in (q, k, v, table))
    bmap = bmap.cpu().long()
    B, H, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    G, NB = H // Hk, table.shape[1]
    scale = D ** -0.5 if scale is None else scale
    maps = bmap if bmap.dim() == 3 else bmap.expand(B, Lq, Lk)
    out, dq, dk, dv, dt = (torch.zeros_like(t) for t in (q, q, k, v, table))
    for b in range(B):
        n = Lk if lengths is None else int(lengths[b])
        m = maps[b, :, :n]
        seen = m < NB
        if causal:
            seen = seen & (torch.arange(n)[None] <= torch.arange(Lq)[:, None] + (n - Lq))
        for h in range(H):
            kk, vv = k[b, h // G, :n], v[b, h // G, :n]
            s = scale * (q[b, h] @ kk.T) + table[h][m.clamp(max=NB - 1)]
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(1, keepdim=True) if n else torch.zeros(Lq, 1, dtype=torch.float64)
            p = torch.exp(s - torch.where(top.isinf(), 0.0, top))
            total = p.sum(1, keepdim=True)
            p = torch.where(total > 0, p / total, 0.0)
            out[b, h] = p @ vv
            if grad is not None:
                g = grad[b, h].double().cpu()
                ds = p * (g @ vv.T - (g * out[b, h]).sum(1, keepdim=True))
                dq[b, h] = scale * ds @ kk
                dk[b, h // G, :n] += scale * ds.T @ q[b, h]
                dv[b, h // G, :n] += p.T @ g
                dt[h].index_add_(0, m[seen], ds[seen])
    return out if grad is None else (out, dq, dk, dv, dt)


def _close(got, want, tol, terms=0.0):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    assert bool(torch.isfinite(got).all())
    if got.numel():
        assert float((got - want).abs().max()) <= tol * float(want.abs().max()) + 2.0 ** -22 * terms


def _terms(q, k, v, do):
    """Size of the terms that cancel in the gradients: |do| |v| of a pair times the other operand."""
    each = float(do.detach().double().norm(dim=-1).max() * v.detach().double().norm(dim=-1).max())
    return (0.0, each * float(k.detach().abs().max()), each * float(q.detach().abs().max()), 0.0, each)


def _inputs(B, H, Hk, Lq, Lk, D, NB, dtype, seed, out_share=0.0, per_batch=False):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(*s, generator=g).to(dtype).to(DEV)
                   for s in ((B, H, Lq, D), (B, Hk, Lk, D), (B, Hk, Lk, D), (B, H, Lq, D)))
    table = torch.randn(H, NB, generator=g).to(DEV)
    bmap = torch.randint(0, NB, ((B, Lq, Lk) if per_batch else (Lq, Lk)), generator=g)
    if out_share:
        bmap[torch.rand(bmap.shape, generator=g) < out_share] = 255
    return q, k, v, table, bmap.to(torch.uint8).to(DEV), do


SHAPES = [  # B, H, Hk, Lq, Lk, D, buckets
    (1, 1, 1, 1, 1, 8, 1),
    (2, 3, 1, 7, 5, 16, 2),
    (1, 4, 2, 31, 33, 24, 9),
    (2, 2, 2, 64, 64, 32, 32),
    (1, 6, 2, 65, 127, 40, 33),
    (1, 2, 1, 129, 191, 64, 64),
    (2, 4, 1, 128, 257, 72, 65),
    (1, 3, 3, 200, 130, 128, 129),
    (1, 2, 2, 33, 700, 96, 250),
    (1, 8, 1, 5, 600, 128, 256),
    (2, 2, 1, 9, 300, 88, 12),
    (1, 2, 2, 40, 90, 112, 17),
    (1, 4, 1, 150, 140, 96, 40),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(shape, dtype):
    from spherical_distortion import functional as F
    B, H, Hk, Lq, Lk, D, NB = shape
    q, k, v, table, bmap, do = _inputs(*shape, dtype, seed=sum(shape), out_share=0.1 if NB < 255 else 0.0)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    out = F.bucket_attention(*leaves, bmap)
    grads = torch.autograd.grad(out, leaves, do)
    want = _exact(q, k, v, table, bmap, grad=do)
    for got, ref, terms in zip((out, *grads), want, _terms(q, k, v, do)):
        _close(got, ref, TOL[dtype], terms)
    assert [g.dtype for g in grads] == [dtype] * 3 + [torch.float32]
    with torch.no_grad():
        assert torch.equal(F.bucket_attention(*leaves, bmap), out)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", [(100, 100), (37, 260), (260, 37), (1, 300), (3, 70)])
def test_lengths_causal_and_maps_of_each_sequence(dtype, causal, lq, lk):
    """Lengths of zero, one and all; keys and values beyond a length hold NaN and infinity."""
    from spherical_distortion import functional as F
    lengths = torch.tensor([lk, 0, 1, lk // 2], dtype=torch.int32)
    q, k, v, table, bmap, do = _inputs(4, 4, 2, lq, lk, 48, 20, dtype, seed=lq + lk, out_share=0.2, per_batch=True)
    for b in range(4):
        k[b, :, int(lengths[b]):] = math.nan
        v[b, :, int(lengths[b]):] = math.inf
    clean_k, clean_v = k.nan_to_num(0, 0, 0), v.nan_to_num(0, 0, 0)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    out = F.bucket_attention(*leaves, bmap, key_lengths=lengths.to(DEV), causal=causal)
    grads = torch.autograd.grad(out, leaves, do)
    want = _exact(q, clean_k, clean_v, table, bmap, lengths, causal, grad=do)
    for got, ref, terms in zip((out, *grads), want, _terms(q, clean_k, clean_v, do)):
        _close(got, ref, TOL[dtype], terms)
    assert not bool(out[1].any())   # a sequence without keys


def test_rows_and_columns_without_pairs():
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(2, 2, 1, 150, 170, 32, 12, torch.float32, seed=3)
    bmap[17] = 200
    bmap[128:] = 12          # the first value that is no bucket
    bmap[:, 40:60] = 255
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    out = F.bucket_attention(*leaves, bmap)
    grads = torch.autograd.grad(out, leaves, do)
    for got, ref in zip((out, *grads), _exact(q, k, v, table, bmap, grad=do)):
        _close(got, ref, TOL[torch.float32])
    for t in (out[:, :, 17], out[:, :, 128:], grads[0][:, :, 17], grads[1][:, :, 40:60], grads[2][:, :, 40:60]):
        assert not bool(t.any())
    everything = torch.full_like(bmap, 255)
    out = F.bucket_attention(*leaves, everything)
    assert not bool(out.any())
    for t in torch.autograd.grad(out, leaves, do):
        assert not bool(t.any())


@pytest.mark.parametrize("lowest", [torch.finfo(torch.float32).min, -math.inf, -1e30])
def test_biases_that_mask(lowest):
    """A bias of the type's lowest value: the pair's weight is zero beside others, and equal among
    themselves; -inf leaves the pair out."""
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(1, 2, 2, 70, 90, 64, 6, torch.float32, seed=5)
    table[0, 2] = lowest
    table[1, :] = lowest
    bmap[9] = 2
    out = F.bucket_attention(q, k, v, table, bmap)
    want = _exact(q, k, v, table, bmap)
    _close(out, want, TOL[torch.float32])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lowest", [torch.finfo(torch.float32).min, -1e30])
@pytest.mark.parametrize("buckets", [6, 40, 200])
@pytest.mark.parametrize("lq,lk", [(70, 90), (150, 700), (3, 700)])
def test_gradients_of_rows_that_biases_mask(lq, lk, buckets, lowest, dtype):
    """Rows all of whose biases are one lowest value (beside ordinary rows): equal weights, forward and backward,
    whatever part of the keys a workgroup takes."""
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(2, 4, 2, lq, lk, 64, buckets, dtype, seed=16 + lk)
    table[1] = lowest
    table[:, 2] = lowest
    bmap[1::5] = 2
    bmap[2] = 255
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    out = F.bucket_attention(*leaves, bmap)
    grads = torch.autograd.grad(out, leaves, do)
    want = _exact(q, k, v, table, bmap, grad=do)
    for got, ref, terms in zip((out, *grads), want, _terms(q, k, v, do)):
        _close(got, ref, TOL[dtype], terms)


@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** 12])
def test_small_and_large_gradients_of_float16(size):
    """Gradients as a loss scale leaves them: weights of 1 / 600 times gradients of 2^-12 lie far below float16's
    normal numbers, and times 2^12 near its largest.  Results that fall below 2^-14 are rounded to 2^-25."""
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(1, 4, 2, 300, 600, 64, 20, torch.float16, seed=7)
    do = do * size
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    grads = torch.autograd.grad(F.bucket_attention(*leaves, bmap), leaves, do)
    for got, ref in zip(grads, _exact(q, k, v, table, bmap, grad=do)[1:]):
        assert float((got.double().cpu() - ref).abs().max()) <= TOL[torch.float16] * float(ref.abs().max()) + 2.0 ** -25


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_table_gradients_that_cancel(dtype):
    """Two buckets: one key of each row, and all others.  Their gradients are opposite and small beside the terms
    summed: what one rounding of the output to 16 bits does to D (2^-9 or 2^-12 of about 0.3 a row) would show."""
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(1, 4, 2, 24, 1500, 112, 2, dtype, seed=19)
    bmap.fill_(1)
    bmap[torch.arange(24), torch.arange(24)] = 0
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    got, = torch.autograd.grad(F.bucket_attention(*leaves, bmap), leaves[3:], do)
    _close(got, _exact(q, k, v, table, bmap, grad=do)[4], TOL[dtype])


def test_bias_table_of_the_queries_type_and_scale():
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(2, 4, 2, 90, 110, 64, 30, torch.bfloat16, seed=6)
    table = table.to(torch.bfloat16)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    for scale in (0.01, 1.5):
        out = F.bucket_attention(*leaves, bmap, scale=scale)
        grads = torch.autograd.grad(out, leaves, do)
        assert grads[3].dtype == torch.bfloat16
        for got, ref in zip((out, *grads), _exact(q, k, v, table, bmap, scale=scale, grad=do)):
            _close(got, ref, TOL[torch.bfloat16])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_unaligned_views(dtype):
    """Heads packed beside each other, a map that is a view of a larger one at an odd address, rows that
    are not 16-byte aligned."""
    from spherical_distortion import functional as F
    g = torch.Generator().manual_seed(8)
    B, H, L, D, NB = 2, 3, 77, 32, 11
    packed = torch.randn(B, L, 3, H, D, generator=g).to(dtype).to(DEV)
    q, k, v = (packed[:, :, i].transpose(1, 2) for i in range(3))
    table = torch.randn(H, NB, generator=g).to(DEV)
    big = torch.randint(0, NB, (L + 2, L + 6), generator=g).to(torch.uint8).to(DEV)
    bmap = big[1:-1, 5:-1]
    _close(F.bucket_attention(q, k, v, table, bmap), _exact(q, k, v, table, bmap), TOL[dtype])
    wide = torch.randn(B, H, L, D + 3, generator=g).to(dtype).to(DEV)
    odd = wide[..., 1:-2]
    do = torch.randn(B, H, D, L, generator=g).to(dtype).to(DEV).transpose(2, 3)
    leaves = [t.detach().requires_grad_() for t in (odd, k, v, table)]
    out = F.bucket_attention(*leaves, bmap.t().contiguous().t())
    grads = torch.autograd.grad(out, leaves, do)
    for got, ref in zip((out, *grads), _exact(odd, k, v, table, bmap, grad=do)):
        _close(got, ref, TOL[dtype])


def test_gradients_against_differences():
    """Central differences of a weighted sum of the outputs in float32: its value is about 10, so a step of
    2^-6 gives quotients off by about 10 * 2^-22 / 2^-6 = 2e-4 from rounding and 1e-4 from the third
    derivative: 2e-3 of a gradient of order one."""
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(1, 2, 1, 9, 11, 16, 5, torch.float32, seed=11)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    grads = torch.autograd.grad(F.bucket_attention(*leaves, bmap), leaves, do)
    step = 2.0 ** -6
    g = torch.Generator().manual_seed(1)
    for i, grad in enumerate(grads):
        for _ in range(4):
            at = [int(torch.randint(0, n, (1,), generator=g)) for n in grad.shape]
            sides = []
            for sign in (1, -1):
                moved = [t.detach().clone() for t in leaves]
                moved[i][tuple(at)] += sign * step
                sides.append((F.bucket_attention(*moved, bmap).double() * do.double()).sum())
            want = float(sides[0] - sides[1]) / (2 * step)
            assert abs(float(grad[tuple(at)]) - want) <= 2e-3 * max(1.0, abs(want))


def test_gradients_that_are_not_wanted_and_repeated_runs():
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(2, 4, 2, 140, 150, 64, 40, torch.bfloat16, seed=12)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]
    full = torch.autograd.grad(F.bucket_attention(*leaves, bmap), leaves, do)
    again = torch.autograd.grad(F.bucket_attention(*leaves, bmap), leaves, do)
    for a, b in zip(full, again):
        assert torch.equal(a, b)   # every sum has one order
    for i in range(4):
        one = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        got, = torch.autograd.grad(F.bucket_attention(*one, bmap), [one[i]], do)
        assert torch.equal(got, full[i])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_empty_sizes(dtype):
    from spherical_distortion import functional as F
    for B, Lq, Lk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k, v, table, bmap, do = _inputs(B, 2, 1, Lq, Lk, 16, 3, dtype, seed=1)
        leaves = [t.requires_grad_() for t in (q, k, v, table)]
        out = F.bucket_attention(*leaves, bmap)
        assert out.shape == (B, 2, Lq, 16) and not bool(out.any())
        for t, g in zip(leaves, torch.autograd.grad(out, leaves, do)):
            assert g.shape == t.shape and not bool(g.any())


def test_another_stream_and_a_graph():
    """The pass on a side stream, and a captured one replayed with new inputs."""
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(1, 4, 1, 2, 900, 64, 30, torch.bfloat16, seed=13)
    want = F.bucket_attention(q, k, v, table, bmap)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = F.bucket_attention(q, k, v, table, bmap)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = F.bucket_attention(q, k, v, table, bmap)
    for seed in (20, 21, 22):
        fresh = _inputs(1, 4, 1, 2, 900, 64, 30, torch.bfloat16, seed=seed)
        for old, new in zip((q, k, v, table), fresh):
            old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, F.bucket_attention(q, k, v, table, bmap))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_expanded_keys(dtype):
    """One key head expanded over all heads, one token expanded over all positions: the bits of the same keys laid
    out."""
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(2, 4, 1, 90, 100, 32, 7, dtype, seed=14)
    for kk in (k.expand(2, 4, 100, 32), k[:, :, :1].expand(2, 1, 100, 32)):
        vv = v.expand(2, kk.shape[1], 100, 32)
        results = []
        for pair in ((kk, vv), (kk.contiguous(), vv.contiguous())):
            leaves = [t.detach().requires_grad_() for t in (q, *pair, table)]
            out = F.bucket_attention(*leaves, bmap)
            results.append((out, *torch.autograd.grad(out, leaves, do)))
        assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradients_in_a_graph(dtype):
    """Forward and backward captured, replayed with new inputs between eager calls: the same bits."""
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(1, 4, 2, 150, 170, 64, 30, dtype, seed=15)
    leaves = [t.requires_grad_() for t in (q, k, v, table)]

    def run():
        out = F.bucket_attention(*leaves, bmap)
        return [out.detach(), *torch.autograd.grad(out, leaves, do)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    for seed in (30, 31, 32):
        fresh = _inputs(1, 4, 2, 150, 170, 64, 30, dtype, seed=seed)
        with torch.no_grad():
            for old, new in zip((q, k, v, table, bmap, do), fresh):
                old.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, run()))


def test_no_second_derivative():
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(1, 1, 1, 4, 5, 8, 2, torch.float32, seed=1)
    q.requires_grad_()
    first, = torch.autograd.grad(F.bucket_attention(q, k, v, table, bmap), [q], do, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), [q])


@pytest.mark.parametrize("queries", [2, 200])
def test_offsets_beyond_32_bits(queries):
    """Keys and values whose tokens lie 2^22 elements apart, in 5.9 GB: the bits of dense ones, forward and backward."""
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(1, 2, 1, queries, 700, 64, 20, torch.bfloat16, seed=17)
    apart = 1 << 22
    memory = torch.empty(700 * apart, dtype=torch.bfloat16, device=DEV)
    results = []
    for far in (False, True):
        pair = []
        for i, t in enumerate((k, v)):
            if far:
                view = memory[64 * i:].as_strided((1, 1, 700, 64), (apart, apart, apart, 1), storage_offset=64 * i)
                view.copy_(t)
                t = view
            pair.append(t)
        leaves = [t.detach().requires_grad_() for t in (q, *pair, table)]
        out = F.bucket_attention(*leaves, bmap)
        results.append((out, *torch.autograd.grad(out, leaves, do)))
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_a_map_of_more_than_4_gb():
    """66000 x 66000 pairs: the last queries against a call of their own, forward and gradient."""
    from spherical_distortion import functional as F
    n, last = 66000, 300
    g = torch.Generator(device=DEV).manual_seed(18)
    q, k, v = (torch.randn(1, 1, n, 8, generator=g, device=DEV).to(torch.bfloat16) for _ in range(3))
    table = torch.randn(1, 40, generator=g, device=DEV)
    bmap = torch.randint(0, 40, (n, n), generator=g, device=DEV, dtype=torch.uint8)
    do = torch.zeros_like(q)
    do[:, :, -last:] = torch.randn(1, 1, last, 8, generator=g, device=DEV).to(torch.bfloat16)
    results = []
    for first in (0, n - last):
        leaves = [t.detach().requires_grad_() for t in (q[:, :, first:], k, v, table)]
        out = F.bucket_attention(*leaves, bmap[first:])
        grads = torch.autograd.grad(out, leaves, do[:, :, first:])
        results.append([t.detach().double().cpu() for t in (out[:, :, -last:], grads[0][:, :, -last:], *grads[1:])])
    for a, b in zip(*results):   # sums over 66000 keys in other parts: each within the type's bound of the exact one
        assert float((a - b).abs().max()) <= 2 * TOL[torch.bfloat16] * float(b.abs().max())


def test_refusals():
    from spherical_distortion import functional as F
    q, k, v, table, bmap, do = _inputs(2, 4, 2, 8, 9, 16, 3, torch.float32, seed=1)
    call = F.bucket_attention
    call(q, k, v, table, bmap)
    for bad in (dict(query=q.double()), dict(key=k.half()), dict(query=q[0]), dict(value=v[:, :, :-1]),
                dict(key=k[:, :1].expand(2, 3, 9, 16)[:, :3], value=v[:, :1].expand(2, 3, 9, 16)),
                dict(query=q[..., :12], key=k[..., :12], value=v[..., :12]), dict(bias_table=table[:2]),
                dict(bias_table=table.half()), dict(bias_table=table.repeat(1, 100)), dict(bucket_map=bmap.int()),
                dict(bucket_map=bmap[:, :-1]), dict(bucket_map=bmap.expand(3, 8, 9)), dict(scale=0.0),
                dict(scale=math.inf), dict(scale=-1.0), dict(key_lengths=torch.tensor([1, 2], device=DEV)),
                dict(key_lengths=torch.ones(3, dtype=torch.int32, device=DEV)),
                dict(key_lengths=torch.ones(2, dtype=torch.int32)), dict(bucket_map=bmap.cpu())):
        args = dict(query=q, key=k, value=v, bias_table=table, bucket_map=bmap) | bad
        with pytest.raises(RuntimeError):
            call(**args)
