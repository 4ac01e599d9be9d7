"""float16 gradients of attention with a bias for each bucket where rows, keys and heads differ in size by many powers of
two: each keeps float16's precision beside the others.

Bounds, of one row's (dq) or one key's (dk, dv) own terms: a sum over n pairs of products of three factors.  The
weight and the ds of a pair are each rounded to 11 bits (2^-11 of the pair's term, in either direction), D is as
exact as a float32 sum, and the result is rounded once: 4 * 2^-11 of the sum of the terms' magnitudes holds all of it.
The terms of dq_i are |ds_ij| |k_j| scale, with |ds_ij| no more than p_ij (|do_i v_j| + |D_i|), and so on.  Results below
2^-14 are float16's subnormal numbers: 2^-25 each.  What lies far below a row's or key's own largest pair may be lost:
2^-24 of that pair's term for each of n pairs, far less than the first bound for n below 2^10."""
import math

import pytest
import torch

from test_gpu_bucket_attention import DEV, _exact, _inputs

pytestmark = pytest.mark.gpu
U = 2.0 ** -11


def _bounds(q, k, v, table, bmap, do, causal=False):
    """Sums of the magnitudes of each gradient's terms, in float64 on the CPU."""
    q, k, v, table, do = (t.detach().double().cpu() for t in (q, k, v, table, do))
    bmap = bmap.cpu().long()
    B, H, Lq, D = q.shape
    Hk, Lk = k.shape[1:3]
    G, NB, scale = H // Hk, table.shape[1], D ** -0.5
    seen = bmap < NB
    if causal:
        seen = seen & (torch.arange(Lk)[None] <= torch.arange(Lq)[:, None] + (Lk - Lq))
    dq, dk, dv, dt = (torch.zeros_like(t) for t in (q, k, v, table))
    for b in range(B):
        for h in range(H):
            kk, vv, g = k[b, h // G], v[b, h // G], do[b, h]
            s = (scale * q[b, h] @ kk.T + table[h][bmap.clamp(max=NB - 1)]).masked_fill(~seen, -math.inf)
            p = torch.softmax(s, 1).nan_to_num(0.0)
            each = g.abs() @ vv.abs().T                       # the terms of do v
            ds = p * (each + (p * each).sum(1, keepdim=True))
            dq[b, h] = scale * ds @ kk.abs()
            dk[b, h // G] += scale * ds.T @ q[b, h].abs()
            dv[b, h // G] += p.T @ g.abs()
            dt[h].index_add_(0, bmap[seen], ds[seen])
    return dq, dk, dv, dt


def _check(q, k, v, table, bmap, do, causal=False):
    from spherical_distortion import functional as F
    leaves = [t.detach().requires_grad_() for t in (q, k, v, table)]
    grads = torch.autograd.grad(F.bucket_attention(*leaves, bmap, causal=causal), leaves, do)
    want = _exact(q, k, v, table, bmap, causal=causal, grad=do)[1:]
    for name, got, ref, bound in zip(("query", "key", "value", "table"), grads, want,
                                     _bounds(q, k, v, table, bmap, do, causal)):
        got = got.double().cpu()
        inside = ref.abs() < 60000                            # beyond it float16 has no such number
        assert bool(torch.isfinite(got[inside]).all()), name
        worst = ((got - ref).abs() / (4 * U * bound + 2.0 ** -25))[inside].max()
        assert float(worst) <= 1, (name, float(worst))


@pytest.mark.parametrize("buckets", [20, 100, 200])
@pytest.mark.parametrize("dim", [24, 64, 96, 128])
def test_one_large_row(dim, buckets):
    """The gradient of one query is 2^14 times the others'."""
    q, k, v, table, bmap, do = _inputs(1, 4, 2, 150, 170, dim, buckets, torch.float16, seed=50 + dim + buckets)
    do = do * 2.0 ** -8
    do[0, 1, 70] *= 2.0 ** 14
    _check(q, k, v, table, bmap, do)


def test_rows_of_every_size():
    """Rows from 2^-14 to 2^12, neighbours far apart."""
    q, k, v, table, bmap, do = _inputs(2, 4, 2, 200, 260, 64, 30, torch.float16, seed=61)
    g = torch.Generator().manual_seed(61)
    do = (do.float() * 2.0 ** torch.randint(-14, 13, (2, 4, 200, 1), generator=g).to(DEV)).half()
    _check(q, k, v, table, bmap, do)


def test_a_large_row_that_later_keys_do_not_see():
    """Causal, the first query's gradient 2^15 times the others': keys that it does not see keep their own size."""
    q, k, v, table, bmap, do = _inputs(1, 4, 1, 300, 300, 64, 30, torch.float16, seed=62)
    do = do * 2.0 ** -9
    do[:, :, 0] *= 2.0 ** 15
    _check(q, k, v, table, bmap, do, causal=True)


@pytest.mark.parametrize("head", [0, 1])
def test_one_large_head(head):
    """The gradient of a sequence's head is 2^14 times the others', first or last."""
    q, k, v, table, bmap, do = _inputs(2, 2, 2, 90, 140, 40, 12, torch.float16, seed=63)
    do = do * 2.0 ** -6
    do[head, head] *= 2.0 ** 14
    _check(q, k, v, table, bmap, do)


@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** 6, 2.0 ** 10, 2.0 ** 13])
@pytest.mark.parametrize("dim,keys", [(32, 3), (128, 3), (32, 200), (128, 200)])
def test_values_of_any_size(dim, keys, size):
    """Values far from one, gradients along them: do v and ds lie far beyond 65504, or among the smallest numbers,
    before they are summed."""
    q, k, v, table, bmap, do = _inputs(1, 2, 1, 70, keys, dim, 12, torch.float16, seed=64 + dim + keys)
    v = (v.float().clamp(-4, 4) * size).half()
    do = (v[:, :, torch.arange(70) % keys].float() / size * 2.0 ** -3).expand(1, 2, 70, dim).half().contiguous()
    _check(q, k, v, table, bmap, do)


def test_growing_and_shrinking_rows():
    """Rows that grow, and rows that shrink, by 2^27 over the walk: the sums' power of two follows."""
    q, k, v, table, bmap, do = _inputs(1, 2, 2, 500, 100, 64, 12, torch.float16, seed=66)
    ramp = 2.0 ** torch.linspace(-14, 13, 500, device=DEV)
    do = (do.float() * torch.stack([ramp, ramp.flip(0)])[None, :, :, None]).half()
    _check(q, k, v, table, bmap, do)
