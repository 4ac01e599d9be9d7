"""Sizes of which one launch cannot hold every workgroup (fewer than 2^32 threads along a grid's axis): the bits of calls
on parts of the data."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _room(gib):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip("needs %d GiB of free GPU memory" % gib)


def test_norms_of_more_than_2_to_26_rows():
    from spherical_distortion import functional as F
    _room(16)
    rows, width, cut = (1 << 26) + 37, 16, 1 << 26
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(rows, width, generator=g, device=DEV, dtype=torch.bfloat16)
    w = torch.rand(width, generator=g, device=DEV)
    parts = [slice(0, 100), slice(cut - 100, cut - 1), slice(cut - 8, None)]
    y, h = F.add_rms_norm(x, x, w)
    for part in parts:
        a, b = F.add_rms_norm(x[part], x[part], w)
        assert torch.equal(y[part], a) and torch.equal(h[part], b)
    del y, h
    for dtype in (torch.int8, torch.float8_e4m3fn):
        codes, scales, h = F.add_rms_norm_quantized(x, x, w, dtype=dtype)
        for part in parts:
            a, b, c = F.add_rms_norm_quantized(x[part], x[part], w, dtype=dtype)
            assert torch.equal(codes[part].view(torch.uint8), a.view(torch.uint8))
            assert torch.equal(scales[part], b) and torch.equal(h[part], c)


def test_gradients_of_more_than_2_to_28_rows():
    """64 x 1024 heads of 4097 queries: the terms of each row."""
    from spherical_distortion import functional as F
    _room(60)
    B, H, L = 64, 1024, 4097
    g = torch.Generator(device=DEV).manual_seed(2)
    q, do = (torch.randn(B, H, L, 8, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    k, v = (torch.randn(B, H, 2, 8, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    table = torch.randn(H, 3, generator=g, device=DEV)
    bmap = torch.randint(0, 3, (L, 2), generator=g, device=DEV, dtype=torch.uint8)

    def run(part):
        leaves = [t[part].detach().requires_grad_() for t in (q, k, v)]
        return torch.autograd.grad(F.bucket_attention(*leaves, table, bmap), leaves, do[part])
    whole = run(slice(None))
    for part in (slice(0, 1), slice(B - 1, None)):
        for a, b in zip(whole, run(part)):
            assert torch.equal(a[part], b)


def test_a_bias_table_of_2_to_24_entries():
    from spherical_distortion import functional as F
    _room(4)
    H = 1 << 16
    g = torch.Generator(device=DEV).manual_seed(3)
    q, k, v, do = (torch.randn(1, H, 2, 8, generator=g, device=DEV) for _ in range(4))
    table = torch.randn(H, 256, generator=g, device=DEV).requires_grad_()
    bmap = torch.tensor([[0, 255], [7, 255]], device=DEV, dtype=torch.uint8)
    whole, = torch.autograd.grad(F.bucket_attention(q, k, v, table, bmap), [table], do)
    for part in (slice(0, 64), slice(H - 64, None)):
        some = table[part].detach().requires_grad_()
        got, = torch.autograd.grad(F.bucket_attention(q[:, part], k[:, part], v[:, part], some, bmap), [some], do[:, part])
        assert torch.equal(whole[part], got) and bool(got.any())


def test_a_map_of_2_to_36_pairs():
    """262144 x 262145 pairs: gradients of the last keys against a call on those alone.  Only the last queries have a
    gradient, and every other key is out of their reach."""
    from spherical_distortion import functional as F
    _room(190)
    n, last = 1 << 18, 256
    g = torch.Generator(device=DEV).manual_seed(4)
    q, do = (torch.randn(1, 1, n, 8, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    k, v = (torch.randn(1, 1, n + 1, 8, generator=g, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    table = torch.randn(1, 40, generator=g, device=DEV)
    bmap = torch.full((n, n + 1), 255, device=DEV, dtype=torch.uint8)
    bmap[-last:, -last:] = torch.randint(0, 40, (last, last), generator=g, device=DEV, dtype=torch.uint8)
    results = []
    for m, keys in ((bmap, slice(None)), (bmap[-last:, -last:].contiguous(), slice(-last, None))):
        leaves = [t.detach().requires_grad_() for t in (q[:, :, -m.shape[0]:], k[:, :, keys], v[:, :, keys])]
        grads = torch.autograd.grad(F.bucket_attention(*leaves, table, m), leaves, do[:, :, -m.shape[0]:])
        results.append([t[:, :, -last:] for t in grads])
    for a, b in zip(*results):   # the sums of a row in other parts and order: a rounding of bfloat16 apart
        assert float((a.double() - b.double()).abs().max()) <= 2.0 ** -7 * float(b.abs().max())


def test_codes_of_more_than_2_to_35_values():
    from spherical_distortion import functional as F
    _room(130)
    width = 1 << 20
    rows, cut = (1 << 15) + 3, 1 << 15
    codes = torch.randint(-127, 128, (rows, width), device=DEV, dtype=torch.int8)
    scales = torch.rand(rows, device=DEV)
    out = F.dequantize_rows(codes, scales, dtype=torch.bfloat16)
    for part in (slice(0, 2), slice(cut - 2, cut), slice(cut - 1, None)):
        assert torch.equal(out[part], F.dequantize_rows(codes[part], scales[part], dtype=torch.bfloat16))
        assert torch.equal(out[part], (codes[part].float() * scales[part, None]).to(torch.bfloat16))


@pytest.mark.parametrize("second", [False, True])
def test_moments_of_more_than_2_to_36_values(second):
    from spherical_distortion import functional as F
    _room(220)
    size, cut = (1 << 36) + 777, 1 << 36
    codes = torch.empty(size, device=DEV, dtype=torch.uint8 if second else torch.int8)
    parts = [slice(0, 1024), slice(cut - 8192, cut), slice(cut - 4096, None)]
    for part in parts:
        codes[part] = torch.randint(0, 127, codes[part].shape, device=DEV, dtype=codes.dtype)
    scales = torch.ones(-(-size // 256), device=DEV)
    out = F.adamw_moment_values(codes, scales, dtype=torch.bfloat16)
    for part in parts:
        some = codes[part].clone()
        assert torch.equal(out[part], F.adamw_moment_values(some, torch.ones(-(-some.numel() // 256), device=DEV),
                                                            dtype=torch.bfloat16))
