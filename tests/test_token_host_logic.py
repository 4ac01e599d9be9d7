"""The operators on token sequences without a GPU: argument checks of the C entries (all of them before anything
touches the device), workspace sizes, and what the Python layer refuses."""
import ctypes

import pytest
import torch

ONE = ctypes.c_void_p(256)   # aligned, never dereferenced


@pytest.fixture(scope="module")
def lib():
    from _spherical_distortion_ext import _capi
    handle = _capi.load()
    handle.sdk_last_error.restype = ctypes.c_char_p
    return handle


def _attention(**changes):
    from _spherical_distortion_ext import _capi
    a = _capi.BucketAttention()
    for name in ("query", "key", "value", "bias_table", "bucket_map", "output", "lse", "grad_output"):
        setattr(a, name, 256)
    a.batch, a.heads, a.key_heads, a.queries, a.keys, a.dim, a.buckets = 2, 4, 2, 64, 4096, 64, 9
    for name in ("query", "key", "value", "output", "grad_output", "grad_query", "grad_key", "grad_value"):
        setattr(a, name + "_strides", (ctypes.c_int64 * 3)(1 << 20, 1 << 18, 64))
    a.map_strides = (ctypes.c_int64 * 2)(0, 4096)
    a.scale = 0.125
    for name, value in changes.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("changes,message", [
    (dict(dtype=1), "dtype"), (dict(dtype=9), "dtype"), (dict(table_dtype=2), "bias_table"), (dict(batch=-1), "negative"),
    (dict(heads=3), "multiple"), (dict(key_heads=0), "multiple"), (dict(dim=12), "dim"), (dict(dim=136), "dim"),
    (dict(dim=0), "dim"), (dict(buckets=0), "buckets"), (dict(buckets=257), "buckets"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(queries=1 << 30), "tokens"),
    (dict(batch=1 << 16), "batch"), (dict(query=None), "query"), (dict(key=None), "key"), (dict(value=264), "value"),
    (dict(bias_table=None), "bias_table"), (dict(bucket_map=None), "bucket_map"), (dict(output=None), "output"),
    (dict(query_strides=(ctypes.c_int64 * 3)(1 << 20, 1 << 18, 66)), "aligned"),
    (dict(key_strides=(ctypes.c_int64 * 3)(0, 0, 1 << 30)), "far"), (dict(output_rest=258, dtype=2, table_dtype=2), "output_rest"),
])
def test_attention_refuses(lib, changes, message):
    a = _attention(**changes)
    for entry in (lib.sdk_bucket_attention_forward, lib.sdk_bucket_attention_backward):
        assert entry(ctypes.byref(a), None, 0, None) == -1
        assert message in lib.sdk_last_error().decode()


def test_attention_workspaces(lib):
    size = lib.sdk_bucket_attention_workspace_bytes
    few = _attention(queries=1)
    parts = size(ctypes.byref(few), 0)
    # 4 key heads in all: 16 parts of 256 keys at most, dim + 2 floats a row and part
    assert parts == 16 * 2 * 4 * 1 * (64 + 2) * 4
    assert lib.sdk_bucket_attention_forward(ctypes.byref(few), None, 0, None) == -3
    assert lib.sdk_bucket_attention_forward(ctypes.byref(few), ONE, parts - 1, None) == -3
    assert "workspace" in lib.sdk_last_error().decode()
    full = _attention(batch=64, queries=2048)
    assert size(ctypes.byref(full), 0) == 0
    need = size(ctypes.byref(full), 1)
    assert need >= 64 * 4 * 2048 * 8 + 4096 * 2048   # D and level of each row, the map turned
    assert lib.sdk_bucket_attention_backward(ctypes.byref(full), None, 0, None) == -3
    assert size(ctypes.byref(_attention(dim=7)), 1) == 0
    assert size(ctypes.byref(_attention(batch=0)), 1) == 0
    # nothing to do is no error, pointers or not
    assert lib.sdk_bucket_attention_forward(ctypes.byref(_attention(batch=0, query=None)), None, 0, None) == 0
    assert lib.sdk_bucket_attention_forward(ctypes.byref(_attention(queries=0, query=None)), None, 0, None) == 0


def test_norm_refuses(lib):
    def run(x=ONE, weight=ONE, out=ONE, scales=None, rows=4, width=64, eps=1e-6, codes=0, dtype=0, weight_dtype=0):
        return lib.sdk_add_rms_norm(x, None, weight, out, scales, None, None, rows, width, eps, codes, dtype,
                                    weight_dtype, None)
    for bad in (dict(x=None), dict(weight=None), dict(out=None), dict(rows=-1), dict(rows=1 << 31), dict(width=0),
                dict(width=16385), dict(eps=-1.0), dict(codes=3), dict(codes=1), dict(dtype=1), dict(weight_dtype=2),
                dict(dtype=2, weight_dtype=3)):
        assert run(**bad) == -1, bad
    assert run(rows=0, x=None) == 0
    back = lib.sdk_add_rms_norm_backward
    assert back(ONE, None, ONE, ONE, ONE, ONE, ONE, None, 0, 4, 64, 0, 0, None) == -3
    assert back(ONE, None, ONE, ONE, ONE, None, None, None, 0, 4, 64, 0, 0, None) == -1
    assert back(None, None, ONE, ONE, ONE, ONE, None, None, 0, 4, 64, 0, 0, None) == -1
    assert lib.sdk_add_rms_norm_backward_workspace_bytes(4, 64) == 64 * 4
    assert lib.sdk_add_rms_norm_backward_workspace_bytes(4, 20000) == 0
    for bad in ((None, ONE, ONE, 4, 8, 1, 0), (ONE, ONE, ONE, 4, 0, 1, 0), (ONE, ONE, ONE, 4, 8, 0, 0),
                (ONE, ONE, ONE, 4, 8, 1, 1), (ONE, ONE, ONE, -1, 8, 1, 0)):
        assert lib.sdk_dequantize_rows(*bad, None) == -1


def test_adamw_refuses(lib):
    one, none = (ctypes.c_void_p * 1)(256), (ctypes.c_void_p * 1)()
    sizes = (ctypes.c_int64 * 1)(5)

    def run(p=one, g=one, m=one, v=one, n=sizes, count=1, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, step=1, dtype=0):
        return lib.sdk_adamw_step(p, g, m, v, n, count, lr, b1, b2, eps, wd, step, dtype, None)
    for bad in (dict(p=none), dict(g=none), dict(m=none), dict(v=none), dict(n=(ctypes.c_int64 * 1)(-1)), dict(count=-1),
                dict(p=None), dict(lr=-1.0), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(wd=-1.0), dict(step=0),
                dict(dtype=1), dict(lr=float("nan"))):
        assert run(**bad) == -1, bad
    assert run(count=0) == 0
    assert run(n=(ctypes.c_int64 * 1)(0), p=none) == 0   # an empty tensor has no memory
    assert lib.sdk_adamw_step_8bit(one, one, one, none, one, one, sizes, 1, 1e-3, 0.9, 0.99, 1e-8, 0.0, 1, 0, None) == -1
    assert lib.sdk_adamw_moment_values(None, ONE, ONE, 4, 0, 0, None) == -1
    assert lib.sdk_adamw_moment_values(ONE, ONE, ONE, -4, 0, 0, None) == -1
    assert lib.sdk_adamw_moment_values(None, None, None, 0, 0, 0, None) == 0


def test_cpu_tensors_are_refused():
    from spherical_distortion import functional as F
    q = torch.zeros(1, 1, 4, 8)
    x, w = torch.zeros(2, 8), torch.ones(8)
    calls = [lambda: F.bucket_attention(q, q, q, torch.zeros(1, 2), torch.zeros(4, 4, dtype=torch.uint8)),
             lambda: F.bucket_attention(q.requires_grad_(), q, q, torch.zeros(1, 2), torch.zeros(4, 4, dtype=torch.uint8)),
             lambda: F.add_rms_norm(x, None, w), lambda: F.add_rms_norm_quantized(x, None, w),
             lambda: F.dequantize_rows(torch.zeros(2, 8, dtype=torch.int8), torch.zeros(2)),
             lambda: F.adamw_step([x], [x], [x], [x], step=1),
             lambda: F.adamw_moment_values(torch.zeros(2, dtype=torch.int8), torch.zeros(1))]
    for call in calls:
        with pytest.raises((NotImplementedError, RuntimeError)):
            call()
    F.adamw_step([], [], [], [], step=1)   # nothing to step


def test_bucket_maps_on_the_cpu():
    from spherical_distortion import util
    lonlat = torch.tensor([[0.0, 0.0], [3.0, 0.1], [0.0, 1.5]])
    got = util.great_circle_bucket_map(lonlat, num_buckets=8)
    assert got.dtype == torch.uint8 and got.shape == (3, 3)
    assert not bool(got.diagonal().any()) and torch.equal(got, got.T) and int(got.max()) <= 7
    assert util.sequence_bucket_map(2, 5, 4, device="cpu").tolist()[1][-1] == 0
