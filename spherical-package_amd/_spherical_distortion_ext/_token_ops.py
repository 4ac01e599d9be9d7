"""PyTorch-ROCm custom operators on token sequences over the C ABI: attention with a learned bias
for each bucket of relative positions, a gated linear recurrence, residual addition with root-mean-square
and layer norm, AdamW, Muon.

Registered beside the mapped operators in ``torch.ops.sdk_mapped_ops``, for the CUDA (= HIP on
ROCm) dispatch key only.  The reference has none of them.  Where libsdk_torch_ops.so is built, its
implementations (csrc/torch_token_ops.cpp) serve the names it lists; PYTHON_IMPL keeps the functions
below.
"""
import ctypes

import torch

from . import _capi, _ops

_DTYPES = {torch.float32: _capi.SDK_F32, torch.bfloat16: _capi.SDK_BF16, torch.float16: _capi.SDK_F16}
CODES = {torch.int8: 1, torch.float8_e4m3fn: 2}
BLOCK = 256   # values of a moment in 8 bits that share a scale


def _dtype(name, t):
    if t.dtype not in _DTYPES:
        raise RuntimeError("unsupported dtype %s of %s (float32, bfloat16 and float16 only)" % (t.dtype, name))
    return _DTYPES[t.dtype]


def _on_gpu(ref, **tensors):
    if not ref.is_cuda:
        raise RuntimeError("this backend runs on the GPU only: tensors must be CUDA/HIP tensors")
    for name, t in tensors.items():
        if t is not None and (not t.is_cuda or t.device != ref.device):
            raise RuntimeError("%s must be a CUDA tensor on %s" % (name, ref.device))


def _dense(**tensors):
    for name, t in tensors.items():
        if t is not None and not t.is_contiguous():
            raise RuntimeError("%s must be contiguous" % name)


# --------------------------------------------------------------------------- attention
def _rows_fit(t):
    """Whether the kernels read `t` where it lies: last axis dense, rows 16-byte aligned, 64 tokens within 2^31 bytes."""
    each = 16 // t.element_size()
    return (t.data_ptr() % 16 == 0 and (t.shape[-1] == 1 or t.stride(-1) == 1)
            and all(t.stride(i) % each == 0 or t.shape[i] == 1 for i in range(3))
            and (t.shape[2] == 1 or t.stride(2) < 2 ** 31 // (64 * t.element_size())))


def _laid_out(t):
    """A dense copy, of a dense tensor too (which may lie at any address)."""
    return t.clone(memory_format=torch.contiguous_format)


def _rows_ready(t):
    return t if _rows_fit(t) else _laid_out(t)


def _strides(t):
    """Batch, head and token strides; those of axes of length one do not count."""
    return (ctypes.c_int64 * 3)(*(t.stride(i) if t.shape[i] != 1 else 0 for i in range(3)))


def _check_attention(query, key, value, bias_table, bucket_map, key_lengths, scale):
    _on_gpu(query, key=key, value=value, bias_table=bias_table, bucket_map=bucket_map, key_lengths=key_lengths)
    _dtype("query", query)
    if query.dim() != 4 or key.dim() != 4:
        raise RuntimeError("query and key must be [batch, heads, tokens, dim], got %s and %s"
                           % (tuple(query.shape), tuple(key.shape)))
    B, H, Lq, D = query.shape
    if key.shape != value.shape or key.shape[0] != B or key.shape[3] != D:
        raise RuntimeError("key %s and value %s must be [%d, key heads, keys, %d]"
                           % (tuple(key.shape), tuple(value.shape), B, D))
    Hk, Lk = key.shape[1:3]
    if Hk < 1 or H < 1 or H % Hk:
        raise RuntimeError("heads = %d must be a multiple of key heads = %d" % (H, Hk))
    if key.dtype != query.dtype or value.dtype != query.dtype:
        raise RuntimeError("key and value must have dtype %s (got %s and %s)"
                           % (query.dtype, key.dtype, value.dtype))
    if D < 8 or D > 128 or D % 8:
        raise RuntimeError("dim = %d must be a multiple of 8 up to 128" % D)
    if bias_table.dim() != 2 or bias_table.shape[0] != H or not 1 <= bias_table.shape[1] <= 256:
        raise RuntimeError("bias_table %s must be [%d, buckets], 1 to 256 buckets" % (tuple(bias_table.shape), H))
    if bias_table.dtype not in (query.dtype, torch.float32):
        raise RuntimeError("bias_table must have dtype %s or float32 (got %s)" % (query.dtype, bias_table.dtype))
    if bucket_map.dtype != torch.uint8:
        raise RuntimeError("bucket_map must have dtype uint8 (got %s)" % bucket_map.dtype)
    if tuple(bucket_map.shape) not in ((Lq, Lk), (B, Lq, Lk)):
        raise RuntimeError("bucket_map %s must be [%d, %d] or [%d, %d, %d]"
                           % (tuple(bucket_map.shape), Lq, Lk, B, Lq, Lk))
    if key_lengths is not None and (key_lengths.dtype != torch.int32 or tuple(key_lengths.shape) != (B,)):
        raise RuntimeError("key_lengths must be int32 of shape [%d], got %s %s"
                           % (B, key_lengths.dtype, tuple(key_lengths.shape)))
    _dense(key_lengths=key_lengths)
    if not 2.0 ** -32 <= scale <= 2.0 ** 32:
        raise RuntimeError("scale must be between 2^-32 and 2^32, got %s" % scale)


def _args(query, key, value, bias_table, bucket_map, key_lengths, causal, scale):
    """The argument block and the tensors whose memory it names (aligned copies among them)."""
    query, key, value = (_rows_ready(t) for t in (query, key, value))
    bias_table = bias_table.contiguous()
    if bucket_map.stride(-1) != 1 and bucket_map.shape[-1] != 1:
        bucket_map = bucket_map.contiguous()
    a = _capi.BucketAttention()
    a.query, a.key, a.value = query.data_ptr(), key.data_ptr(), value.data_ptr()
    a.bias_table, a.bucket_map = bias_table.data_ptr(), bucket_map.data_ptr()
    a.key_lengths = 0 if key_lengths is None else key_lengths.data_ptr()
    a.batch, a.heads, a.queries, a.dim = query.shape
    a.key_heads, a.keys = key.shape[1:3]
    a.buckets = bias_table.shape[1]
    a.query_strides, a.key_strides, a.value_strides = _strides(query), _strides(key), _strides(value)
    a.map_strides = (ctypes.c_int64 * 2)(bucket_map.stride(0) if bucket_map.dim() == 3 else 0, bucket_map.stride(-2))
    a.scale, a.causal = scale, int(causal)
    a.dtype, a.table_dtype = _DTYPES[query.dtype], _DTYPES[bias_table.dtype]
    return a, (query, key, value, bias_table, bucket_map)


def _run(name, a, backward, ref):
    need = _capi.load().sdk_bucket_attention_workspace_bytes(ctypes.byref(a), backward)
    ws = torch.empty(need, dtype=torch.uint8, device=ref.device) if need else None
    _capi.call(name, ctypes.byref(a), _ops._ptr(ws), need, _ops._stream(ref))


def bucket_attention_forward(query, key, value, bias_table, bucket_map, key_lengths, causal, scale):
    """-> (output like query, what rounding took from it (float32: an empty tensor), lse [2, batch, heads, queries]
    float32: two numbers whose sum is log2 of the row's sum of exponentials)."""
    _check_attention(query, key, value, bias_table, bucket_map, key_lengths, scale)
    with torch.cuda.device(query.device):
        a, keep = _args(query, key, value, bias_table, bucket_map, key_lengths, causal, scale)
        out = torch.empty_like(keep[0])
        lse = torch.empty((2,) + tuple(query.shape[:3]), dtype=torch.float32, device=query.device)
        rest = out.new_empty(0) if out.dtype == torch.float32 else torch.empty_like(out)
        a.output, a.output_strides, a.lse = out.data_ptr(), _strides(out), lse.data_ptr()
        a.output_rest = 0 if out.dtype == torch.float32 else rest.data_ptr()
        _run("sdk_bucket_attention_forward", a, 0, query)
    return out, rest, lse


def bucket_attention_backward(grad_output, query, key, value, bias_table, bucket_map, key_lengths, output, rest,
                              lse, causal, scale, need_query, need_keys, need_table):
    """-> gradients of query, key, value and bias_table; those not asked for are empty tensors."""
    _check_attention(query, key, value, bias_table, bucket_map, key_lengths, scale)
    _on_gpu(query, grad_output=grad_output, output=output, rest=rest, lse=lse)
    if grad_output.shape != query.shape or output.shape != query.shape or tuple(lse.shape) != (2,) + tuple(query.shape[:3]):
        raise RuntimeError("grad_output, output and lse must have the shapes of the forward's results")
    if grad_output.dtype != query.dtype or output.dtype != query.dtype or lse.dtype != torch.float32:
        raise RuntimeError("grad_output and output must have dtype %s, lse float32" % query.dtype)
    if rest.numel() and (rest.shape != output.shape or rest.dtype != output.dtype or rest.stride() != output.stride()):
        raise RuntimeError("the output's rest must be like the output, or empty")
    with torch.cuda.device(query.device):
        a, keep = _args(query, key, value, bias_table, bucket_map, key_lengths, causal, scale)
        grad_output, lse = _rows_ready(grad_output), lse.contiguous()
        if not _rows_fit(output) or (rest.numel() and not _rows_fit(rest)):   # both are read by the output's strides
            output, rest = _laid_out(output), _laid_out(rest)
        if rest.numel():
            a.output_rest = rest.data_ptr()
        a.grad_output, a.grad_output_strides = grad_output.data_ptr(), _strides(grad_output)
        a.output, a.output_strides, a.lse = output.data_ptr(), _strides(output), lse.data_ptr()
        dq, dk, dv = (torch.empty_like(t) if need else t.new_empty(0)
                      for t, need in zip(keep, (need_query, need_keys, need_keys)))
        dt = torch.empty_like(keep[3]) if need_table else bias_table.new_empty(0)
        if need_query:
            a.grad_query, a.grad_query_strides = dq.data_ptr(), _strides(dq)
        if need_keys:
            a.grad_key, a.grad_key_strides = dk.data_ptr(), _strides(dk)
            a.grad_value, a.grad_value_strides = dv.data_ptr(), _strides(dv)
        if need_table:
            a.grad_table = dt.data_ptr()
        _run("sdk_bucket_attention_backward", a, 1, query)
    return dq, dk, dv, dt


# --------------------------------------------------------------------------- norm
def _check_norm(x, residual, weight):
    _on_gpu(x, residual=residual, weight=weight)
    _dense(x=x, residual=residual, weight=weight)
    _dtype("x", x)
    if x.dim() < 1 or weight.dim() != 1 or weight.shape[0] != x.shape[-1]:
        raise RuntimeError("weight %s must have one value for each of the last axis of x %s"
                           % (tuple(weight.shape), tuple(x.shape)))
    if not 1 <= x.shape[-1] <= 16384:
        raise RuntimeError("width = %d must be between 1 and 16384" % x.shape[-1])
    if weight.dtype not in (x.dtype, torch.float32):
        raise RuntimeError("weight must have dtype %s or float32 (got %s)" % (x.dtype, weight.dtype))
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise RuntimeError("residual must be like x: %s %s, got %s %s"
                           % (tuple(x.shape), x.dtype, tuple(residual.shape), residual.dtype))


def _norm(x, residual, weight, out, scales, summed, inverse, eps, codes):
    width = x.shape[-1]
    with torch.cuda.device(x.device):
        _capi.call("sdk_add_rms_norm", *(_ops._ptr(t) for t in (x, residual, weight, out, scales, summed, inverse)),
                   x.numel() // width, width, float(eps), codes, _DTYPES[x.dtype], _DTYPES[weight.dtype],
                   _ops._stream(x))


def add_rms_norm(x, residual, weight, eps):
    """-> (norm, x + residual, reciprocal root mean square of each row); without a residual the second is
    an empty tensor."""
    _check_norm(x, residual, weight)
    out = torch.empty_like(x)
    summed = x.new_empty(0) if residual is None else torch.empty_like(x)
    inverse = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _norm(x, residual, weight, out, None, None if residual is None else summed, inverse, eps, 0)
    return out, summed, inverse


def add_rms_norm_quantized(x, residual, weight, eps, fp8):
    """-> (codes: int8, or float8_e4m3fn with fp8, scale of each row, x + residual or an empty tensor)."""
    _check_norm(x, residual, weight)
    codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn if fp8 else torch.int8, device=x.device)
    summed = x.new_empty(0) if residual is None else torch.empty_like(x)
    scales = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    _norm(x, residual, weight, codes, scales, None if residual is None else summed, None, eps, 2 if fp8 else 1)
    return codes, scales, summed


def add_rms_norm_backward(grad, grad_sum, summed, weight, inverse, need_x, need_weight):
    """-> (gradient of x and of residual, gradient of weight); those not asked for are empty tensors."""
    _check_norm(summed, None, weight)
    _on_gpu(summed, grad=grad, grad_sum=grad_sum, inverse=inverse)
    for name, t in (("grad", grad), ("grad_sum", grad_sum)):
        if t is not None and (t.shape != summed.shape or t.dtype != summed.dtype):
            raise RuntimeError("%s must be like the sums: %s %s, got %s %s"
                               % (name, tuple(summed.shape), summed.dtype, tuple(t.shape), t.dtype))
    _dense(grad=grad, grad_sum=grad_sum, inverse=inverse)
    width = summed.shape[-1]
    rows = summed.numel() // width
    if inverse.dtype != torch.float32 or inverse.numel() != rows:
        raise RuntimeError("inverse must be float32 with one value for each row")
    dx = torch.empty_like(summed) if need_x else summed.new_empty(0)
    dw = torch.empty_like(weight) if need_weight else weight.new_empty(0)
    if not need_x and not need_weight:
        return dx, dw
    with torch.cuda.device(summed.device):
        need = _capi.load().sdk_add_rms_norm_backward_workspace_bytes(rows, width) if need_weight else 0
        ws = torch.empty(need, dtype=torch.uint8, device=summed.device) if need else None
        _capi.call("sdk_add_rms_norm_backward", *(_ops._ptr(t) for t in (grad, grad_sum, summed, weight, inverse)),
                   _ops._ptr(dx if need_x else None), _ops._ptr(dw if need_weight else None), _ops._ptr(ws), need,
                   rows, width, _DTYPES[summed.dtype], _DTYPES[weight.dtype], _ops._stream(summed))
    return dx, dw


def dequantize_rows(codes, scales, dtype):
    """-> codes * scale of the row, in `dtype`."""
    _on_gpu(codes, scales=scales)
    _dense(codes=codes, scales=scales)
    if codes.dtype not in CODES:
        raise RuntimeError("codes must be int8 or float8_e4m3fn (got %s)" % codes.dtype)
    if dtype not in _DTYPES:
        raise RuntimeError("unsupported dtype %s (float32, bfloat16 and float16 only)" % dtype)
    if codes.dim() < 1 or codes.shape[-1] < 1 or scales.dtype != torch.float32 or scales.shape != codes.shape[:-1]:
        raise RuntimeError("scales must be float32 of shape %s, got %s %s"
                           % (tuple(codes.shape[:-1]), scales.dtype, tuple(scales.shape)))
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    width = codes.shape[-1]
    with torch.cuda.device(codes.device):
        _capi.call("sdk_dequantize_rows", _ops._ptr(codes), _ops._ptr(scales), _ops._ptr(out),
                   codes.numel() // width, width, CODES[codes.dtype], _DTYPES[dtype], _ops._stream(codes))
    return out


# --------------------------------------------------------------------------- AdamW
def _pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*(t.data_ptr() for t in tensors))


def _check_lists(params, lists):
    """lists: name -> (tensors, dtype or None for the parameter's, values of a scale or None)."""
    if not params:
        return
    ref = params[0]
    if not ref.is_cuda:
        raise RuntimeError("this backend runs on the GPU only: tensors must be CUDA/HIP tensors")
    _dtype("params", ref)
    for name, (tensors, dtype, each) in lists.items():
        if len(tensors) != len(params):
            raise RuntimeError("%d %s for %d params" % (len(tensors), name, len(params)))
        for i, (p, t) in enumerate(zip(params, tensors)):
            want = dtype or ref.dtype
            if t.dtype != want or t.device != ref.device:
                raise RuntimeError("%s[%d] must have dtype %s on %s (got %s on %s)"
                                   % (name, i, want, ref.device, t.dtype, t.device))
            shape = p.shape if each is None else (-(-p.numel() // each),)
            if tuple(t.shape) != tuple(shape):
                raise RuntimeError("%s[%d] must have shape %s (got %s)" % (name, i, tuple(shape), tuple(t.shape)))
            if not t.is_contiguous():
                raise RuntimeError("%s[%d] must be contiguous" % (name, i))


def _step(name, params, lists, lr, beta1, beta2, eps, weight_decay, step):
    sizes = (ctypes.c_int64 * len(params))(*(p.numel() for p in params))
    with torch.cuda.device(params[0].device):
        _capi.call(name, _pointers(params), *(_pointers(t) for t in lists), sizes, len(params), lr, beta1, beta2,
                   eps, weight_decay, step, _DTYPES[params[0].dtype], _ops._stream(params[0]))
    # the kernels write through pointers: autograd has to learn of it to refuse a backward through the former values
    for t in (t for tensors in (params, *lists[1:]) for t in tensors):
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, lr, beta1, beta2, eps, weight_decay, step):
    _check_lists(params, {"params": (params, None, None), "grads": (grads, None, None),
                          "exp_avgs": (exp_avgs, torch.float32, None),
                          "exp_avg_sqs": (exp_avg_sqs, torch.float32, None)})
    if params:
        _step("sdk_adamw_step", params, (grads, exp_avgs, exp_avg_sqs), lr, beta1, beta2, eps, weight_decay, step)


def adamw_step_8bit(params, grads, avg_codes, avg_scales, sq_codes, sq_scales, lr, beta1, beta2, eps, weight_decay,
                    step):
    _check_lists(params, {"params": (params, None, None), "grads": (grads, None, None),
                          "avg_codes": (avg_codes, torch.int8, None), "avg_scales": (avg_scales, torch.float32, BLOCK),
                          "sq_codes": (sq_codes, torch.uint8, None), "sq_scales": (sq_scales, torch.float32, BLOCK)})
    if params:
        _step("sdk_adamw_step_8bit", params, (grads, avg_codes, avg_scales, sq_codes, sq_scales), lr, beta1, beta2,
              eps, weight_decay, step)


def adamw_moment_values(codes, scales, dtype):
    """-> the values that the codes of a first (int8) or second (uint8) moment stand for."""
    _on_gpu(codes, scales=scales)
    _dense(codes=codes, scales=scales)
    if codes.dtype not in (torch.int8, torch.uint8):
        raise RuntimeError("codes must be int8 (first moment) or uint8 (second), got %s" % codes.dtype)
    if dtype not in _DTYPES:
        raise RuntimeError("unsupported dtype %s (float32, bfloat16 and float16 only)" % dtype)
    if scales.dtype != torch.float32 or tuple(scales.shape) != (-(-codes.numel() // BLOCK),):
        raise RuntimeError("scales must be float32 of shape [%d], got %s %s"
                           % (-(-codes.numel() // BLOCK), scales.dtype, tuple(scales.shape)))
    out = torch.empty(codes.shape, dtype=dtype, device=codes.device)
    with torch.cuda.device(codes.device):
        _capi.call("sdk_adamw_moment_values", _ops._ptr(codes), _ops._ptr(scales), _ops._ptr(out), codes.numel(),
                   int(codes.dtype == torch.uint8), _DTYPES[dtype], _ops._stream(codes))
    return out


# --------------------------------------------------------------------------- layer norm
def _check_layer_norm(x, residual, weight, bias):
    _check_norm(x, residual, weight)
    _on_gpu(x, bias=bias)
    _dense(bias=bias)
    if bias is not None and (bias.shape != weight.shape or bias.dtype != weight.dtype):
        raise RuntimeError("bias must be like weight: %s %s, got %s %s"
                           % (tuple(weight.shape), weight.dtype, tuple(bias.shape), bias.dtype))


def add_layer_norm(x, residual, weight, bias, eps):
    """-> (norm, x + residual, mean and reciprocal standard deviation of each row); without a residual the second
    is an empty tensor."""
    _check_layer_norm(x, residual, weight, bias)
    out = torch.empty_like(x)
    summed = x.new_empty(0) if residual is None else torch.empty_like(x)
    mean, inverse = (torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) for _ in range(2))
    width = x.shape[-1]
    with torch.cuda.device(x.device):
        _capi.call("sdk_add_layer_norm", *(_ops._ptr(t) for t in (x, residual, weight, bias, out, None if residual is None
                                                                  else summed, mean, inverse)),
                   x.numel() // width, width, float(eps), _DTYPES[x.dtype], _DTYPES[weight.dtype], _ops._stream(x))
    return out, summed, mean, inverse


def add_layer_norm_backward(grad, grad_sum, x, residual, weight, mean, inverse, need_x, need_weight, need_bias):
    """-> (gradient of x and of residual, of weight, of bias); those not asked for are empty tensors.  x and residual as
    the forward got them, or its sum alone (one read less; 16-bit gradients are then off by the sum's rounding)."""
    _check_norm(x, residual, weight)
    _on_gpu(x, grad=grad, grad_sum=grad_sum, mean=mean, inverse=inverse)
    for name, t in (("grad", grad), ("grad_sum", grad_sum)):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise RuntimeError("%s must be like x: %s %s, got %s %s"
                               % (name, tuple(x.shape), x.dtype, tuple(t.shape), t.dtype))
    _dense(grad=grad, grad_sum=grad_sum, mean=mean, inverse=inverse)
    width = x.shape[-1]
    rows = x.numel() // width
    for t in (mean, inverse):
        if t.dtype != torch.float32 or t.numel() != rows:
            raise RuntimeError("mean and inverse must be float32 with one value for each row")
    dx = torch.empty_like(x) if need_x else x.new_empty(0)
    dw, db = (torch.empty_like(weight) if need else weight.new_empty(0) for need in (need_weight, need_bias))
    if not need_x and not need_weight and not need_bias:
        return dx, dw, db
    with torch.cuda.device(x.device):
        need = 0
        if need_weight or need_bias:
            need = _capi.load().sdk_add_layer_norm_backward_workspace_bytes(rows, width)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
        _capi.call("sdk_add_layer_norm_backward",
                   *(_ops._ptr(t) for t in (grad, grad_sum, x, residual, weight, mean, inverse, dx if need_x else None,
                                            dw if need_weight else None, db if need_bias else None, ws)), need,
                   rows, width, _DTYPES[x.dtype], _DTYPES[weight.dtype], _ops._stream(x))
    return dx, dw, db


# --------------------------------------------------------------------------- gated scan
def _check_scan(x, gate, state, lengths):
    _on_gpu(x, gate=gate, state=state, lengths=lengths)
    _dtype("x", x)
    if x.dim() != 3:
        raise RuntimeError("x must be [batch, tokens, width], got %s" % (tuple(x.shape),))
    if gate.shape != x.shape or gate.dtype != x.dtype:
        raise RuntimeError("gate must be like x: %s %s, got %s %s"
                           % (tuple(x.shape), x.dtype, tuple(gate.shape), gate.dtype))
    B, _, D = x.shape
    if state is not None and (tuple(state.shape) != (B, D) or state.dtype != torch.float32):
        raise RuntimeError("state must be float32 of shape [%d, %d], got %s %s"
                           % (B, D, state.dtype, tuple(state.shape)))
    if lengths is not None and (lengths.dtype != torch.int32 or tuple(lengths.shape) != (B,)):
        raise RuntimeError("lengths must be int32 of shape [%d], got %s %s" % (B, lengths.dtype, tuple(lengths.shape)))
    _dense(lengths=lengths)


def _tokens_ready(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else _laid_out(t)


def _token_strides(t):
    """Batch and token strides; those of axes of length one do not count."""
    return (ctypes.c_int64 * 2)(*(t.stride(i) if t.shape[i] != 1 else 0 for i in range(2)))


def _scan_args(x, gate, state, lengths, reverse):
    """The argument block and the tensors whose memory it names."""
    x, gate = _tokens_ready(x), _tokens_ready(gate)
    state = None if state is None else state.contiguous()
    a = _capi.GatedScan()
    a.x, a.gate, a.state = x.data_ptr(), gate.data_ptr(), 0 if state is None else state.data_ptr()
    a.lengths = 0 if lengths is None else lengths.data_ptr()
    a.batch, a.tokens, a.width = x.shape
    a.x_strides, a.gate_strides = _token_strides(x), _token_strides(gate)
    a.reverse, a.dtype = int(reverse), _DTYPES[x.dtype]
    return a, (x, gate, state, lengths)


def _run_scan(name, a, backward, ref):
    need = _capi.load().sdk_gated_scan_workspace_bytes(ctypes.byref(a), backward)
    ws = torch.empty(need, dtype=torch.uint8, device=ref.device) if need else None
    _capi.call(name, ctypes.byref(a), _ops._ptr(ws), need, _ops._stream(ref))


def gated_scan_forward(x, gate, state, lengths, reverse):
    """-> (output [batch, tokens, width], the last state [batch, width] float32)."""
    _check_scan(x, gate, state, lengths)
    with torch.cuda.device(x.device):
        a, keep = _scan_args(x, gate, state, lengths, reverse)
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        last = torch.empty((x.shape[0], x.shape[2]), dtype=torch.float32, device=x.device)
        a.output, a.last = out.data_ptr(), last.data_ptr()
        _run_scan("sdk_gated_scan_forward", a, 0, x)
    return out, last


def gated_scan_backward(grad_output, grad_last, x, gate, state, lengths, output, reverse, need_x, need_gate,
                        need_state):
    """-> gradients of x, gate and state; those not asked for are empty tensors."""
    _check_scan(x, gate, state, lengths)
    _on_gpu(x, grad_output=grad_output, grad_last=grad_last, output=output)
    B, _, D = x.shape
    for name, t in (("grad_output", grad_output), ("output", output)):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise RuntimeError("%s must be like x: %s %s, got %s %s"
                               % (name, tuple(x.shape), x.dtype, tuple(t.shape), t.dtype))
    if grad_last is not None and (tuple(grad_last.shape) != (B, D) or grad_last.dtype != torch.float32):
        raise RuntimeError("grad_last must be float32 of shape [%d, %d]" % (B, D))
    dx, dgate = (torch.empty(x.shape if need else (0,), dtype=x.dtype, device=x.device) for need in (need_x, need_gate))
    dstate = torch.empty((B, D) if need_state else (0,), dtype=torch.float32, device=x.device)
    if not need_x and not need_gate and not need_state:
        return dx, dgate, dstate
    with torch.cuda.device(x.device):
        a, keep = _scan_args(x, gate, state, lengths, reverse)
        output = output.contiguous()
        a.output = output.data_ptr()
        if grad_output is not None:
            grad_output = _tokens_ready(grad_output)
            a.grad_output, a.grad_output_strides = grad_output.data_ptr(), _token_strides(grad_output)
        if grad_last is not None:
            grad_last = grad_last.contiguous()
            a.grad_last = grad_last.data_ptr()
        for name, t, need in (("grad_x", dx, need_x), ("grad_gate", dgate, need_gate), ("grad_state", dstate, need_state)):
            if need:
                setattr(a, name, t.data_ptr())
        _run_scan("sdk_gated_scan_backward", a, 1, x)
    return dx, dgate, dstate


def gated_scan_step(x, gate, state):
    """One token of each sequence; state [batch, width] is updated in place. -> output like x, dense."""
    _on_gpu(x, gate=gate, state=state)
    _dtype("x", x)
    if x.dim() != 2 or gate.shape != x.shape or gate.dtype != x.dtype:
        raise RuntimeError("x and gate must be [batch, width] of one type, got %s %s and %s %s"
                           % (tuple(x.shape), x.dtype, tuple(gate.shape), gate.dtype))
    B, D = x.shape
    if state.shape != x.shape or state.dtype != torch.float32:
        raise RuntimeError("state must be float32 of shape [%d, %d], got %s %s"
                           % (B, D, state.dtype, tuple(state.shape)))
    if (D > 1 and state.stride(1) != 1) or (B > 1 and state.stride(0) < D):
        raise RuntimeError("state must have dense rows that do not overlap (it is changed in place), got strides %s"
                           % (state.stride(),))
    x, gate = _tokens_ready(x), _tokens_ready(gate)
    out = torch.empty((B, D), dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):
        _capi.call("sdk_gated_scan_step", _ops._ptr(x), x.stride(0), _ops._ptr(gate), gate.stride(0), _ops._ptr(state),
                   state.stride(0), _ops._ptr(out), B, D, _DTYPES[x.dtype], _ops._stream(x))
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)
    return out


# --------------------------------------------------------------------------- matrices made orthogonal, Muon
def _coefficients(values):
    if len(values) != 3:
        raise RuntimeError("coefficients must be three numbers, got %d" % len(values))
    return (ctypes.c_double * 3)(*values)


def check_newton_schulz(steps, coefficients, eps):
    """Raises where orthogonalize and muon_step would refuse these settings; touches no device."""
    _capi.call("sdk_orthogonalize", None, None, 0, 0, 0, steps, _coefficients(coefficients), eps, None, 0,
               _DTYPES[torch.float32], None)


def orthogonalize(x, steps, coefficients, eps):
    """-> a dense tensor like x [.., rows, columns]."""
    _on_gpu(x)
    dtype = _dtype("x", x)
    if x.dim() < 2:
        raise RuntimeError("x must be [.., rows, columns], got %s" % (tuple(x.shape),))
    c = _coefficients(coefficients)
    x = x.contiguous()
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    rows, columns = x.shape[-2:]
    count = x.numel() // (rows * columns) if x.numel() else 0
    with torch.cuda.device(x.device):
        need = _capi.load().sdk_orthogonalize_workspace_bytes(rows, columns, count, dtype)
        ws = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
        _capi.call("sdk_orthogonalize", _ops._ptr(x), _ops._ptr(out), rows, columns, count, steps, c, eps,
                   _ops._ptr(ws), need, dtype, _ops._stream(x))
    return out


def muon_step(params, grads, momenta, lr, momentum, nesterov, weight_decay, steps, coefficients, eps):
    _check_lists(params, {"params": (params, None, None), "grads": (grads, None, None),
                          "momenta": (momenta, torch.float32, None)})
    if not params:
        if len(grads) or len(momenta):
            raise RuntimeError("gradients or momenta without params")
        return
    for i, p in enumerate(params):
        if p.dim() < 2:
            raise RuntimeError("params[%d] must have two axes at least, got %s" % (i, tuple(p.shape)))
    c, n = _coefficients(coefficients), len(params)
    rows = (ctypes.c_int64 * n)(*(p.shape[0] for p in params))
    columns = (ctypes.c_int64 * n)(*(p.numel() // p.shape[0] if p.shape[0] else 0 for p in params))
    dtype = _DTYPES[params[0].dtype]
    with torch.cuda.device(params[0].device):
        need = _capi.load().sdk_muon_step_workspace_bytes(rows, columns, n, dtype)
        ws = torch.empty(need, dtype=torch.uint8, device=params[0].device) if need else None
        _capi.call("sdk_muon_step", _pointers(params), _pointers(grads), _pointers(momenta), rows, columns, n, lr,
                   momentum, int(nesterov), weight_decay, steps, c, eps, _ops._ptr(ws), need, dtype,
                   _ops._stream(params[0]))
    for t in (*params, *momenta):
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


# --------------------------------------------------------------------------- forms with gradients
# Registered with autograd by the compiled layer alone; without it functional/token_ops.py's autograd functions serve.
def bucket_attention(query, key, value, bias_table, bucket_map, key_lengths, causal, scale):
    return bucket_attention_forward(query, key, value, bias_table, bucket_map, key_lengths, causal, scale)[0]


def rms_norm_pair(x, residual, weight, eps):
    """-> [norm, x + residual], or [norm] without a residual."""
    return list(add_rms_norm(x, residual, weight, eps)[:1 if residual is None else 2])


def layer_norm_pair(x, residual, weight, bias, eps):
    """-> [norm, x + residual], or [norm] without a residual."""
    return list(add_layer_norm(x, residual, weight, bias, eps)[:1 if residual is None else 2])


def gated_scan(x, gate, state, lengths, reverse):
    """-> [output, last state]."""
    return list(gated_scan_forward(x, gate, state, lengths, reverse))


# --------------------------------------------------------------------------- registration
_SETTINGS = " float lr, float beta1, float beta2, float eps, float weight_decay, int step) -> ()"
_SCHEMAS = (
    ("bucket_attention",
     "(Tensor query, Tensor key, Tensor value, Tensor bias_table, Tensor bucket_map, Tensor? key_lengths,"
     " bool causal, float scale) -> Tensor", bucket_attention),
    ("rms_norm_pair", "(Tensor x, Tensor? residual, Tensor weight, float eps) -> Tensor[]", rms_norm_pair),
    ("bucket_attention_forward",
     "(Tensor query, Tensor key, Tensor value, Tensor bias_table, Tensor bucket_map, Tensor? key_lengths,"
     " bool causal, float scale) -> (Tensor, Tensor, Tensor)", bucket_attention_forward),
    ("bucket_attention_backward",
     "(Tensor grad_output, Tensor query, Tensor key, Tensor value, Tensor bias_table, Tensor bucket_map,"
     " Tensor? key_lengths, Tensor output, Tensor rest, Tensor lse, bool causal, float scale, bool need_query, bool need_keys,"
     " bool need_table) -> (Tensor, Tensor, Tensor, Tensor)", bucket_attention_backward),
    ("add_rms_norm", "(Tensor x, Tensor? residual, Tensor weight, float eps) -> (Tensor, Tensor, Tensor)",
     add_rms_norm),
    ("add_rms_norm_quantized",
     "(Tensor x, Tensor? residual, Tensor weight, float eps, bool fp8) -> (Tensor, Tensor, Tensor)",
     add_rms_norm_quantized),
    ("add_rms_norm_backward",
     "(Tensor grad, Tensor? grad_sum, Tensor summed, Tensor weight, Tensor inverse, bool need_x, bool need_weight)"
     " -> (Tensor, Tensor)", add_rms_norm_backward),
    ("dequantize_rows", "(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor", dequantize_rows),
    ("adamw_step",
     "(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avgs, Tensor(c!)[] exp_avg_sqs," + _SETTINGS,
     adamw_step),
    ("adamw_step_8bit",
     "(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] avg_codes, Tensor(c!)[] avg_scales,"
     " Tensor(d!)[] sq_codes, Tensor(e!)[] sq_scales," + _SETTINGS, adamw_step_8bit),
    ("adamw_moment_values", "(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor", adamw_moment_values),
    ("layer_norm_pair", "(Tensor x, Tensor? residual, Tensor weight, Tensor? bias, float eps) -> Tensor[]",
     layer_norm_pair),
    ("add_layer_norm",
     "(Tensor x, Tensor? residual, Tensor weight, Tensor? bias, float eps) -> (Tensor, Tensor, Tensor, Tensor)",
     add_layer_norm),
    ("add_layer_norm_backward",
     "(Tensor grad, Tensor? grad_sum, Tensor x, Tensor? residual, Tensor weight, Tensor mean, Tensor inverse,"
     " bool need_x, bool need_weight, bool need_bias) -> (Tensor, Tensor, Tensor)", add_layer_norm_backward),
    ("gated_scan", "(Tensor x, Tensor gate, Tensor? state, Tensor? lengths, bool reverse) -> Tensor[]", gated_scan),
    ("gated_scan_forward", "(Tensor x, Tensor gate, Tensor? state, Tensor? lengths, bool reverse) -> (Tensor, Tensor)",
     gated_scan_forward),
    ("gated_scan_backward",
     "(Tensor? grad_output, Tensor? grad_last, Tensor x, Tensor gate, Tensor? state, Tensor? lengths, Tensor output,"
     " bool reverse, bool need_x, bool need_gate, bool need_state) -> (Tensor, Tensor, Tensor)", gated_scan_backward),
    ("gated_scan_step", "(Tensor x, Tensor gate, Tensor(a!) state) -> Tensor", gated_scan_step),
    ("orthogonalize", "(Tensor x, int steps, float[] coefficients, float eps) -> Tensor", orthogonalize),
    ("muon_step",
     "(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] momenta, float lr, float momentum, bool nesterov,"
     " float weight_decay, int steps, float[] coefficients, float eps) -> ()", muon_step),
)


def _native_names():
    if _ops._native is None:
        return frozenset()
    _ops._native.sdk_torch_token_ops.restype = ctypes.c_char_p
    return frozenset(_ops._native.sdk_torch_token_ops().decode().split(","))


NATIVE_OPS = _native_names()
_library = torch.library.Library(_ops._NS, "FRAGMENT")
for _name, _schema, _fn in _SCHEMAS:
    _library.define(_name + _schema)
    if _name not in NATIVE_OPS:
        _library.impl(_name, _fn, "CUDA")
ops = _ops.ops
PYTHON_IMPL = {_name: _fn for _name, _schema, _fn in _SCHEMAS}
