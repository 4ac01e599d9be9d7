"""Functional entry points of the operators on token sequences.

Spherical samples as tokens (the pixels of a coarse grid, the vertices of an icosphere, the patches of
tangent images): attention whose learned bias goes by the bucket of a pair's relative position, a gated
recurrence along the tokens, the norms of a block with its residual, and the optimizers' steps.  The reference has none of them.
float32, bfloat16 and float16; sums, softmax statistics and norms are float32.
"""
import functools
import math

import torch
from torch.autograd import forward_ad

from _spherical_distortion_ext import _token_ops
from _spherical_distortion_ext._ops import ops as _sdk_ops


class _NoSecondDerivative(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *grads):
        return tuple(g if g is None else g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("second derivatives of this operator are not implemented")


def _only_first(backward):
    """A backward whose gradients, where it is itself recorded (create_graph), ask for a gradient and raise when it is
    formed.  Plain tensors would be constants to whatever is differentiated beside them."""
    @functools.wraps(backward)
    def run(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled():
            return out
        return _NoSecondDerivative.apply(*(g if g is None else g.detach().requires_grad_() for g in out))
    return run


def _wants_gradient(*tensors):
    """Whether autograd is to see the call (of the Python functions; the compiled layer finds out by itself)."""
    tensors = [t for t in tensors if t is not None]
    if any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("forward-mode derivatives of this operator are not implemented")
    return torch.is_grad_enabled() and any(t.requires_grad for t in tensors)


class BucketAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, query, key, value, bias_table, bucket_map, key_lengths, causal, scale):
        out, rest, lse = _sdk_ops.bucket_attention_forward(query, key, value, bias_table, bucket_map, key_lengths,
                                                           causal, scale)
        ctx.save_for_backward(query, key, value, bias_table, bucket_map, key_lengths, out, rest, lse)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @_only_first
    def backward(ctx, grad_output):
        query, key, value, bias_table, bucket_map, key_lengths, out, rest, lse = ctx.saved_tensors
        need_q, need_k, need_v, need_t = ctx.needs_input_grad[:4]
        dq, dk, dv, dt = _sdk_ops.bucket_attention_backward(
            grad_output, query, key, value, bias_table, bucket_map, key_lengths, out, rest, lse, ctx.causal, ctx.scale,
            need_q, need_k or need_v, need_t)
        return (dq if need_q else None, dk if need_k else None, dv if need_v else None, dt if need_t else None,
                None, None, None, None)


def bucket_attention(query, key, value, bias_table, bucket_map, key_lengths=None, causal=False, scale=None):
    """softmax(scale query key^T + bias_table[:, bucket_map]) value, head by head.

    query [B, heads, queries, dim]; key and value [B, key heads, keys, dim], heads a multiple of key
    heads; any strides whose last axis is dense (rows that are not 16-byte aligned are copied first).
    dim: a multiple of 8 up to 128.  bias_table [heads, buckets], of the queries' type or float32, 1 to
    256 buckets.  bucket_map: uint8 [queries, keys], or [B, queries, keys] where each sequence has its
    own.  A pair whose bucket is not below `buckets` does not count; nor do keys from key_lengths[b] on
    (int32 [B]; keys and values there are not read), nor, with `causal`, key j of query i where
    j > i + key_lengths[b] - queries: the last query sees every key.  A query without pairs gives
    zeros.  A bias of -inf leaves its bucket out; finite biases beyond 7e5 in magnitude count as one value: a
    mask by the type's lowest weighs nothing beside others, and the same among themselves.  scale: dim ** -0.5
    if None.

    With gradients for query, key, value and bias_table; second derivatives and forward mode raise.  A few
    queries against many keys (one new token and its cache) are dealt to the GPU along the keys."""
    scale = 1.0 / math.sqrt(query.shape[-1]) if scale is None else float(scale)
    if "bucket_attention" in _token_ops.NATIVE_OPS:
        return _sdk_ops.bucket_attention(query, key, value, bias_table, bucket_map, key_lengths, bool(causal), scale)
    if _wants_gradient(query, key, value, bias_table):
        return BucketAttentionFunction.apply(query, key, value, bias_table, bucket_map, key_lengths, bool(causal),
                                             scale)
    return _sdk_ops.bucket_attention_forward(query, key, value, bias_table, bucket_map, key_lengths, bool(causal),
                                             scale)[0]


class AddRMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        out, summed, inverse = _sdk_ops.add_rms_norm(x, residual, weight, eps)
        ctx.save_for_backward(x if residual is None else summed, weight, inverse)
        ctx.alone = residual is None
        ctx.set_materialize_grads(False)
        return (out, x.view_as(x)) if ctx.alone else (out, summed)

    @staticmethod
    @_only_first
    def backward(ctx, grad, grad_sum):
        summed, weight, inverse = ctx.saved_tensors
        need_x, need_r, need_w, _ = ctx.needs_input_grad
        if grad is None:   # only the sum was used
            return (grad_sum if need_x else None, grad_sum if need_r else None,
                    torch.zeros_like(weight) if need_w else None, None)
        dx, dw = _sdk_ops.add_rms_norm_backward(grad.contiguous(), None if grad_sum is None else grad_sum.contiguous(),
                                                summed, weight, inverse, need_x or need_r, need_w)
        return dx if need_x else None, dx if need_r else None, dw if need_w else None, None


def add_rms_norm(input, residual, weight, eps=1e-6):
    """(weight * h / sqrt(mean(h ** 2) + eps), h) with h = input + residual, over the last axis; a
    residual of None adds nothing.  weight: one value for each of the last axis (up to 16384), of the
    input's type or float32.  The sum is normalised before it is rounded to the input's type.  Second
    derivatives and forward mode raise."""
    if "rms_norm_pair" in _token_ops.NATIVE_OPS:
        both = _sdk_ops.rms_norm_pair(input, residual, weight, float(eps))
        return (both[0], input) if residual is None else (both[0], both[1])
    if _wants_gradient(input, residual, weight):
        return AddRMSNormFunction.apply(input, residual, weight, float(eps))
    out, summed, _ = _sdk_ops.add_rms_norm(input, residual, weight, float(eps))
    return out, input if residual is None else summed


def add_rms_norm_quantized(input, residual, weight, eps=1e-6, dtype=torch.int8):
    """(codes, scales, input + residual): the rows of add_rms_norm in 8 bits, codes * scales[..., None].
    dtype: torch.int8 (scale = largest magnitude / 127) or torch.float8_e4m3fn (/ 448).  Rows whose
    largest magnitude is below 2 ** -100 have scale 0; a row with a NaN has scale NaN.  No gradients."""
    if dtype not in _token_ops.CODES:
        raise RuntimeError("dtype must be torch.int8 or torch.float8_e4m3fn, got %s" % dtype)
    with torch.no_grad():
        codes, scales, summed = _sdk_ops.add_rms_norm_quantized(input, residual, weight, float(eps),
                                                                dtype == torch.float8_e4m3fn)
    return codes, scales, input if residual is None else summed


def dequantize_rows(codes, scales, dtype=torch.float32):
    """codes * scales[..., None] in `dtype`; codes int8 or float8_e4m3fn, one scale a row."""
    return _sdk_ops.dequantize_rows(codes, scales, dtype)


class AddLayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        out, summed, mean, inverse = _sdk_ops.add_layer_norm(x, residual, weight, bias, eps)
        # 16-bit sums would bring their rounding into the gradients
        rows = (summed, None) if residual is not None and x.dtype == torch.float32 else (x, residual)
        ctx.save_for_backward(*rows, weight, mean, inverse)
        ctx.alone = residual is None
        ctx.set_materialize_grads(False)
        return (out, x.view_as(x)) if ctx.alone else (out, summed)

    @staticmethod
    @_only_first
    def backward(ctx, grad, grad_sum):
        x, residual, weight, mean, inverse = ctx.saved_tensors
        need_x, need_r, need_w, need_b, _ = ctx.needs_input_grad
        if grad is None:   # only the sum was used
            return (grad_sum if need_x else None, grad_sum if need_r else None,
                    torch.zeros_like(weight) if need_w else None, torch.zeros_like(weight) if need_b else None, None)
        dx, dw, db = _sdk_ops.add_layer_norm_backward(
            grad.contiguous(), None if grad_sum is None else grad_sum.contiguous(), x, residual, weight, mean, inverse,
            need_x or need_r, need_w, need_b)
        return (dx if need_x else None, dx if need_r else None, dw if need_w else None, db if need_b else None, None)


def add_layer_norm(input, residual, weight, bias=None, eps=1e-5):
    """(weight * (h - mean(h)) / sqrt(var(h) + eps) + bias, h) with h = input + residual, over the last axis (var: mean
    square of h - mean(h)); a residual of None adds nothing.  weight and bias (None: none): one value for each of the
    last axis (up to 16384), both of the input's type or float32.  The sum is normalised before it is rounded to the
    input's type.  Second derivatives and forward mode raise."""
    if "layer_norm_pair" in _token_ops.NATIVE_OPS:
        both = _sdk_ops.layer_norm_pair(input, residual, weight, bias, float(eps))
        return (both[0], input) if residual is None else (both[0], both[1])
    if _wants_gradient(input, residual, weight, bias):
        return AddLayerNormFunction.apply(input, residual, weight, bias, float(eps))
    out, summed = _sdk_ops.add_layer_norm(input, residual, weight, bias, float(eps))[:2]
    return out, input if residual is None else summed


class GatedScanFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, state, lengths, reverse):
        out, last = _sdk_ops.gated_scan_forward(x, gate, state, lengths, reverse)
        ctx.save_for_backward(x, gate, state, lengths, out)
        ctx.reverse = reverse
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @_only_first
    def backward(ctx, grad_output, grad_last):
        x, gate, state, lengths, out = ctx.saved_tensors
        need_x, need_gate, need_state = ctx.needs_input_grad[:3]
        dx, dgate, dstate = _sdk_ops.gated_scan_backward(grad_output, grad_last, x, gate, state, lengths, out, ctx.reverse,
                                                         need_x, need_gate, need_state)
        return dx if need_x else None, dgate if need_gate else None, dstate if need_state else None, None, None


def gated_scan(input, gate, state=None, lengths=None, reverse=False):
    """(h, last state) of h_t = f_t h_{t-1} + (1 - f_t) input_t, f = sigmoid(gate), each channel by itself.

    input and gate [B, tokens, width] of one type (float32, bfloat16, float16), any strides whose last axis is dense
    (others are copied); h like them, dense.  state: h in front of the first token, float32 [B, width] (None: zeros);
    the last state, float32 too, is h behind the last token.  lengths (int32 [B]): tokens from lengths[b] on do not
    count; input and gate are not read there, h and the gradients are zeros.  reverse: from the last token that counts
    to the first.  The state is float32 throughout and h is rounded once; of f and 1 - f the lesser is formed to its own
    precision, so closed gates (of -8 and below) have all their digits too.  Inputs or states that are not finite give NaN
    or infinities from there on.  With gradients for input, gate and state; second derivatives and forward mode raise.

    Long sequences of few channels are cut into segments that are worked on side by side."""
    if "gated_scan" in _token_ops.NATIVE_OPS:
        both = _sdk_ops.gated_scan(input, gate, state, lengths, bool(reverse))
        return both[0], both[1]
    if _wants_gradient(input, gate, state):
        return GatedScanFunction.apply(input, gate, state, lengths, bool(reverse))
    return _sdk_ops.gated_scan_forward(input, gate, state, lengths, bool(reverse))


def gated_scan_step(input, gate, state):
    """One token of each sequence: state (float32 [B, width]) = f state + (1 - f) input with f = sigmoid(gate), in place;
    returns it in the input's type.  input and gate [B, width].  No gradients: raises where one would be wanted."""
    if _wants_gradient(input, gate, state):
        raise RuntimeError("gated_scan_step has no gradients: call it under torch.no_grad(), or gated_scan")
    return _sdk_ops.gated_scan_step(input, gate, state)


def _no_tensors(*lists):
    return not any(len(tensors) for tensors in lists)


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=1e-2):
    """One AdamW step over lists of tensors, in place and in few launches; step: 1 for the first.

    params and grads: float32, bfloat16 or float16, all of one type; both moments float32.
    m = m b1 + g (1 - b1);  v = v b2 + g g (1 - b2);
    p = p (1 - lr wd) - lr / (1 - b1 ** step) m / (sqrt(v / (1 - b2 ** step)) + eps)."""
    if _no_tensors(params, grads, exp_avgs, exp_avg_sqs):
        return
    with torch.no_grad():
        _sdk_ops.adamw_step(params, grads, exp_avgs, exp_avg_sqs, lr, betas[0], betas[1], eps, weight_decay, step)


def adamw_step_8bit(params, grads, avg_codes, avg_scales, sq_codes, sq_scales, *, step, lr=1e-3,
                    betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
    """adamw_step with both moments in 8 bits: each 256 consecutive values of a parameter share a float32
    scale s, the largest magnitude among them.  int8 code c of the first moment stands for
    c |c| / 127 ** 2 s, uint8 code c of the second for (c / 255) ** 4 s (1 at least where it is not
    zero).  Codes have the parameter's shape, scales [ceil(size / 256)].  The step itself uses the
    moments before they are rounded.  A block that meets a gradient that is not finite has a scale
    that is not finite from then on."""
    if _no_tensors(params, grads, avg_codes, avg_scales, sq_codes, sq_scales):
        return
    with torch.no_grad():
        _sdk_ops.adamw_step_8bit(params, grads, avg_codes, avg_scales, sq_codes, sq_scales, lr, betas[0], betas[1],
                                 eps, weight_decay, step)


def adamw_moment_values(codes, scales, dtype=torch.float32):
    """The values that the codes of a first (int8) or second (uint8) moment stand for."""
    return _sdk_ops.adamw_moment_values(codes, scales, dtype)


#: a, b, c of orthogonalize: steep at zero (3.4 times a step), so that five steps bring singular values from 0.002 of the
#: norm on to between 0.68 and 1.21.
NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)


def orthogonalize(input, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7):
    """Matrices [.., rows, columns] with their singular values brought towards one by products alone: X = input / (its
    Frobenius norm + eps), then `steps` times X = a X + (b S + c S S) X with S = X X^T of the smaller side.

    float32 and float16 matrices are multiplied with 22 bits a value, bfloat16 with 11 (but for S's diagonal and the
    polynomial's); sums are float32.
    Coefficients with which a singular value could pass 3.8, or a + b s + c s ** 2 pass 15 (s: its square), within the
    steps raise, also where only roundings (2 ** -10 a step) would take it there.  eps: 2 ** -100 to 1.  No gradients: raises where one would be wanted."""
    if _wants_gradient(input):
        raise RuntimeError("orthogonalize has no gradients: call it under torch.no_grad(), or of a detached input")
    return _sdk_ops.orthogonalize(input, steps, coefficients, eps)


def muon_step(params, grads, momenta, *, lr=2e-2, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
              coefficients=NEWTON_SCHULZ, eps=1e-7):
    """One Muon step over lists of parameters, in place and in few launches (64 parameters at a time).

    params and grads: float32, bfloat16 or float16, all of one type, two axes at least: [out, ..] counts as a matrix of
    `out` rows (weights [out, in, taps] of mapped convolutions among them); momenta float32.  No two tensors may overlap;
    one that is in the lists twice raises.
    m = momentum m + (1 - momentum) g;  u = momentum m + (1 - momentum) g with nesterov, else m;
    p = p (1 - lr weight_decay) - lr sqrt(max(1, rows / columns)) orthogonalize(u)."""
    if _no_tensors(params, grads, momenta):
        return
    with torch.no_grad():
        _sdk_ops.muon_step(params, grads, momenta, lr, momentum, nesterov, weight_decay, steps, coefficients, eps)
