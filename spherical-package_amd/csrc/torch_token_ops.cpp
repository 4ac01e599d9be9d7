// Compiled PyTorch-ROCm layer of the operators on token sequences: the checks, allocation, stream fetch and
// C-ABI call of _spherical_distortion_ext/_token_ops.py (which defines the schemas and keeps a Python
// implementation of each) in C++, where a call of a few microseconds on the GPU is not bound by its host side.
// Part of libsdk_torch_ops.so; no device code here.
#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <cstdint>
#include <optional>
#include <vector>

#include "sdk_mapped_ops.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kBlock = 256;   // values of a moment in 8 bits that share a scale

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
void* ptr(const Tensor& t) { return t.data_ptr(); }
void* ptr(const OptTensor& t) { return has(t) ? t->data_ptr() : nullptr; }

int dtype_of(at::ScalarType t, const char* name) {
  if (t == at::kFloat) return SDK_F32;
  if (t == at::kBFloat16) return SDK_BF16;
  TORCH_CHECK(t == at::kHalf, "unsupported dtype ", t, " of ", name, " (float32, bfloat16 and float16 only)");
  return SDK_F16;
}

void on_gpu(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "this backend runs on the GPU only: tensors must be CUDA/HIP tensors");
}
void beside(const Tensor& ref, const char* name, const Tensor& t) {
  TORCH_CHECK(t.is_cuda() && t.device() == ref.device(), name, " must be a CUDA tensor on ", ref.device());
}
void beside(const Tensor& ref, const char* name, const OptTensor& t) {
  if (has(t)) beside(ref, name, *t);
}
void dense(const char* name, const Tensor& t) { TORCH_CHECK(t.is_contiguous(), name, " must be contiguous"); }
void dense(const char* name, const OptTensor& t) {
  if (has(t)) dense(name, *t);
}

hipStream_t stream_of(const Tensor& ref) {
  return c10::hip::getCurrentHIPStream(ref.device().index()).stream();
}

#define TOKEN_CALL(name, ...)                                                                             \
  do {                                                                                                    \
    const int rc__ = name(__VA_ARGS__);                                                                   \
    TORCH_CHECK(rc__ == 0, #name, " failed (status ", rc__, "): ", sdk_last_error());                     \
  } while (0)

Tensor nothing(const Tensor& like) { return at::empty({0}, like.options()); }

// ------------------------------------------------------------------------------------------ attention
// Whether the kernels read `t` where it lies: last axis dense, rows 16-byte aligned, 64 tokens within 2^31 bytes.
bool rows_fit(const Tensor& t) {
  const int64_t each = 16 / (int64_t)t.element_size();
  bool ok = (uintptr_t)t.data_ptr() % 16 == 0 && (t.size(-1) == 1 || t.stride(-1) == 1);
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) == 1 || t.stride(i) % each == 0);
  return ok && (t.size(2) == 1 || t.stride(2) < ((int64_t)1 << 31) / (64 * (int64_t)t.element_size()));
}
// A dense copy, of a dense tensor too (which may lie at any address).
Tensor laid_out(const Tensor& t) { return t.clone(at::MemoryFormat::Contiguous); }
Tensor rows_ready(const Tensor& t) { return rows_fit(t) ? t : laid_out(t); }

// Batch, head and token strides; those of axes of length one do not count.
void strides(const Tensor& t, int64_t (&s)[3]) {
  for (int i = 0; i < 3; ++i) s[i] = t.size(i) == 1 ? 0 : t.stride(i);
}

void check_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& map,
                     const OptTensor& lengths, double scale) {
  on_gpu(q);
  beside(q, "key", k), beside(q, "value", v), beside(q, "bias_table", table), beside(q, "bucket_map", map);
  beside(q, "key_lengths", lengths);
  (void)dtype_of(q.scalar_type(), "query");
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4, "query and key must be [batch, heads, tokens, dim], got ", q.sizes(),
              " and ", k.sizes());
  const int64_t B = q.size(0), H = q.size(1), Lq = q.size(2), D = q.size(3);
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == B && k.size(3) == D, "key ", k.sizes(), " and value ",
              v.sizes(), " must be [", B, ", key heads, keys, ", D, "]");
  const int64_t Hk = k.size(1), Lk = k.size(2);
  TORCH_CHECK(Hk >= 1 && H >= 1 && H % Hk == 0, "heads = ", H, " must be a multiple of key heads = ", Hk);
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
              "key and value must have dtype ", q.scalar_type(), " (got ", k.scalar_type(), " and ", v.scalar_type(),
              ")");
  TORCH_CHECK(D >= 8 && D <= 128 && D % 8 == 0, "dim = ", D, " must be a multiple of 8 up to 128");
  TORCH_CHECK(table.dim() == 2 && table.size(0) == H && table.size(1) >= 1 && table.size(1) <= 256, "bias_table ",
              table.sizes(), " must be [", H, ", buckets], 1 to 256 buckets");
  TORCH_CHECK(table.scalar_type() == q.scalar_type() || table.scalar_type() == at::kFloat,
              "bias_table must have dtype ", q.scalar_type(), " or float32 (got ", table.scalar_type(), ")");
  TORCH_CHECK(map.scalar_type() == at::kByte, "bucket_map must have dtype uint8 (got ", map.scalar_type(), ")");
  TORCH_CHECK((map.dim() == 2 || (map.dim() == 3 && map.size(0) == B)) && map.size(-2) == Lq && map.size(-1) == Lk,
              "bucket_map ", map.sizes(), " must be [", Lq, ", ", Lk, "] or [", B, ", ", Lq, ", ", Lk, "]");
  if (has(lengths)) {
    TORCH_CHECK(lengths->scalar_type() == at::kInt && lengths->dim() == 1 && lengths->size(0) == B,
                "key_lengths must be int32 of shape [", B, "], got ", lengths->scalar_type(), " ", lengths->sizes());
    dense("key_lengths", lengths);
  }
  TORCH_CHECK(scale >= 0x1p-32 && scale <= 0x1p32, "scale must be between 2^-32 and 2^32, got ", scale);
}

// The argument block; the tensors may be replaced by dense copies, which the caller keeps.
sdk_bucket_attention attention_args(Tensor& q, Tensor& k, Tensor& v, Tensor& table, Tensor& map,
                                    const OptTensor& lengths, bool causal, double scale) {
  q = rows_ready(q), k = rows_ready(k), v = rows_ready(v), table = table.contiguous();
  if (map.size(-1) != 1 && map.stride(-1) != 1) map = map.contiguous();
  sdk_bucket_attention a = {};
  a.query = ptr(q), a.key = ptr(k), a.value = ptr(v), a.bias_table = ptr(table);
  a.bucket_map = (const uint8_t*)ptr(map), a.key_lengths = (const int32_t*)ptr(lengths);
  a.batch = q.size(0), a.heads = q.size(1), a.queries = q.size(2), a.dim = q.size(3);
  a.key_heads = k.size(1), a.keys = k.size(2), a.buckets = table.size(1);
  strides(q, a.query_strides), strides(k, a.key_strides), strides(v, a.value_strides);
  a.map_strides[0] = map.dim() == 3 ? map.stride(0) : 0, a.map_strides[1] = map.stride(-2);
  a.scale = scale, a.causal = causal;
  a.dtype = dtype_of(q.scalar_type(), "query"), a.table_dtype = dtype_of(table.scalar_type(), "bias_table");
  return a;
}

Tensor workspace(const Tensor& ref, size_t bytes) {
  return bytes ? at::empty({(int64_t)bytes}, ref.options().dtype(at::kByte)) : Tensor();
}

// for_backward: with the lse and, of 16-bit types, what rounding took from the output.
std::tuple<Tensor, Tensor, Tensor> attend(Tensor q, Tensor k, Tensor v, Tensor table, Tensor map,
                                          const OptTensor& lengths, bool causal, double scale, bool for_backward) {
  check_attention(q, k, v, table, map, lengths, scale);
  c10::DeviceGuard guard(q.device());
  sdk_bucket_attention a = attention_args(q, k, v, table, map, lengths, causal, scale);
  Tensor out = at::empty_like(q), rest, lse;
  a.output = ptr(out);
  if (for_backward) {
    lse = at::empty({2, q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
    a.lse = (float*)ptr(lse);
    rest = q.scalar_type() == at::kFloat ? nothing(q) : at::empty_like(out);
    if (rest.numel()) a.output_rest = ptr(rest);
  }
  strides(out, a.output_strides);
  const size_t need = sdk_bucket_attention_workspace_bytes(&a, 0);
  Tensor ws = workspace(q, need);
  TOKEN_CALL(sdk_bucket_attention_forward, &a, need ? ptr(ws) : nullptr, need, stream_of(q));
  return {out, rest, lse};
}

std::tuple<Tensor, Tensor, Tensor> bucket_attention_forward(const Tensor& q, const Tensor& k, const Tensor& v,
                                                            const Tensor& table, const Tensor& map,
                                                            const OptTensor& lengths, bool causal, double scale) {
  return attend(q, k, v, table, map, lengths, causal, scale, true);
}

std::tuple<Tensor, Tensor, Tensor, Tensor> bucket_attention_backward(
    Tensor grad, Tensor q, Tensor k, Tensor v, Tensor table, Tensor map, const OptTensor& lengths, Tensor out,
    Tensor rest, Tensor lse, bool causal, double scale, bool need_query, bool need_keys, bool need_table) {
  check_attention(q, k, v, table, map, lengths, scale);
  beside(q, "grad_output", grad), beside(q, "output", out), beside(q, "rest", rest), beside(q, "lse", lse);
  TORCH_CHECK(grad.sizes() == q.sizes() && out.sizes() == q.sizes() && lse.dim() == 4 && lse.size(0) == 2 &&
                  lse.sizes().slice(1) == q.sizes().slice(0, 3),
              "grad_output, output and lse must have the shapes of the forward's results");
  TORCH_CHECK(grad.scalar_type() == q.scalar_type() && out.scalar_type() == q.scalar_type() &&
                  lse.scalar_type() == at::kFloat,
              "grad_output and output must have dtype ", q.scalar_type(), ", lse float32");
  TORCH_CHECK(rest.numel() == 0 || (rest.sizes() == out.sizes() && rest.strides() == out.strides() &&
                                    rest.scalar_type() == out.scalar_type()),
              "the output's rest must be like the output, or empty");
  c10::DeviceGuard guard(q.device());
  sdk_bucket_attention a = attention_args(q, k, v, table, map, lengths, causal, scale);
  grad = rows_ready(grad), lse = lse.contiguous();
  if (!rows_fit(out) || (rest.numel() && !rows_fit(rest)))   // both are read by the output's strides
    out = laid_out(out), rest = laid_out(rest);
  a.grad_output = ptr(grad), a.output = ptr(out), a.lse = (float*)ptr(lse);
  strides(grad, a.grad_output_strides), strides(out, a.output_strides);
  if (rest.numel()) a.output_rest = ptr(rest);
  Tensor dq = need_query ? at::empty_like(q) : nothing(q);
  Tensor dk = need_keys ? at::empty_like(k) : nothing(k), dv = need_keys ? at::empty_like(v) : nothing(v);
  Tensor dt = need_table ? at::empty_like(table) : nothing(table);
  if (need_query) a.grad_query = ptr(dq), strides(dq, a.grad_query_strides);
  if (need_keys) {
    a.grad_key = ptr(dk), a.grad_value = ptr(dv);
    strides(dk, a.grad_key_strides), strides(dv, a.grad_value_strides);
  }
  if (need_table) a.grad_table = ptr(dt);
  const size_t need = sdk_bucket_attention_workspace_bytes(&a, 1);
  Tensor ws = workspace(q, need);
  TOKEN_CALL(sdk_bucket_attention_backward, &a, need ? ptr(ws) : nullptr, need, stream_of(q));
  return {dq, dk, dv, dt};
}

// ------------------------------------------------------------------------------------------ norm
void check_norm(const Tensor& x, const OptTensor& residual, const Tensor& weight) {
  on_gpu(x);
  beside(x, "residual", residual), beside(x, "weight", weight);
  dense("x", x), dense("residual", residual), dense("weight", weight);
  (void)dtype_of(x.scalar_type(), "x");
  TORCH_CHECK(x.dim() >= 1 && weight.dim() == 1 && weight.size(0) == x.size(-1), "weight ", weight.sizes(),
              " must have one value for each of the last axis of x ", x.sizes());
  TORCH_CHECK(x.size(-1) >= 1 && x.size(-1) <= 16384, "width = ", x.size(-1), " must be between 1 and 16384");
  TORCH_CHECK(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat,
              "weight must have dtype ", x.scalar_type(), " or float32 (got ", weight.scalar_type(), ")");
  if (has(residual))
    TORCH_CHECK(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(),
                "residual must be like x: ", x.sizes(), " ", x.scalar_type(), ", got ", residual->sizes(), " ",
                residual->scalar_type());
}

void norm(const Tensor& x, const OptTensor& residual, const Tensor& weight, const Tensor& out, float* scales,
          const Tensor& summed, float* inverse, double eps, int codes) {
  const int64_t width = x.size(-1);
  TOKEN_CALL(sdk_add_rms_norm, ptr(x), ptr(residual), ptr(weight), ptr(out), scales,
             has(residual) ? ptr(summed) : nullptr, inverse, x.numel() / width, width, eps, codes,
             dtype_of(x.scalar_type(), "x"), dtype_of(weight.scalar_type(), "weight"), stream_of(x));
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm(const Tensor& x, const OptTensor& residual, const Tensor& weight,
                                                double eps) {
  check_norm(x, residual, weight);
  c10::DeviceGuard guard(x.device());
  Tensor out = at::empty_like(x), summed = has(residual) ? at::empty_like(x) : nothing(x);
  Tensor inverse = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  norm(x, residual, weight, out, nullptr, summed, (float*)ptr(inverse), eps, 0);
  return {out, summed, inverse};
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_quantized(const Tensor& x, const OptTensor& residual,
                                                          const Tensor& weight, double eps, bool fp8) {
  check_norm(x, residual, weight);
  c10::DeviceGuard guard(x.device());
  Tensor codes = at::empty(x.sizes(), x.options().dtype(fp8 ? at::kFloat8_e4m3fn : at::kChar));
  Tensor summed = has(residual) ? at::empty_like(x) : nothing(x);
  Tensor scales = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  norm(x, residual, weight, codes, (float*)ptr(scales), summed, nullptr, eps, fp8 ? 2 : 1);
  return {codes, scales, summed};
}

std::tuple<Tensor, Tensor> add_rms_norm_backward(const Tensor& grad, const OptTensor& grad_sum, const Tensor& summed,
                                                 const Tensor& weight, const Tensor& inverse, bool need_x,
                                                 bool need_weight) {
  check_norm(summed, OptTensor(), weight);
  beside(summed, "grad", grad), beside(summed, "grad_sum", grad_sum), beside(summed, "inverse", inverse);
  for (const auto& t : {std::pair<const char*, OptTensor>{"grad", grad}, {"grad_sum", grad_sum}})
    if (has(t.second))
      TORCH_CHECK(t.second->sizes() == summed.sizes() && t.second->scalar_type() == summed.scalar_type(), t.first,
                  " must be like the sums: ", summed.sizes(), " ", summed.scalar_type(), ", got ", t.second->sizes(),
                  " ", t.second->scalar_type());
  dense("grad", grad), dense("grad_sum", grad_sum), dense("inverse", inverse);
  const int64_t width = summed.size(-1), rows = summed.numel() / width;
  TORCH_CHECK(inverse.scalar_type() == at::kFloat && inverse.numel() == rows,
              "inverse must be float32 with one value for each row");
  c10::DeviceGuard guard(summed.device());
  Tensor dx = need_x ? at::empty_like(summed) : nothing(summed);
  Tensor dw = need_weight ? at::empty_like(weight) : nothing(weight);
  if (!need_x && !need_weight) return {dx, dw};
  const size_t need = need_weight ? sdk_add_rms_norm_backward_workspace_bytes(rows, width) : 0;
  Tensor ws = workspace(summed, need);
  TOKEN_CALL(sdk_add_rms_norm_backward, ptr(grad), ptr(grad_sum), ptr(summed), ptr(weight),
             (const float*)ptr(inverse), need_x ? ptr(dx) : nullptr, need_weight ? ptr(dw) : nullptr,
             need ? ptr(ws) : nullptr, need, rows, width, dtype_of(summed.scalar_type(), "summed"),
             dtype_of(weight.scalar_type(), "weight"), stream_of(summed));
  return {dx, dw};
}

Tensor dequantize_rows(const Tensor& codes, const Tensor& scales, at::ScalarType dtype) {
  on_gpu(codes);
  beside(codes, "scales", scales);
  dense("codes", codes), dense("scales", scales);
  const bool fp8 = codes.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(fp8 || codes.scalar_type() == at::kChar, "codes must be int8 or float8_e4m3fn (got ",
              codes.scalar_type(), ")");
  const int to = dtype_of(dtype, "the result");
  TORCH_CHECK(codes.dim() >= 1 && codes.size(-1) >= 1 && scales.scalar_type() == at::kFloat &&
                  scales.sizes() == codes.sizes().slice(0, codes.dim() - 1),
              "scales must be float32 with one value for each row of codes ", codes.sizes(), ", got ",
              scales.scalar_type(), " ", scales.sizes());
  c10::DeviceGuard guard(codes.device());
  Tensor out = at::empty(codes.sizes(), codes.options().dtype(dtype));
  const int64_t width = codes.size(-1);
  TOKEN_CALL(sdk_dequantize_rows, ptr(codes), (const float*)ptr(scales), ptr(out), codes.numel() / width, width,
             fp8 ? 2 : 1, to, stream_of(codes));
  return out;
}

// ------------------------------------------------------------------------------------------ layer norm
void check_layer_norm(const Tensor& x, const OptTensor& residual, const Tensor& weight, const OptTensor& bias) {
  check_norm(x, residual, weight);
  beside(x, "bias", bias);
  dense("bias", bias);
  if (has(bias))
    TORCH_CHECK(bias->sizes() == weight.sizes() && bias->scalar_type() == weight.scalar_type(),
                "bias must be like weight: ", weight.sizes(), " ", weight.scalar_type(), ", got ", bias->sizes(), " ",
                bias->scalar_type());
}

// for_backward: with each row's mean and reciprocal standard deviation.
std::tuple<Tensor, Tensor, Tensor, Tensor> layer_norm(const Tensor& x, const OptTensor& residual, const Tensor& weight,
                                                      const OptTensor& bias, double eps, bool for_backward) {
  check_layer_norm(x, residual, weight, bias);
  c10::DeviceGuard guard(x.device());
  Tensor out = at::empty_like(x), summed = has(residual) ? at::empty_like(x) : nothing(x), mean, inverse;
  if (for_backward) {
    mean = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
    inverse = at::empty_like(mean);
  }
  const int64_t width = x.size(-1);
  TOKEN_CALL(sdk_add_layer_norm, ptr(x), ptr(residual), ptr(weight), ptr(bias), ptr(out),
             has(residual) ? ptr(summed) : nullptr, for_backward ? (float*)ptr(mean) : nullptr,
             for_backward ? (float*)ptr(inverse) : nullptr, x.numel() / width, width, eps,
             dtype_of(x.scalar_type(), "x"), dtype_of(weight.scalar_type(), "weight"), stream_of(x));
  return {out, summed, mean, inverse};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> add_layer_norm(const Tensor& x, const OptTensor& residual,
                                                          const Tensor& weight, const OptTensor& bias, double eps) {
  return layer_norm(x, residual, weight, bias, eps, true);
}

std::tuple<Tensor, Tensor, Tensor> add_layer_norm_backward(const Tensor& grad, const OptTensor& grad_sum,
                                                           const Tensor& x, const OptTensor& residual, const Tensor& weight,
                                                           const Tensor& mean, const Tensor& inverse, bool need_x,
                                                           bool need_weight, bool need_bias) {
  check_norm(x, residual, weight);
  beside(x, "grad", grad), beside(x, "grad_sum", grad_sum);
  beside(x, "mean", mean), beside(x, "inverse", inverse);
  for (const auto& t : {std::pair<const char*, OptTensor>{"grad", grad}, {"grad_sum", grad_sum}})
    if (has(t.second))
      TORCH_CHECK(t.second->sizes() == x.sizes() && t.second->scalar_type() == x.scalar_type(), t.first,
                  " must be like x: ", x.sizes(), " ", x.scalar_type(), ", got ", t.second->sizes(),
                  " ", t.second->scalar_type());
  dense("grad", grad), dense("grad_sum", grad_sum), dense("mean", mean), dense("inverse", inverse);
  const int64_t width = x.size(-1), rows = x.numel() / width;
  for (const Tensor& t : {mean, inverse})
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.numel() == rows,
                "mean and inverse must be float32 with one value for each row");
  c10::DeviceGuard guard(x.device());
  Tensor dx = need_x ? at::empty_like(x) : nothing(x);
  Tensor dw = need_weight ? at::empty_like(weight) : nothing(weight);
  Tensor db = need_bias ? at::empty_like(weight) : nothing(weight);
  if (!need_x && !need_weight && !need_bias) return {dx, dw, db};
  const size_t need = need_weight || need_bias ? sdk_add_layer_norm_backward_workspace_bytes(rows, width) : 0;
  Tensor ws = workspace(x, need);
  TOKEN_CALL(sdk_add_layer_norm_backward, ptr(grad), ptr(grad_sum), ptr(x), ptr(residual), ptr(weight), (const float*)ptr(mean),
             (const float*)ptr(inverse), need_x ? ptr(dx) : nullptr, need_weight ? ptr(dw) : nullptr,
             need_bias ? ptr(db) : nullptr, need ? ptr(ws) : nullptr, need, rows, width,
             dtype_of(x.scalar_type(), "x"), dtype_of(weight.scalar_type(), "weight"), stream_of(x));
  return {dx, dw, db};
}

// ------------------------------------------------------------------------------------------ gated scan
void check_scan(const Tensor& x, const Tensor& gate, const OptTensor& state, const OptTensor& lengths) {
  on_gpu(x);
  beside(x, "gate", gate), beside(x, "state", state), beside(x, "lengths", lengths);
  (void)dtype_of(x.scalar_type(), "x");
  TORCH_CHECK(x.dim() == 3, "x must be [batch, tokens, width], got ", x.sizes());
  TORCH_CHECK(gate.sizes() == x.sizes() && gate.scalar_type() == x.scalar_type(), "gate must be like x: ", x.sizes(), " ",
              x.scalar_type(), ", got ", gate.sizes(), " ", gate.scalar_type());
  const int64_t B = x.size(0), D = x.size(2);
  if (has(state))
    TORCH_CHECK(state->dim() == 2 && state->size(0) == B && state->size(1) == D && state->scalar_type() == at::kFloat,
                "state must be float32 of shape [", B, ", ", D, "], got ", state->scalar_type(), " ", state->sizes());
  if (has(lengths)) {
    TORCH_CHECK(lengths->scalar_type() == at::kInt && lengths->dim() == 1 && lengths->size(0) == B,
                "lengths must be int32 of shape [", B, "], got ", lengths->scalar_type(), " ", lengths->sizes());
    dense("lengths", lengths);
  }
}

Tensor tokens_ready(const Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : laid_out(t); }

// Batch and token strides; those of axes of length one do not count.
void token_strides(const Tensor& t, int64_t (&s)[2]) {
  for (int i = 0; i < 2; ++i) s[i] = t.size(i) == 1 ? 0 : t.stride(i);
}

// The argument block; the tensors may be replaced by dense copies, which the caller keeps.
sdk_gated_scan scan_args(Tensor& x, Tensor& gate, OptTensor& state, const OptTensor& lengths, bool reverse) {
  x = tokens_ready(x), gate = tokens_ready(gate);
  if (has(state)) state = state->contiguous();
  sdk_gated_scan a = {};
  a.x = ptr(x), a.gate = ptr(gate), a.state = (const float*)ptr(state), a.lengths = (const int32_t*)ptr(lengths);
  a.batch = x.size(0), a.tokens = x.size(1), a.width = x.size(2);
  token_strides(x, a.x_strides), token_strides(gate, a.gate_strides);
  a.reverse = reverse, a.dtype = dtype_of(x.scalar_type(), "x");
  return a;
}

std::tuple<Tensor, Tensor> gated_scan_forward(Tensor x, Tensor gate, OptTensor state, const OptTensor& lengths,
                                              bool reverse) {
  check_scan(x, gate, state, lengths);
  c10::DeviceGuard guard(x.device());
  sdk_gated_scan a = scan_args(x, gate, state, lengths, reverse);
  Tensor out = at::empty(x.sizes(), x.options());
  Tensor last = at::empty({x.size(0), x.size(2)}, x.options().dtype(at::kFloat));
  a.output = ptr(out), a.last = (float*)ptr(last);
  const size_t need = sdk_gated_scan_workspace_bytes(&a, 0);
  Tensor ws = workspace(x, need);
  TOKEN_CALL(sdk_gated_scan_forward, &a, need ? ptr(ws) : nullptr, need, stream_of(x));
  return {out, last};
}

std::tuple<Tensor, Tensor, Tensor> gated_scan_backward(OptTensor grad, OptTensor grad_last, Tensor x, Tensor gate,
                                                       OptTensor state, const OptTensor& lengths, Tensor output,
                                                       bool reverse, bool need_x, bool need_gate, bool need_state) {
  check_scan(x, gate, state, lengths);
  beside(x, "grad_output", grad), beside(x, "grad_last", grad_last), beside(x, "output", output);
  const int64_t B = x.size(0), D = x.size(2);
  for (const auto& t : {std::pair<const char*, OptTensor>{"grad_output", grad}, {"output", output}})
    if (has(t.second))
      TORCH_CHECK(t.second->sizes() == x.sizes() && t.second->scalar_type() == x.scalar_type(), t.first,
                  " must be like x: ", x.sizes(), " ", x.scalar_type(), ", got ", t.second->sizes(), " ",
                  t.second->scalar_type());
  if (has(grad_last))
    TORCH_CHECK(grad_last->dim() == 2 && grad_last->size(0) == B && grad_last->size(1) == D &&
                    grad_last->scalar_type() == at::kFloat,
                "grad_last must be float32 of shape [", B, ", ", D, "]");
  c10::DeviceGuard guard(x.device());
  Tensor dx = need_x ? at::empty(x.sizes(), x.options()) : nothing(x);
  Tensor dgate = need_gate ? at::empty(x.sizes(), x.options()) : nothing(x);
  Tensor dstate = need_state ? at::empty({B, D}, x.options().dtype(at::kFloat))
                             : at::empty({0}, x.options().dtype(at::kFloat));
  if (!need_x && !need_gate && !need_state) return {dx, dgate, dstate};
  sdk_gated_scan a = scan_args(x, gate, state, lengths, reverse);
  output = output.contiguous();
  a.output = ptr(output);
  if (has(grad)) {
    grad = tokens_ready(*grad);
    a.grad_output = ptr(grad), token_strides(*grad, a.grad_output_strides);
  }
  if (has(grad_last)) grad_last = grad_last->contiguous(), a.grad_last = (const float*)ptr(grad_last);
  if (need_x) a.grad_x = ptr(dx);
  if (need_gate) a.grad_gate = ptr(dgate);
  if (need_state) a.grad_state = (float*)ptr(dstate);
  const size_t need = sdk_gated_scan_workspace_bytes(&a, 1);
  Tensor ws = workspace(x, need);
  TOKEN_CALL(sdk_gated_scan_backward, &a, need ? ptr(ws) : nullptr, need, stream_of(x));
  return {dx, dgate, dstate};
}

// ------------------------------------------------------------------------------------------ AdamW
// The pointers of `tensors`, one for each parameter: like it, or `each` values to a scale.
std::vector<void*> pointers(const char* name, at::TensorList params, at::TensorList tensors, at::ScalarType dtype,
                            bool scales) {
  TORCH_CHECK(tensors.size() == params.size(), tensors.size(), " ", name, " for ", params.size(), " params");
  std::vector<void*> out(tensors.size());
  for (size_t i = 0; i < tensors.size(); ++i) {
    const Tensor &t = tensors[i], &p = params[i];
    TORCH_CHECK(t.scalar_type() == dtype && t.device() == params[0].device(), name, "[", i, "] must have dtype ",
                dtype, " on ", params[0].device(), " (got ", t.scalar_type(), " on ", t.device(), ")");
    const bool fits = scales ? t.dim() == 1 && t.size(0) == (p.numel() + kBlock - 1) / kBlock : t.sizes() == p.sizes();
    TORCH_CHECK(fits, name, "[", i, "] has shape ", t.sizes(), " for a parameter ", p.sizes());
    TORCH_CHECK(t.is_contiguous(), name, "[", i, "] must be contiguous");
    out[i] = t.data_ptr();
  }
  return out;
}

std::vector<int64_t> sizes_of(at::TensorList params) {
  std::vector<int64_t> n(params.size());
  for (size_t i = 0; i < params.size(); ++i) n[i] = params[i].numel();
  return n;
}

// The kernels write through pointers: autograd has to learn of it to refuse a backward through the former values.
void changed(std::initializer_list<at::TensorList> lists) {
  for (const at::TensorList& tensors : lists)
    for (const Tensor& t : tensors)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void adamw_step(at::TensorList params, at::TensorList grads, at::TensorList avgs, at::TensorList sqs, double lr,
                double beta1, double beta2, double eps, double weight_decay, int64_t step) {
  if (params.empty()) return;
  on_gpu(params[0]);
  const at::ScalarType type = params[0].scalar_type();
  const int dtype = dtype_of(type, "params");
  const auto p = pointers("params", params, params, type, false), g = pointers("grads", params, grads, type, false);
  const auto m = pointers("exp_avgs", params, avgs, at::kFloat, false);
  const auto v = pointers("exp_avg_sqs", params, sqs, at::kFloat, false);
  const auto n = sizes_of(params);
  c10::DeviceGuard guard(params[0].device());
  TOKEN_CALL(sdk_adamw_step, p.data(), g.data(), (float* const*)m.data(), (float* const*)v.data(), n.data(),
             (int64_t)n.size(), lr, beta1, beta2, eps, weight_decay, step, dtype, stream_of(params[0]));
  changed({params, avgs, sqs});
}

void adamw_step_8bit(at::TensorList params, at::TensorList grads, at::TensorList avg_codes, at::TensorList avg_scales,
                     at::TensorList sq_codes, at::TensorList sq_scales, double lr, double beta1, double beta2,
                     double eps, double weight_decay, int64_t step) {
  if (params.empty()) return;
  on_gpu(params[0]);
  const at::ScalarType type = params[0].scalar_type();
  const int dtype = dtype_of(type, "params");
  const auto p = pointers("params", params, params, type, false), g = pointers("grads", params, grads, type, false);
  const auto mc = pointers("avg_codes", params, avg_codes, at::kChar, false);
  const auto ms = pointers("avg_scales", params, avg_scales, at::kFloat, true);
  const auto vc = pointers("sq_codes", params, sq_codes, at::kByte, false);
  const auto vs = pointers("sq_scales", params, sq_scales, at::kFloat, true);
  const auto n = sizes_of(params);
  c10::DeviceGuard guard(params[0].device());
  TOKEN_CALL(sdk_adamw_step_8bit, p.data(), g.data(), (int8_t* const*)mc.data(), (float* const*)ms.data(),
             (uint8_t* const*)vc.data(), (float* const*)vs.data(), n.data(), (int64_t)n.size(), lr, beta1, beta2, eps,
             weight_decay, step, dtype, stream_of(params[0]));
  changed({params, avg_codes, avg_scales, sq_codes, sq_scales});
}

Tensor adamw_moment_values(const Tensor& codes, const Tensor& scales, at::ScalarType dtype) {
  on_gpu(codes);
  beside(codes, "scales", scales);
  dense("codes", codes), dense("scales", scales);
  const bool second = codes.scalar_type() == at::kByte;
  TORCH_CHECK(second || codes.scalar_type() == at::kChar,
              "codes must be int8 (first moment) or uint8 (second), got ", codes.scalar_type());
  const int to = dtype_of(dtype, "the result");
  TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.dim() == 1 &&
                  scales.size(0) == (codes.numel() + kBlock - 1) / kBlock,
              "scales must be float32 of shape [", (codes.numel() + kBlock - 1) / kBlock, "], got ",
              scales.scalar_type(), " ", scales.sizes());
  c10::DeviceGuard guard(codes.device());
  Tensor out = at::empty(codes.sizes(), codes.options().dtype(dtype));
  TOKEN_CALL(sdk_adamw_moment_values, ptr(codes), (const float*)ptr(scales), ptr(out), codes.numel(), (int)second, to,
             stream_of(codes));
  return out;
}

// One token of each sequence, the state in place.
Tensor gated_scan_step(Tensor x, Tensor gate, const Tensor& state) {
  on_gpu(x);
  beside(x, "gate", gate), beside(x, "state", state);
  const int dtype = dtype_of(x.scalar_type(), "x");
  TORCH_CHECK(x.dim() == 2 && gate.sizes() == x.sizes() && gate.scalar_type() == x.scalar_type(),
              "x and gate must be [batch, width] of one type, got ", x.sizes(), " ", x.scalar_type(), " and ",
              gate.sizes(), " ", gate.scalar_type());
  const int64_t B = x.size(0), D = x.size(1);
  TORCH_CHECK(state.sizes() == x.sizes() && state.scalar_type() == at::kFloat, "state must be float32 of shape [", B,
              ", ", D, "], got ", state.scalar_type(), " ", state.sizes());
  TORCH_CHECK((D <= 1 || state.stride(1) == 1) && (B <= 1 || state.stride(0) >= D),
              "state must have dense rows that do not overlap (it is changed in place), got strides ", state.strides());
  c10::DeviceGuard guard(x.device());
  x = tokens_ready(x), gate = tokens_ready(gate);
  Tensor out = at::empty({B, D}, x.options());
  TOKEN_CALL(sdk_gated_scan_step, ptr(x), x.stride(0), ptr(gate), gate.stride(0), (float*)ptr(state), state.stride(0),
             ptr(out), B, D, dtype, stream_of(x));
  changed({state});
  return out;
}

// ------------------------------------------------------------------------------------------ Muon
Tensor orthogonalize(Tensor x, int64_t steps, at::ArrayRef<double> coefficients, double eps) {
  on_gpu(x);
  const int dtype = dtype_of(x.scalar_type(), "x");
  TORCH_CHECK(x.dim() >= 2, "x must be [.., rows, columns], got ", x.sizes());
  TORCH_CHECK(coefficients.size() == 3, "coefficients must be three numbers, got ", coefficients.size());
  TORCH_CHECK(steps >= 1 && steps <= 100, "steps = ", steps, " must be between 1 and 100");
  c10::DeviceGuard guard(x.device());
  x = x.contiguous();
  Tensor out = at::empty(x.sizes(), x.options());
  const int64_t rows = x.size(-2), columns = x.size(-1), count = x.numel() ? x.numel() / (rows * columns) : 0;
  const size_t need = sdk_orthogonalize_workspace_bytes(rows, columns, count, dtype);
  Tensor ws = workspace(x, need);
  TOKEN_CALL(sdk_orthogonalize, ptr(x), ptr(out), rows, columns, count, (int)steps, coefficients.data(), eps,
             need ? ptr(ws) : nullptr, need, dtype, stream_of(x));
  return out;
}

void muon_step(at::TensorList params, at::TensorList grads, at::TensorList momenta, double lr, double momentum,
               bool nesterov, double weight_decay, int64_t steps, at::ArrayRef<double> coefficients, double eps) {
  if (params.empty()) {
    TORCH_CHECK(grads.empty() && momenta.empty(), "gradients or momenta without params");
    return;
  }
  on_gpu(params[0]);
  const at::ScalarType type = params[0].scalar_type();
  const int dtype = dtype_of(type, "params");
  const auto p = pointers("params", params, params, type, false), g = pointers("grads", params, grads, type, false);
  const auto m = pointers("momenta", params, momenta, at::kFloat, false);
  TORCH_CHECK(coefficients.size() == 3, "coefficients must be three numbers, got ", coefficients.size());
  TORCH_CHECK(steps >= 1 && steps <= 100, "steps = ", steps, " must be between 1 and 100");
  std::vector<int64_t> rows(params.size()), columns(params.size());
  for (size_t i = 0; i < params.size(); ++i) {
    TORCH_CHECK(params[i].dim() >= 2, "params[", i, "] must have two axes at least, got ", params[i].sizes());
    rows[i] = params[i].size(0), columns[i] = rows[i] ? params[i].numel() / rows[i] : 0;
  }
  c10::DeviceGuard guard(params[0].device());
  const int64_t n = (int64_t)params.size();
  const size_t need = sdk_muon_step_workspace_bytes(rows.data(), columns.data(), n, dtype);
  Tensor ws = workspace(params[0], need);
  TOKEN_CALL(sdk_muon_step, p.data(), g.data(), (float* const*)m.data(), rows.data(), columns.data(), n, lr, momentum,
             (int)nesterov, weight_decay, (int)steps, coefficients.data(), eps, need ? ptr(ws) : nullptr, need, dtype,
             stream_of(params[0]));
  changed({params, momenta});
}

// ------------------------------------------------------------------------------------------ autograd
// The differentiable forms: what functional/token_ops.py's autograd functions do, without an interpreter in the
// backward.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Below autograd a tangent would be left out.
void no_tangent(std::initializer_list<const Tensor*> tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : tensors)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(/*level=*/0).defined(),
                "forward-mode derivatives of this operator are not implemented");
}

bool wants_gradient(std::initializer_list<const Tensor*> tensors) {
  no_tangent(tensors);
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : tensors)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// Gradients of a backward that is itself recorded (create_graph): they ask for a gradient, and raise when it is formed.
// Plain tensors would be constants to whatever is differentiated beside them.
variable_list only_first(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);
  const auto node = std::make_shared<torch::autograd::DelayedError>(
      "second derivatives of this operator are not implemented", (int64_t)grads.size());
  return (*node)(std::move(grads));
}

struct BucketAttention : torch::autograd::Function<BucketAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table,
                        const Tensor& map, const OptTensor& lengths, bool causal, double scale) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [out, rest, lse] = bucket_attention_forward(q, k, v, table, map, lengths, causal, scale);
    ctx->save_for_backward({q, k, v, table, map, has(lengths) ? *lengths : Tensor(), out, rest, lse});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) { return only_first(gradients(ctx, grads)); }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const OptTensor n = saved[5].defined() ? OptTensor(saved[5]) : OptTensor();
    const bool need_q = ctx->needs_input_grad(0), need_k = ctx->needs_input_grad(1), need_v = ctx->needs_input_grad(2),
               need_t = ctx->needs_input_grad(3);
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [dq, dk, dv, dt] = bucket_attention_backward(
        grads[0], saved[0], saved[1], saved[2], saved[3], saved[4], n, saved[6], saved[7], saved[8],
        ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble(), need_q, need_k || need_v, need_t);
    return {need_q ? dq : Tensor(), need_k ? dk : Tensor(), need_v ? dv : Tensor(), need_t ? dt : Tensor(),
            Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor bucket_attention_only(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& map,
                             const OptTensor& lengths, bool causal, double scale) {
  return std::get<0>(attend(q, k, v, table, map, lengths, causal, scale, false));
}

Tensor bucket_attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& table,
                                 const Tensor& map, const OptTensor& lengths, bool causal, double scale) {
  if (wants_gradient({&q, &k, &v, &table}))
    return BucketAttention::apply(q, k, v, table, map, lengths, causal, scale);
  at::AutoDispatchBelowADInplaceOrView guard;
  return bucket_attention_only(q, k, v, table, map, lengths, causal, scale);
}

struct AddRmsNorm : torch::autograd::Function<AddRmsNorm> {
  // x and weight first: gradients are counted over the tensors that are there
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& residual,
                               double eps) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const bool alone = !has(residual);
    auto [out, summed, inverse] = add_rms_norm(x, residual, weight, eps);
    ctx->saved_data["alone"] = alone;
    ctx->save_for_backward({alone ? x : summed, weight, inverse});
    ctx->set_materialize_grads(false);
    return alone ? variable_list{out} : variable_list{out, summed};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) { return only_first(gradients(ctx, grads)); }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const bool alone = ctx->saved_data["alone"].toBool();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1),
               need_r = !alone && ctx->needs_input_grad(2);
    const Tensor sum = grads.size() > 1 ? grads[1] : Tensor();
    at::AutoDispatchBelowADInplaceOrView guard;
    if (!grads[0].defined())   // only the sum was used, or nothing
      return {need_x ? sum : Tensor(), need_w ? at::zeros_like(saved[1]) : Tensor(), need_r ? sum : Tensor(), Tensor()};
    auto [dx, dw] = add_rms_norm_backward(grads[0].contiguous(), sum.defined() ? OptTensor(sum.contiguous()) : OptTensor(),
                                          saved[0], saved[1], saved[2], need_x || need_r, need_w);
    return {need_x ? dx : Tensor(), need_w ? dw : Tensor(), need_r ? dx : Tensor(), Tensor()};
  }
};

std::vector<Tensor> rms_norm_pair(const Tensor& x, const OptTensor& residual, const Tensor& weight, double eps) {
  auto [out, summed, inverse] = add_rms_norm(x, residual, weight, eps);
  return has(residual) ? std::vector<Tensor>{out, summed} : std::vector<Tensor>{out};
}

std::vector<Tensor> rms_norm_pair_autograd(const Tensor& x, const OptTensor& residual, const Tensor& weight,
                                           double eps) {
  const Tensor other = has(residual) ? *residual : Tensor();
  if (wants_gradient({&x, &weight, &other})) return AddRmsNorm::apply(x, weight, residual, eps);
  at::AutoDispatchBelowADInplaceOrView guard;
  return rms_norm_pair(x, residual, weight, eps);
}

struct AddLayerNorm : torch::autograd::Function<AddLayerNorm> {
  // x and weight first: gradients are counted over the tensors that are there
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const OptTensor& residual,
                               const OptTensor& bias, double eps) {
    at::AutoDispatchBelowADInplaceOrView guard;
    const bool alone = !has(residual);
    auto [out, summed, mean, inverse] = add_layer_norm(x, residual, weight, bias, eps);
    ctx->saved_data["alone"] = alone;
    ctx->saved_data["bias"] = has(bias);
    // 16-bit sums would bring their rounding into the gradients
    const bool sum = !alone && x.scalar_type() == at::kFloat;
    ctx->save_for_backward({sum ? summed : x, alone || sum ? Tensor() : *residual, weight, mean, inverse});
    ctx->set_materialize_grads(false);
    return alone ? variable_list{out} : variable_list{out, summed};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) { return only_first(gradients(ctx, grads)); }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    const bool alone = ctx->saved_data["alone"].toBool(), biased = ctx->saved_data["bias"].toBool();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1),
               need_r = !alone && ctx->needs_input_grad(2), need_b = biased && ctx->needs_input_grad(alone ? 2 : 3);
    const Tensor sum = grads.size() > 1 ? grads[1] : Tensor();
    at::AutoDispatchBelowADInplaceOrView guard;
    if (!grads[0].defined())   // only the sum was used, or nothing
      return {need_x ? sum : Tensor(), need_w ? at::zeros_like(saved[2]) : Tensor(), need_r ? sum : Tensor(),
              need_b ? at::zeros_like(saved[2]) : Tensor(), Tensor()};
    auto [dx, dw, db] = add_layer_norm_backward(
        grads[0].contiguous(), sum.defined() ? OptTensor(sum.contiguous()) : OptTensor(), saved[0],
        saved[1].defined() ? OptTensor(saved[1]) : OptTensor(), saved[2], saved[3], saved[4], need_x || need_r, need_w,
        need_b);
    return {need_x ? dx : Tensor(), need_w ? dw : Tensor(), need_r ? dx : Tensor(), need_b ? db : Tensor(), Tensor()};
  }
};

std::vector<Tensor> layer_norm_pair(const Tensor& x, const OptTensor& residual, const Tensor& weight,
                                    const OptTensor& bias, double eps) {
  auto [out, summed, mean, inverse] = layer_norm(x, residual, weight, bias, eps, false);
  return has(residual) ? std::vector<Tensor>{out, summed} : std::vector<Tensor>{out};
}

std::vector<Tensor> layer_norm_pair_autograd(const Tensor& x, const OptTensor& residual, const Tensor& weight,
                                             const OptTensor& bias, double eps) {
  const Tensor other = has(residual) ? *residual : Tensor(), more = has(bias) ? *bias : Tensor();
  if (wants_gradient({&x, &weight, &other, &more})) return AddLayerNorm::apply(x, weight, residual, bias, eps);
  at::AutoDispatchBelowADInplaceOrView guard;
  return layer_norm_pair(x, residual, weight, bias, eps);
}

struct GatedScan : torch::autograd::Function<GatedScan> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const OptTensor& state,
                               const OptTensor& lengths, bool reverse) {
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [out, last] = gated_scan_forward(x, gate, state, lengths, reverse);
    ctx->saved_data["reverse"] = reverse;
    ctx->saved_data["state"] = has(state);
    ctx->save_for_backward({x, gate, has(state) ? *state : Tensor(), has(lengths) ? *lengths : Tensor(), out});
    ctx->set_materialize_grads(false);
    return {out, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) { return only_first(gradients(ctx, grads)); }
  static variable_list gradients(AutogradContext* ctx, const variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    auto optional = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    const bool need_x = ctx->needs_input_grad(0), need_gate = ctx->needs_input_grad(1),
               need_state = ctx->saved_data["state"].toBool() && ctx->needs_input_grad(2);
    at::AutoDispatchBelowADInplaceOrView guard;
    auto [dx, dgate, dstate] = gated_scan_backward(
        optional(grads[0]), optional(grads[1]), saved[0], saved[1], optional(saved[2]), optional(saved[3]), saved[4],
        ctx->saved_data["reverse"].toBool(), need_x, need_gate, need_state);
    return {need_x ? dx : Tensor(), need_gate ? dgate : Tensor(), need_state ? dstate : Tensor(), Tensor(), Tensor()};
  }
};

std::vector<Tensor> gated_scan(const Tensor& x, const Tensor& gate, const OptTensor& state, const OptTensor& lengths,
                               bool reverse) {
  auto [out, last] = gated_scan_forward(x, gate, state, lengths, reverse);
  return {out, last};
}

std::vector<Tensor> gated_scan_autograd(const Tensor& x, const Tensor& gate, const OptTensor& state,
                                        const OptTensor& lengths, bool reverse) {
  const Tensor first = has(state) ? *state : Tensor();
  if (wants_gradient({&x, &gate, &first})) return GatedScan::apply(x, gate, state, lengths, reverse);
  at::AutoDispatchBelowADInplaceOrView guard;
  return gated_scan(x, gate, state, lengths, reverse);
}

}  // namespace

TORCH_LIBRARY_IMPL(sdk_mapped_ops, AutogradCUDA, m) {
  m.impl("layer_norm_pair", &layer_norm_pair_autograd);
  m.impl("gated_scan", &gated_scan_autograd);
  m.impl("bucket_attention", &bucket_attention_autograd);
  m.impl("rms_norm_pair", &rms_norm_pair_autograd);
}

TORCH_LIBRARY_IMPL(sdk_mapped_ops, CUDA, m) {
  m.impl("bucket_attention", &bucket_attention_only);
  m.impl("rms_norm_pair", &rms_norm_pair);
  m.impl("bucket_attention_forward", &bucket_attention_forward);
  m.impl("bucket_attention_backward", &bucket_attention_backward);
  m.impl("add_rms_norm", &add_rms_norm);
  m.impl("add_rms_norm_quantized", &add_rms_norm_quantized);
  m.impl("add_rms_norm_backward", &add_rms_norm_backward);
  m.impl("dequantize_rows", &dequantize_rows);
  m.impl("adamw_step", &adamw_step);
  m.impl("adamw_step_8bit", &adamw_step_8bit);
  m.impl("adamw_moment_values", &adamw_moment_values);
  m.impl("layer_norm_pair", &layer_norm_pair);
  m.impl("add_layer_norm", &add_layer_norm);
  m.impl("add_layer_norm_backward", &add_layer_norm_backward);
  m.impl("gated_scan", &gated_scan);
  m.impl("gated_scan_forward", &gated_scan_forward);
  m.impl("gated_scan_backward", &gated_scan_backward);
  m.impl("gated_scan_step", &gated_scan_step);
  m.impl("orthogonalize", &orthogonalize);
  m.impl("muon_step", &muon_step);
}

// Names of the operators above, for the Python side (which implements those that are missing here).
extern "C" const char* sdk_torch_token_ops(void) {
  return "bucket_attention,rms_norm_pair,bucket_attention_forward,bucket_attention_backward,add_rms_norm,add_rms_norm_quantized,"
         "add_rms_norm_backward,dequantize_rows,adamw_step,adamw_step_8bit,adamw_moment_values,layer_norm_pair,add_layer_norm,"
         "add_layer_norm_backward,gated_scan,gated_scan_forward,gated_scan_backward,gated_scan_step,orthogonalize,muon_step";
}
