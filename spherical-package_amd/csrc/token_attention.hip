// C entry points of attention with a bias for each bucket of relative positions: checks and argument blocks.
#include <algorithm>
#include <cmath>

#include "token_attention.hpp"

namespace sdk {
namespace token {

Attention on_device(const sdk_bucket_attention* a) {
  Attention d = {};
  d.q = a->query, d.k = a->key, d.v = a->value, d.table = a->bias_table, d.out = a->output, d.grad = a->grad_output;
  d.map = a->bucket_map, d.lengths = a->key_lengths, d.rest = a->dtype == SDK_F32 ? nullptr : a->output_rest;
  d.dq = a->grad_query, d.dk = a->grad_key, d.dv = a->grad_value, d.dtable = a->grad_table, d.lse = a->lse;
  for (int i = 0; i < 3; ++i) {
    d.qs[i] = a->query_strides[i], d.ks[i] = a->key_strides[i], d.vs[i] = a->value_strides[i];
    d.os[i] = a->output_strides[i], d.gs[i] = a->grad_output_strides[i], d.dqs[i] = a->grad_query_strides[i];
    d.dks[i] = a->grad_key_strides[i], d.dvs[i] = a->grad_value_strides[i];
  }
  d.ms[0] = a->map_strides[0], d.ms[1] = a->map_strides[1];
  d.queries = (int)a->queries, d.keys = (int)a->keys, d.batch = (int)a->batch, d.heads = (int)a->heads;
  d.key_heads = (int)a->key_heads, d.dim = (int)a->dim, d.buckets = (int)a->buckets, d.causal = a->causal != 0;
  d.table_float = a->table_dtype == SDK_F32;
  d.scale = (float)a->scale, d.scale2 = (float)(a->scale * 1.4426950408889634);
  d.limit = (float)std::ldexp(1.0, 90 - std::ilogb(a->scale));
  return d;
}

namespace {

int check(const sdk_bucket_attention* a) {
  SDK_REQUIRE(a, "arguments must not be NULL");
  SDK_REQUIRE(known(a->dtype), "unknown dtype %d (float32, bfloat16 and float16 only)", a->dtype);
  SDK_REQUIRE(a->table_dtype == a->dtype || a->table_dtype == SDK_F32,
              "bias_table's dtype %d must be the queries' or float32", a->table_dtype);
  SDK_REQUIRE(a->batch >= 0 && a->queries >= 0 && a->keys >= 0, "batch, queries and keys must not be negative");
  SDK_REQUIRE(a->heads >= 1 && a->key_heads >= 1 && a->heads % a->key_heads == 0,
              "heads = %lld must be a multiple of key_heads = %lld", (long long)a->heads, (long long)a->key_heads);
  SDK_REQUIRE(a->dim >= 8 && a->dim <= 128 && a->dim % 8 == 0, "dim = %lld must be a multiple of 8 up to 128",
              (long long)a->dim);
  SDK_REQUIRE(a->buckets >= 1 && a->buckets <= 256, "buckets = %lld must be between 1 and 256",
              (long long)a->buckets);
  SDK_REQUIRE(a->scale >= 0x1p-32 && a->scale <= 0x1p32, "scale must be between 2^-32 and 2^32");
  // tokens are counted in 32 bits, with room for a tile beyond the last one
  SDK_REQUIRE(a->batch < 65536 && a->heads < 1 << 20 && a->queries < 1 << 30 && a->keys < 1 << 30,
              "a batch of 65536 or more, 2^20 heads or 2^30 tokens");
  SDK_REQUIRE(ceil_div(a->queries, 64) * ceil_div(a->keys, 64) < (int64_t)1 << 31, "a map of 2^43 pairs or more");
  const int64_t groups = a->batch * a->heads * std::max(ceil_div(a->queries, 128), ceil_div(a->keys, 128));
  SDK_REQUIRE(groups < (int64_t)1 << 24, "%lld tiles of 128 tokens are too many", (long long)groups);
  return SDK_OK;
}

int check_rows(const char* name, const void* p, const int64_t* strides, int dtype) {
  SDK_REQUIRE(p, "%s must not be NULL", name);
  bool ok = aligned16(p);
  for (int i = 0; i < 3; ++i) ok = ok && strides[i] % (16 / (int64_t)bytes_of(dtype)) == 0;
  SDK_REQUIRE(ok, "rows of %s must be 16-byte aligned", name);
  SDK_REQUIRE(strides[2] >= 0 && strides[2] * 64 * (int64_t)bytes_of(dtype) < (int64_t)1 << 31,
              "the tokens of %s lie %lld elements apart: too far", name, (long long)strides[2]);
  return SDK_OK;
}

int check_inputs(const sdk_bucket_attention* a) {
  if (int rc = check_rows("query", a->query, a->query_strides, a->dtype)) return rc;
  if (int rc = check_rows("output", a->output, a->output_strides, a->dtype)) return rc;
  if (a->output_rest)
    if (int rc = check_rows("output_rest", a->output_rest, a->output_strides, a->dtype)) return rc;
  SDK_REQUIRE(a->bias_table, "bias_table must not be NULL");
  if (a->keys == 0) return SDK_OK;
  if (int rc = check_rows("key", a->key, a->key_strides, a->dtype)) return rc;
  if (int rc = check_rows("value", a->value, a->value_strides, a->dtype)) return rc;
  SDK_REQUIRE(a->bucket_map, "bucket_map must not be NULL");
  return SDK_OK;
}

int check_workspace(size_t need, const void* workspace, size_t bytes) {
  if (need && (!workspace || bytes < need))
    return fail(SDK_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", bytes, need);
  return SDK_OK;
}

}  // namespace
}  // namespace token
}  // namespace sdk

using namespace sdk;
using namespace sdk::token;

extern "C" {

size_t sdk_bucket_attention_workspace_bytes(const sdk_bucket_attention* a, int32_t backward) {
  if (check(a) != SDK_OK || a->batch == 0) return 0;
  if (backward) return backward_bytes(a);
  if (a->queries == 0) return 0;
  const int splits = forward_splits(a);
  return splits == 1 ? 0 : (size_t)splits * a->batch * a->heads * a->queries * (a->dim + 2) * sizeof(float);
}

int sdk_bucket_attention_forward(const sdk_bucket_attention* a, void* workspace, size_t workspace_bytes,
                                 sdk_stream_t stream) {
  if (int rc = check(a)) return rc;
  if (a->batch == 0 || a->queries == 0) return SDK_OK;
  if (int rc = check_inputs(a)) return rc;
  if (int rc = check_workspace(sdk_bucket_attention_workspace_bytes(a, 0), workspace, workspace_bytes)) return rc;
  return run_forward(a, workspace, (hipStream_t)stream);
}

int sdk_bucket_attention_backward(const sdk_bucket_attention* a, void* workspace, size_t workspace_bytes,
                                  sdk_stream_t stream) {
  if (int rc = check(a)) return rc;
  const bool any = a->batch > 0 && a->queries > 0, keys = a->batch > 0 && a->keys > 0;
  if (any) {
    if (int rc = check_inputs(a)) return rc;
    if (int rc = check_rows("grad_output", a->grad_output, a->grad_output_strides, a->dtype)) return rc;
    SDK_REQUIRE(a->lse, "lse must not be NULL");
  }
  if (a->grad_query && any)
    if (int rc = check_rows("grad_query", a->grad_query, a->grad_query_strides, a->dtype)) return rc;
  if (a->grad_key && keys)
    if (int rc = check_rows("grad_key", a->grad_key, a->grad_key_strides, a->dtype)) return rc;
  if (a->grad_value && keys)
    if (int rc = check_rows("grad_value", a->grad_value, a->grad_value_strides, a->dtype)) return rc;
  if (int rc = check_workspace(sdk_bucket_attention_workspace_bytes(a, 1), workspace, workspace_bytes)) return rc;
  return run_backward(a, workspace, (hipStream_t)stream);
}

}  // extern "C"
