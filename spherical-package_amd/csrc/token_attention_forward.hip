// Forward of attention with a bias for each bucket of relative positions (token_attention.hpp: operands and tiles).
//
//   s_ij = scale q_i k_j + T[head][map_ij]      o_i = sum_j exp(s_ij - lse_i) v_j
//
// The scores are never written: the running maximum and sum of each query stay in the registers of the lane that
// holds it.
#include "token_attention.hpp"

namespace sdk {
namespace token {
namespace {

__device__ __forceinline__ void put_lse(float* to, int64_t rows, int64_t row, float2 lse) {
  to[row] = lse.x;
  to[rows + row] = lse.y;
}

// ------------------------------------------------------------------------------------------ many queries
// A workgroup takes 128 queries of a head and walks the keys, 32 queries a wave: S^T = K Q^T has the queries in
// columns, so a query's maximum and sum are one lane's (and the lane's 32 further on).  The next tile is requested
// while this one is worked on; with two buffers a step has one barrier.
// Bound by the vector instructions (a lookup's address, fma, exp2, half a conversion and half a sum a pair) beside the
// matrix ones, which overlap by half: 4608 x 4608 pairs of 2 x 16 heads of 64 in bfloat16 take 264 us, 660 TFLOP/s.  32
// queries a wave rather than 64: 1152 workgroups balance over 256 CUs, 576 do not.
// splits > 1: each takes a part of the keys and leaves its normalised output and log2 of its sum (two numbers) for `join`.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads, 2) void attend(const Attention a, int splits, int tiles, float* part_out,
                                                      float* part_lse) {
  constexpr int NT = kParts<T>, KEYS = 32 * NT;
  constexpr int BUFFERS = sizeof(Tile<T, DP, NT>) * 4 <= 72 << 10 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) struct {
    float table[kTable];   // at address zero: a lookup's address is four times the bucket
    Tile<T, DP, NT> keys[BUFFERS], values[BUFFERS];
  } lds;
  auto &table = lds.table;
  auto &keys = lds.keys, &values = lds.values;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, h = lane / 32;
  const Work work(tiles, a.batch * a.heads, splits, a.causal, false);
  const int head = work.head % a.heads, b = work.head / a.heads;
  const int shared_head = head / (a.heads / a.key_heads);
  const T* kp = (const T*)a.k + b * a.ks[0] + shared_head * a.ks[1];
  const T* vp = (const T*)a.v + b * a.vs[0] + shared_head * a.vs[1];
  table[threadIdx.x] = a.bias(head, threadIdx.x, __is_same(T, bf16));

  const int first = work.tile * (32 * kWaves), query = first + wave * 32 + lane % 32;
  const int len = a.length(b), shift = len - a.queries;
  // keys that some query of the workgroup sees
  const int end = a.causal ? std::min(len, std::min(first + 32 * kWaves, a.queries) + shift) : len;
  const int blocks = end > 0 ? (end + KEYS - 1) / KEYS : 0;
  const int from = split_at(blocks, work.split, splits) * KEYS;
  const int to = std::min(end, split_at(blocks, work.split + 1, splits) * KEYS);
  const int clamped = std::min(query, a.queries - 1);
  const uint8_t* map = a.map + b * a.ms[0] + clamped * a.ms[1];
  const int last = a.causal ? std::min(len - 1, clamped + shift) : len - 1;   // this lane's last key

  Operand<T> q[DP / 16];
  load_columns<T, DP>(q, (const T*)a.q + b * a.qs[0] + head * a.qs[1], a.qs[2], query, query < a.queries, a.dim, lane);
  floatx16 o[DP / 32];
  clear(o);
  // level (lse_of): common to both halves, off: the same, 0 where there is none; sum: of this lane's keys
  float level = -INFINITY, off = 0.f, sum = 0.f;

  Carry<T, DP, NT, kThreads> next_k(a.ks[2], a.dim), next_v(a.vs[2], a.dim);
  Buckets bucket[NT], next_bucket[NT];
  auto request = [&](int k0) {
    next_k.load(kp + k0 * a.ks[2], a.ks[2], to - k0, a.dim);
    next_v.load(vp + k0 * a.vs[2], a.vs[2], to - k0, a.dim);
    load_buckets<NT>(next_bucket, map, k0, a.keys, h);
  };
  if (from < to) {
    request(from);
    if (BUFFERS == 2) {
      next_k.store(keys[0]);
      next_v.store(values[0]);
    }
  }
  landed();
  if (BUFFERS == 2) __syncthreads();
  int now_in = 0;
  bool first_tile = true;
  for (int k0 = from; k0 < to; k0 += KEYS) {
    if (BUFFERS == 1) {
      __syncthreads();
      next_k.store(keys[0]);
      next_v.store(values[0]);
      __syncthreads();
    }
    const auto key_view = keys[now_in].view(lane), value_view = values[now_in].view(lane);
#pragma unroll
    for (int t = 0; t < NT; ++t) bucket[t] = next_bucket[t];
    // Beyond the last tile nothing is read.  With two buffers it has landed when it is stored: until then no load is
    // waited for.
    request(k0 + KEYS);
    floatx16 s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
      s[t] = dot_tile<T, DP>(key_view, t, q, [&](int v) { return table[bucket[t][v]]; });
    if (k0 + KEYS > last + 1) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (k0 + 16 * NT * h + 16 * t + v > last) s[t][v] = -INFINITY;
    }
    // The weights go to the matrix unit in the inputs' type, and are summed as rounded: an output's error beside 64 bits
    // is 2.3e-3 of its size in bfloat16, 1.7e-3 of it the output's own rounding, and 2.8e-4 for 2.1e-4 in float16.  In
    // two pieces each, which leaves the output's rounding alone, 4608 x 4608 pairs take 361 us for 264.
    // The weights against the level so far.  It is raised only where they would pass 2^10 in sum (and by the first
    // tile), so that most tiles need no maximum.
    Operand<T> w[NT][2];
    float with = sum;
    auto weigh = [&] {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float p[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[t][8 * half + i], a.scale2, -off));
          w[t][half] = rounded<T>(p);
          with = add_weights<T>(w[t][half], p, with);
        }
    };
    if (!first_tile) weigh();
    if (first_tile || __any(with - sum > 0x1p10f)) {
      float top = s[0][0];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) top = fmaxf(top, s[t][v]);
      const float grown = fmaxf(ceilf(max_halves(top) * a.scale2), level);
      const float by = grown == -INFINITY ? 1.f : exp2f(level - grown);
      level = grown;
      off = grown == -INFINITY ? 0.f : grown;
      first_tile = __any(grown == -INFINITY);   // a query without pairs so far has no level yet
      sum *= by;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= by;
      with = sum;
      weigh();
    }
    sum = with;
#pragma unroll
    for (int t = 0; t < NT; ++t) add_columns<T>(o, value_view, t, w[t]);
    if (BUFFERS == 2) {
      now_in ^= 1;
      next_k.store(keys[now_in]);
      next_v.store(values[now_in]);
      __syncthreads();
    }
  }
  sum += other_half(sum);
  if (query >= a.queries) return;
  const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const float2 lse = lse_of(off, sum);
  const int64_t row = (int64_t)work.head * a.queries + query;
  if (splits > 1) {
    const int64_t rows = (int64_t)a.batch * a.heads * a.queries;
    store_columns<float, DP>(part_out + work.split * rows * a.dim, a.dim, row, a.dim, lane, o, by);
    if (h == 0) put_lse(part_lse + work.split * 2 * rows, rows, row, lse);
    return;
  }
  const int64_t at = b * a.os[0] + head * a.os[1];
  store_output<T, DP>((T*)a.out + at, a.rest ? (T*)a.rest + at : nullptr, a.os[2], query, a.dim, lane, o, by);
  if (a.lse && h == 0) put_lse(a.lse, (int64_t)a.batch * a.heads * a.queries, row, lse);
}

// ------------------------------------------------------------------------------------------ few queries
// At most 32 rows (a key head's query heads times the queries) against many keys: bound by reading the keys and
// values once.  A workgroup takes a part of one key head's keys for all of its rows; its waves walk 32 keys each
// by themselves, without barriers: keys go from memory into the product's registers, values through the wave's
// own tile in LDS, both requested a step ahead.  The waves' states are joined in LDS at the end.  16 sequences of up to
// 16384 keys, 8 key heads of 128 in bfloat16: 154 us, 5.3 TB/s (the other kernel with parts of the keys: 870 us, each
// query head reading the keys for itself).
template <typename T, int DP>
__global__ __launch_bounds__(kThreads, sizeof(T) == 4 && DP > 64 ? 1 : 2) void attend_few(
    const Attention a, int splits, float* part_out, float* part_lse) {
  constexpr int kVectors = DP / kWide<T>, kCount = 32 * kVectors / 64;
  constexpr int kState = 2 * 32 * (DP + 1);   // floats of two waves' states
  __shared__ __attribute__((aligned(16))) union {
    Tile<T, DP, 1> values[kWaves];
    float state[kState];
  } lds;
  __shared__ float level[kWaves / 2][2][32];
  extern __shared__ float table[];   // [query head of the key head][257]: equal buckets of two heads in two banks
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, h = lane / 32;
  const unsigned id = by_die(blockIdx.x, gridDim.x);
  const int split = (int)(id % (unsigned)splits);
  const unsigned bh = id / (unsigned)splits;
  const int shared_head = (int)(bh % (unsigned)a.key_heads), b = (int)(bh / (unsigned)a.key_heads);
  const int group = a.heads / a.key_heads, rows = group * a.queries;
  const int r = std::min(lane % 32, rows - 1), head = shared_head * group + r / a.queries;
  const int query = r % a.queries;
  for (int i = threadIdx.x; i < group * kTable; i += kThreads)
    table[i / kTable * (kTable + 1) + i % kTable] =
        a.bias(shared_head * group + i / kTable, i % kTable, __is_same(T, bf16));
  const float* bias = table + r / a.queries * (kTable + 1);
  const T* kp = (const T*)a.k + b * a.ks[0] + shared_head * a.ks[1];
  const T* vp = (const T*)a.v + b * a.vs[0] + shared_head * a.vs[1];
  const int len = a.length(b), last = a.causal ? len - a.queries + query : len - 1;
  const int blocks = (len + 31) / 32;
  const int from = split_at(blocks, split, splits) * 32, to = std::min(len, split_at(blocks, split + 1, splits) * 32);
  const uint8_t* map = a.map + b * a.ms[0] + query * a.ms[1];
  // the token whose key this lane supplies: row lane % 32 of the product
  const int token = 16 * (lane / 4 % 2) + 4 * (lane % 32 / 8) + lane % 4;

  Operand<T> q[DP / 16];
  load_columns<T, DP>(q, (const T*)a.q + b * a.qs[0] + head * a.qs[1], a.qs[2], query, true, a.dim, lane);
  floatx16 o[DP / 32];
  clear(o);
  float most = -INFINITY, sum = 0.f;   // level and sum (lse_of)
  __syncthreads();

  // the keys in registers as dot_tile asks for them
  struct Held {
    const Operand<T> (&k)[DP / 16];
    __device__ __forceinline__ const Operand<T>& rows(int, int c) const { return k[c]; }
    __device__ __forceinline__ Operand<bf16> first_piece(int, int c) const {
      if constexpr (sizeof(T) == 4)
        return k[c].piece[0];
      else
        return {};
    }
  };
  Operand<T> k[DP / 16];
  Pack<T, kWide<T>> x[kCount];
  Buckets bucket[1];
  auto request = [&](int k0) {
    load_columns<T, DP>(k, kp, a.ks[2], k0 + token, k0 + token < to, a.dim, lane);
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int at = n * 64 + lane, d = at % kVectors * kWide<T>;
      const int row = k0 + at / kVectors;
      if (row < to && d < a.dim) {
        x[n] = *reinterpret_cast<const Pack<T, kWide<T>>*>(vp + row * a.vs[2] + d);
      } else {
#pragma unroll
        for (int e = 0; e < kWide<T>; ++e) x[n].v[e] = (T)0.f;
      }
    }
    load_buckets<1>(bucket, map, k0, a.keys, h);
  };
  Tile<T, DP, 1>& values = lds.values[wave];
  const auto value_view = values.view(lane);
  int k0 = from + 32 * wave;
  if (k0 < to) request(k0);
  for (; k0 < to; k0 += 32 * kWaves) {
    const Held view = {k};
    floatx16 s = dot_tile<T, DP>(view, 0, q, [&](int v) { return bias[bucket[0][v]]; });
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int at = n * 64 + lane;
      values.store(at / kVectors, at % kVectors * kWide<T>, x[n]);
    }
    if (k0 + 32 * kWaves < to) request(k0 + 32 * kWaves);
    if (k0 + 32 > last + 1) {
#pragma unroll
      for (int v = 0; v < 16; ++v)
        if (k0 + 16 * h + v > last) s[v] = -INFINITY;
    }
    float now = s[0];
#pragma unroll
    for (int v = 1; v < 16; ++v) now = fmaxf(now, s[v]);
    now = max_halves(now);
    now = ceilf(now * a.scale2);
    if (__any(now > most)) {
      const float grown = fmaxf(now, most);
      const float by = grown == -INFINITY ? 1.f : exp2f(most - grown);
      most = grown;
      sum *= by;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= by;
    }
    const float off = most == -INFINITY ? 0.f : most;
    float p[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) p[v] = __builtin_amdgcn_exp2f(fmaf(s[v], a.scale2, -off));
    wave_order();
    const Operand<T> w[2] = {rounded<T>(p), rounded<T>(p + 8)};
    sum = add_weights<T>(w[1], p + 8, add_weights<T>(w[0], p, sum));
    add_columns<T>(o, value_view, 0, w);
    wave_order();
  }
  sum += other_half(sum);
  // waves 2 and 3 hand their states to 0 and 1, then 1 to 0
#pragma unroll
  for (int step = kWaves / 2; step > 0; step /= 2) {
    __syncthreads();
    const int slot = wave % step;
    float* state = lds.state + slot * 32 * (DP + 1) + lane % 32 * (DP + 1);   // DP + 1: columns in other banks
    if (wave >= step && wave < 2 * step) {
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) state[32 * d + 8 * (v / 4) + 4 * h + v % 4] = o[d][v];
      level[slot][0][lane % 32] = most;
      level[slot][1][lane % 32] = sum;
    }
    __syncthreads();
    if (wave < step) {
      const float other = level[slot][0][lane % 32], grown = fmaxf(most, other);
      const float mine = grown == -INFINITY ? 1.f : exp2f(most - grown);
      const float theirs = grown == -INFINITY ? 1.f : exp2f(other - grown);
      most = grown;
      sum = sum * mine + level[slot][1][lane % 32] * theirs;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          o[d][v] = o[d][v] * mine + state[32 * d + 8 * (v / 4) + 4 * h + v % 4] * theirs;
    }
  }
  if (wave != 0 || lane % 32 >= rows) return;
  const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const float2 lse = lse_of(most, sum);
  const int64_t row = ((int64_t)b * a.heads + head) * a.queries + query;
  if (splits > 1) {
    const int64_t all = (int64_t)a.batch * a.heads * a.queries;
    store_columns<float, DP>(part_out + split * all * a.dim, a.dim, row, a.dim, lane, o, by);
    if (h == 0) put_lse(part_lse + split * 2 * all, all, row, lse);
    return;
  }
  const int64_t at = b * a.os[0] + head * a.os[1];
  store_output<T, DP>((T*)a.out + at, a.rest ? (T*)a.rest + at : nullptr, a.os[2], query, a.dim, lane, o, by);
  if (a.lse && h == 0) put_lse(a.lse, (int64_t)a.batch * a.heads * a.queries, row, lse);
}

// The splits of a row: weights 2^(lse2 - largest); four values a thread.
template <typename T>
__global__ __launch_bounds__(256) void join(const Attention a, int splits, const float* part_out,
                                            const float* part_lse) {
  const int per_row = a.dim / 4;
  const int64_t rows = (int64_t)a.batch * a.heads * a.queries, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / per_row;
  if (row >= rows) return;
  const int d = (int)(i % per_row) * 4;
  float most = -INFINITY;
  for (int s = 0; s < splits; ++s) most = Largest::of(most, part_lse[s * 2 * rows + row]);
  const float off = most == -INFINITY ? 0.f : most;
  float sum = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) {
    const float* lse = part_lse + s * 2 * rows + row;
    const float w = __builtin_amdgcn_exp2f((lse[0] - off) + lse[rows]);
    float y[4];
    load_pack<float, 4>(part_out + (s * rows + row) * a.dim + d, y);
    sum += w;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += w * y[e];
  }
  const int64_t query = row % a.queries, bh = row / a.queries;
  const int head = (int)(bh % a.heads), b = (int)(bh / a.heads);
  const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] *= by;
  const int64_t at = b * a.os[0] + head * a.os[1] + query * a.os[2] + d;
  store_pack<T, 4>((T*)a.out + at, x);
  if (a.rest) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] -= (float)(T)x[e];
    store_pack<T, 4>((T*)a.rest + at, x);
  }
  if (a.lse && d == 0) put_lse(a.lse, rows, row, lse_of(off, sum));
}

}  // namespace

bool few_rows(const sdk_bucket_attention* a) { return a->heads / a->key_heads * a->queries <= 32; }

// Parts that the keys are dealt to.  Few queries: two workgroups a CU, at least 256 keys each.
int forward_splits(const sdk_bucket_attention* a) {
  if (few_rows(a)) {
    const int64_t groups = a->batch * a->key_heads;
    if (groups >= 512 || groups == 0) return 1;
    return (int)std::max<int64_t>(1, std::min(ceil_div(512, groups), a->keys / 256));
  }
  const int64_t groups = a->batch * a->heads * ceil_div(a->queries, 32 * kWaves);
  const int64_t slots = a->dim <= 64 && a->dtype != SDK_F32 ? 768 : 512;   // by the registers of their waves
  return parts_of(groups, ceil_div(a->keys, 32 * (a->dtype == SDK_F32 ? kParts<float> : kParts<bf16>)), slots, false);
}

int run_forward(const sdk_bucket_attention* a, void* workspace, hipStream_t s) {
  const Attention d = on_device(a);
  const int splits = forward_splits(a), tiles = (int)ceil_div(a->queries, 32 * kWaves);
  const int64_t rows = a->batch * a->heads * a->queries;
  float* part_out = (float*)workspace;
  float* part_lse = part_out ? part_out + splits * rows * a->dim : nullptr;
  SDK_DISPATCH_TOKEN_DTYPE(a->dtype, {
    if (few_rows(a)) {
      const int group = d.heads / d.key_heads;
      ATTENTION_DIM(a->dim, {
        attend_few<T, DP><<<dim3((unsigned)(a->batch * a->key_heads) * splits), dim3(kThreads),
                            group*(kTable + 1) * sizeof(float), s>>>(d, splits, part_out, part_lse);
      });
    } else
      ATTENTION_DIM(a->dim, launch(attend<T, DP>, dim3((unsigned)(tiles * a->batch * a->heads) * splits),
                                   dim3(kThreads), s, d, splits, tiles, part_out, part_lse));
    if (splits > 1)
      launch(join<T>, dim3((unsigned)ceil_div(rows * (a->dim / 4), 256)), dim3(256), s, d, splits, (const float*)part_out,
             (const float*)part_lse);
  });
  SDK_LAUNCH_CHECK("bucket_attention_forward");
  return SDK_OK;
}

}  // namespace token
}  // namespace sdk
