// Attention with a learned bias for each bucket of relative positions: forward, backward, and the few queries of
// serving.
//
//   s_ij = scale q_i k_j + T[head][map_ij]      p_ij = exp(s_ij - lse_i)      o_i = sum_j p_ij v_j
//   D_i = <do_i, o_i>      ds_ij = p_ij (<do_i, v_j> - D_i)
//   dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i      dv_j = sum_i p_ij do_i
//   dT[head][b] = sum of ds_ij over the pairs of bucket b
//
// The scores are never written: the forward keeps the running maximum and sum of each query in the registers of
// the lane that holds it, the backward forms them again from the lse.
#include <algorithm>
#include <cmath>

#include "token_attention.hpp"

namespace sdk {
namespace token {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kTable = 256;

template <typename T>
constexpr int kParts = sizeof(T) == 4 ? 1 : 2;   // 32-token parts of a tile

// Waves of a SIMD in the backward: with two, accumulators lie among the 256 registers of a wave.
template <int DP>
constexpr int kBackwardWaves = DP <= 64 ? 2 : 1;

// A wave's 32 columns of B: rows first + lane % 32 of a tensor, values 16 c + 8 h .. + 7 in operand c; rows at or
// beyond `end` are zeros.
template <typename T, int DP>
__device__ __forceinline__ void load_columns(Operand<T> (&x)[DP / 16], const T* base, int64_t stride, int64_t row,
                                             int64_t end, int dim, int lane) {
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
    const int d = 16 * c + 8 * (lane / 32);
    x[c] = row < end && d < dim ? load_operand<T>(base + row * stride + d) : zeros<T>();
  }
}

// The wave's accumulators D[value 32 d + ..][column] to row `row` of a tensor, times `by`.
template <typename T, int DP>
__device__ __forceinline__ void store_columns(T* base, int64_t stride, int64_t row, int dim, int lane,
                                              const floatx16 (&acc)[DP / 32], float by) {
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const int at = 32 * d + 8 * a + 4 * (lane / 32);
      if (at < dim) {
        const float f[4] = {acc[d][4 * a] * by, acc[d][4 * a + 1] * by, acc[d][4 * a + 2] * by,
                            acc[d][4 * a + 3] * by};
        store_pack<T, 4>(base + row * stride + at, f);
      }
    }
}

// Between a wave's writes to LDS and its other lanes' reads: LDS keeps a wave's order, so it is the compiler alone
// that must not exchange them.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Where split `split` of `splits` begins among `tiles`.
__device__ __forceinline__ int64_t split_at(int64_t tiles, int split, int splits) { return tiles * split / splits; }

// ------------------------------------------------------------------------------------------ forward
// A workgroup takes 128 queries of a head and walks the keys, 32 queries a wave: S^T = K Q^T has the queries in
// columns, so a query's maximum and sum are one lane's (and the lane's 32 further on).
// splits > 1: each takes a part of the keys and leaves its normalised output and log2 of its sum for `join`.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads, 2) void attend(const Attention a, int splits, unsigned tiles, float* part_out,
                                                   float* part_lse) {
  constexpr int NT = kParts<T>, KEYS = 32 * NT;
  __shared__ __attribute__((aligned(16))) Tile<T, DP, NT> keys, values;
  __shared__ float table[kTable];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, h = lane / 32;
  const unsigned id = by_die(blockIdx.x, gridDim.x);
  const int split = (int)(id % (unsigned)splits);
  const unsigned tile = id / (unsigned)splits % tiles, bh = id / (unsigned)splits / tiles;
  const int head = (int)(bh % (unsigned)a.heads), b = (int)(bh / (unsigned)a.heads);
  const int shared_head = head / (a.heads / a.key_heads);
  const T* kp = (const T*)a.k + b * a.ks[0] + shared_head * a.ks[1];
  const T* vp = (const T*)a.v + b * a.vs[0] + shared_head * a.vs[1];
  table[threadIdx.x] = a.bias(head, threadIdx.x, __is_same(T, bf16));

  const int64_t first = (int64_t)tile * (32 * kWaves), query = first + wave * 32 + lane % 32;
  const int64_t len = a.length(b), shift = len - a.queries;
  // keys that some query of the workgroup sees
  int64_t end = len;
  if (a.causal) end = std::min(end, std::min(first + 32 * kWaves, a.queries) + shift);
  const int64_t blocks = end > 0 ? (end + KEYS - 1) / KEYS : 0;
  const int64_t from = split_at(blocks, split, splits) * KEYS, to = std::min(end, split_at(blocks, split + 1, splits) * KEYS);
  const int64_t clamped = std::min(query, a.queries - 1);
  const uint8_t* map = a.map + b * a.ms[0] + clamped * a.ms[1];
  const int64_t last = a.causal ? std::min(len - 1, clamped + shift) : len - 1;   // this lane's last key

  Operand<T> q[DP / 16];
  load_columns<T, DP>(q, (const T*)a.q + b * a.qs[0] + head * a.qs[1], a.qs[2], query, a.queries, a.dim, lane);
  floatx16 o[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.f;
  float most = -INFINITY, sum = 0.f;   // of this lane's keys: `most` is common to both halves, `sum` is not

  Carry<T, DP, NT, kThreads> next_k, next_v;
  Buckets bucket[NT];
  next_k.load(kp, a.ks[2], from, to, a.dim);
  next_v.load(vp, a.vs[2], from, to, a.dim);
  for (int64_t k0 = from; k0 < to; k0 += KEYS) {
#pragma unroll
    for (int t = 0; t < NT; ++t) bucket[t].load(map, k0 + 16 * NT * h + 16 * t, a.keys);
    __syncthreads();
    next_k.store(keys);
    next_v.store(values);
    __syncthreads();
    if (k0 + KEYS < to) {
      next_k.load(kp, a.ks[2], k0 + KEYS, to, a.dim);
      next_v.load(vp, a.vs[2], k0 + KEYS, to, a.dim);
    }
    floatx16 s[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) s[t][v] = table[bucket[t][v]];
#pragma unroll
    for (int c = 0; c < DP / 16; ++c)
#pragma unroll
      for (int t = 0; t < NT; ++t) s[t] = product(keys.rows(t, c, lane), q[c], s[t]);
    if (k0 + KEYS > last + 1) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (k0 + 16 * NT * h + 16 * t + v > last) s[t][v] = -INFINITY;
    }
    float now = s[0][0];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) now = fmaxf(now, s[t][v]);
    now = fmaxf(now, other_half(now));
    if (__any(now > most)) {
      const float grown = fmaxf(now, most);
      const float by = grown == -INFINITY ? 1.f : exp2f((most - grown) * a.scale2);
      most = grown;
      sum *= by;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= by;
    }
    const float off = most == -INFINITY ? 0.f : most * a.scale2;
    float p[NT][16];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        p[t][v] = __builtin_amdgcn_exp2f(fmaf(s[t][v], a.scale2, -off));
        sum += p[t][v];
      }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const Operand<T> w = rounded<T>(p[t] + 8 * half);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) o[d] = product(values.columns(t, half, d, lane), w, o[d]);
      }
  }
  sum += other_half(sum);
  if (query >= a.queries) return;
  const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  const float lse2 = sum > 0.f || sum != sum ? fmaf(most, a.scale2, log2f(sum)) : -INFINITY;
  const int64_t row = ((int64_t)b * a.heads + head) * a.queries + query;
  if (splits > 1) {
    const int64_t rows = (int64_t)a.batch * a.heads * a.queries;
    store_columns<float, DP>(part_out + split * rows * a.dim, a.dim, row, a.dim, lane, o, by);
    if (h == 0) part_lse[split * rows + row] = lse2;
    return;
  }
  store_columns<T, DP>((T*)a.out + b * a.os[0] + head * a.os[1], a.os[2], query, a.dim, lane, o, by);
  if (a.lse && h == 0) a.lse[row] = lse2;
}

// ------------------------------------------------------------------------------------------ few queries
// At most 32 rows (a key head's query heads times the queries) against many keys: bound by reading the keys and
// values once.  A workgroup takes a part of one key head's keys for all of its rows; its waves walk 32 keys each
// by themselves, without barriers: keys go from memory into the product's registers, values through the wave's
// own tile in LDS, both requested a step ahead.  The waves' states are joined in LDS at the end.
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
  const int group = a.heads / a.key_heads, rows = group * (int)a.queries;
  const int r = std::min(lane % 32, rows - 1), head = shared_head * group + r / (int)a.queries;
  const int64_t query = r % (int)a.queries;
  for (int i = threadIdx.x; i < group * kTable; i += kThreads)
    table[i / kTable * (kTable + 1) + i % kTable] =
        a.bias(shared_head * group + i / kTable, i % kTable, __is_same(T, bf16));
  const float* bias = table + r / (int)a.queries * (kTable + 1);
  const T* kp = (const T*)a.k + b * a.ks[0] + shared_head * a.ks[1];
  const T* vp = (const T*)a.v + b * a.vs[0] + shared_head * a.vs[1];
  const int64_t len = a.length(b);
  const int64_t last = a.causal ? len - a.queries + query : len - 1;
  const int64_t blocks = (len + 31) / 32;
  const int64_t from = split_at(blocks, split, splits) * 32, to = std::min(len, split_at(blocks, split + 1, splits) * 32);
  const uint8_t* map = a.map + b * a.ms[0] + query * a.ms[1];
  // the token whose key this lane supplies: row lane % 32 of the product
  const int token = 16 * (lane / 4 % 2) + 4 * (lane % 32 / 8) + lane % 4;

  Operand<T> q[DP / 16];
  load_columns<T, DP>(q, (const T*)a.q + b * a.qs[0] + head * a.qs[1], a.qs[2], query, a.queries, a.dim, lane);
  floatx16 o[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.f;
  float most = -INFINITY, sum = 0.f;
  __syncthreads();

  Operand<T> k[DP / 16];
  Pack<T, kWide<T>> x[kCount];
  Buckets bucket;
  auto request = [&](int64_t k0) {
    load_columns<T, DP>(k, kp, a.ks[2], k0 + token, to, a.dim, lane);
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int at = n * 64 + lane, d = at % kVectors * kWide<T>;
      const int64_t row = k0 + at / kVectors;
      if (row < to && d < a.dim) {
        x[n] = *reinterpret_cast<const Pack<T, kWide<T>>*>(vp + row * a.vs[2] + d);
      } else {
#pragma unroll
        for (int e = 0; e < kWide<T>; ++e) x[n].v[e] = (T)0.f;
      }
    }
    bucket.load(map, k0 + 16 * h, a.keys);
  };
  Tile<T, DP, 1>& values = lds.values[wave];
  int64_t k0 = from + 32 * wave;
  if (k0 < to) request(k0);
  for (; k0 < to; k0 += 32 * kWaves) {
    floatx16 s;
#pragma unroll
    for (int v = 0; v < 16; ++v) s[v] = bias[bucket[v]];
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) s = product(k[c], q[c], s);
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int at = n * 64 + lane;
      *reinterpret_cast<Pack<T, kWide<T>>*>(
          &values.v[row_of<1>(at / kVectors) * Tile<T, DP, 1>::kStride + at % kVectors * kWide<T>]) = x[n];
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
    now = fmaxf(now, other_half(now));
    if (__any(now > most)) {
      const float grown = fmaxf(now, most);
      const float by = grown == -INFINITY ? 1.f : exp2f((most - grown) * a.scale2);
      most = grown;
      sum *= by;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= by;
    }
    const float off = most == -INFINITY ? 0.f : most * a.scale2;
    float p[16];
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      p[v] = __builtin_amdgcn_exp2f(fmaf(s[v], a.scale2, -off));
      sum += p[v];
    }
    wave_order();
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const Operand<T> w = rounded<T>(p + 8 * half);
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) o[d] = product(values.columns(0, half, d, lane), w, o[d]);
    }
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
      const float mine = grown == -INFINITY ? 1.f : exp2f((most - grown) * a.scale2);
      const float theirs = grown == -INFINITY ? 1.f : exp2f((other - grown) * a.scale2);
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
  const float lse2 = sum > 0.f || sum != sum ? fmaf(most, a.scale2, log2f(sum)) : -INFINITY;
  const int64_t row = ((int64_t)b * a.heads + head) * a.queries + query;
  if (splits > 1) {
    const int64_t all = (int64_t)a.batch * a.heads * a.queries;
    store_columns<float, DP>(part_out + split * all * a.dim, a.dim, row, a.dim, lane, o, by);
    if (h == 0) part_lse[split * all + row] = lse2;
    return;
  }
  store_columns<T, DP>((T*)a.out + b * a.os[0] + head * a.os[1], a.os[2], query, a.dim, lane, o, by);
  if (a.lse && h == 0) a.lse[row] = lse2;
}

// The splits of a row: weights 2^(lse2 - largest), a wave a row.
template <typename T>
__global__ __launch_bounds__(256) void join(const Attention a, int splits, const float* part_out,
                                            const float* part_lse) {
  const int lane = threadIdx.x % 64;
  const int64_t rows = (int64_t)a.batch * a.heads * a.queries, row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (row >= rows) return;
  float most = -INFINITY;
  for (int s = lane; s < splits; s += 64) most = fmaxf(most, part_lse[s * rows + row]);
  most = over_wave<Largest>(most);
  const float off = most == -INFINITY ? 0.f : most;
  float sum = 0.f, x[2] = {0.f, 0.f};
  const int d = 2 * lane;
  for (int s = 0; s < splits; ++s) {
    const float w = __builtin_amdgcn_exp2f(part_lse[s * rows + row] - off);
    sum += w;
    if (d < a.dim) {
      const float2 f = *reinterpret_cast<const float2*>(part_out + (s * rows + row) * a.dim + d);
      x[0] += w * f.x;
      x[1] += w * f.y;
    }
  }
  const int64_t query = row % a.queries, bh = row / a.queries;
  const int head = (int)(bh % a.heads), b = (int)(bh / a.heads);
  const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
  if (d < a.dim) {
    const float f[2] = {x[0] * by, x[1] * by};
    store_pack<T, 2>((T*)a.out + b * a.os[0] + head * a.os[1] + query * a.os[2] + d, f);
  }
  if (a.lse && lane == 0) a.lse[row] = off + log2f(sum);
}

// ------------------------------------------------------------------------------------------ backward
// D_i and log2 of the softmax's sum (+inf for a query without pairs: its p are zeros), a wave a row.
template <typename T>
__global__ __launch_bounds__(256) void row_terms(const Attention a, float* delta, float* lse2) {
  const int lane = threadIdx.x % 64;
  const int64_t rows = (int64_t)a.batch * a.heads * a.queries, row = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  if (row >= rows) return;
  const int64_t query = row % a.queries, bh = row / a.queries;
  const int head = (int)(bh % a.heads), b = (int)(bh / a.heads), d = 2 * lane;
  float dot = 0.f;
  if (d < a.dim) {
    float x[2], y[2];
    load_pack<T, 2>((const T*)a.out + b * a.os[0] + head * a.os[1] + query * a.os[2] + d, x);
    load_pack<T, 2>((const T*)a.grad + b * a.gs[0] + head * a.gs[1] + query * a.gs[2] + d, y);
    dot = x[0] * y[0] + x[1] * y[1];
  }
  dot = over_wave<Add>(dot);
  if (lane == 0) {
    const float l = a.lse[row];
    delta[row] = dot;
    lse2[row] = l == -INFINITY ? INFINITY : l;
  }
}

// map[query][key] to turned[key][query], rows of `pitch` bytes, 64 x 64 bytes a workgroup.
__global__ __launch_bounds__(256) void turn_map(const Attention a, uint8_t* turned, int64_t pitch) {
  __shared__ uint8_t block[64][65];
  const int64_t across = pitch / 64, q0 = blockIdx.x % across * 64, k0 = blockIdx.x / across * 64;
  const uint8_t* map = a.map + (int64_t)blockIdx.y * a.ms[0];
  const int x = threadIdx.x % 64;
  for (int y = threadIdx.x / 64; y < 64; y += 4)
    block[y][x] = q0 + y < a.queries && k0 + x < a.keys ? map[(q0 + y) * a.ms[1] + k0 + x] : 255;
  __syncthreads();
  uint8_t* to = turned + (int64_t)blockIdx.y * a.keys * pitch;
  for (int y = threadIdx.x / 64; y < 64; y += 4)
    if (k0 + y < a.keys) to[(k0 + y) * pitch + q0 + x] = block[x][y];
}

// dq and the bias table's gradient: as the forward, a workgroup walks the keys with 128 queries.  Each lane adds
// its ds to the bucket's sum in a column of its own (COLUMNS of them a wave: 64 up to 64 buckets, fewer beyond,
// then the lanes that share one take turns; 0: no table gradient), so that every sum has one order.
// Four at a time: read, add, write, and where two of the four meet the second takes the first's sum.  (An LDS
// float add of 64 lanes takes 193 cycles of a CU whatever its addresses, this 13.)
template <int COLUMNS>
__device__ __forceinline__ void add_by_bucket(float* column, const Buckets& bucket, int buckets, const float* x) {
#pragma unroll
  for (int v = 0; v < 16; v += 4) {
    int at[4];
    float sum[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) at[i] = std::min((int)bucket[v + i], buckets) * COLUMNS;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = column[at[i]];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum[i] += x[v + i];
#pragma unroll
      for (int j = i + 1; j < 4; ++j) sum[j] = at[j] == at[i] ? sum[i] : sum[j];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) column[at[i]] = sum[i];
  }
}

template <typename T, int DP, int COLUMNS>
__global__ __launch_bounds__(kThreads, kBackwardWaves<DP>) void grad_queries(const Attention a, unsigned tiles, const float* delta,
                                                         const float* lse2, float* table_parts) {
  constexpr int NT = kParts<T>, KEYS = 32 * NT;
  __shared__ __attribute__((aligned(16))) Tile<T, DP, NT> keys, values;
  __shared__ float table[kTable];
  extern __shared__ float sums[];   // [wave][bucket, the last for pairs that do not count][column]
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, h = lane / 32;
  const unsigned id = by_die(blockIdx.x, gridDim.x), tile = id % tiles, bh = id / tiles;
  const int head = (int)(bh % (unsigned)a.heads), b = (int)(bh / (unsigned)a.heads);
  const int shared_head = head / (a.heads / a.key_heads);
  const T* kp = (const T*)a.k + b * a.ks[0] + shared_head * a.ks[1];
  const T* vp = (const T*)a.v + b * a.vs[0] + shared_head * a.vs[1];
  table[threadIdx.x] = a.bias(head, threadIdx.x, __is_same(T, bf16));
  float* mine = sums + wave * (a.buckets + 1) * COLUMNS;
  for (int i = lane; i < (a.buckets + 1) * COLUMNS; i += 64) mine[i] = 0.f;

  const int64_t first = (int64_t)tile * (32 * kWaves), query = first + wave * 32 + lane % 32;
  const int64_t len = a.length(b), shift = len - a.queries;
  int64_t end = len;
  if (a.causal) end = std::min(end, std::min(first + 32 * kWaves, a.queries) + shift);
  const int64_t clamped = std::min(query, a.queries - 1), row = ((int64_t)b * a.heads + head) * a.queries + clamped;
  const uint8_t* map = a.map + b * a.ms[0] + clamped * a.ms[1];
  const int64_t last = a.causal ? std::min(len - 1, clamped + shift) : len - 1;
  const float my_lse = query < a.queries ? lse2[row] : INFINITY, my_delta = query < a.queries ? delta[row] : 0.f;

  Operand<T> q[DP / 16], g[DP / 16];
  load_columns<T, DP>(q, (const T*)a.q + b * a.qs[0] + head * a.qs[1], a.qs[2], query, a.queries, a.dim, lane);
  load_columns<T, DP>(g, (const T*)a.grad + b * a.gs[0] + head * a.gs[1], a.gs[2], query, a.queries, a.dim, lane);
  floatx16 dq[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) dq[d][v] = 0.f;

  Carry<T, DP, NT, kThreads> next_k, next_v;
  Buckets bucket[NT];
  next_k.load(kp, a.ks[2], 0, end, a.dim);
  next_v.load(vp, a.vs[2], 0, end, a.dim);
  for (int64_t k0 = 0; k0 < end; k0 += KEYS) {
#pragma unroll
    for (int t = 0; t < NT; ++t) bucket[t].load(map, k0 + 16 * NT * h + 16 * t, a.keys);
    __syncthreads();
    next_k.store(keys);
    next_v.store(values);
    __syncthreads();
    if (k0 + KEYS < end) {
      next_k.load(kp, a.ks[2], k0 + KEYS, end, a.dim);
      next_v.load(vp, a.vs[2], k0 + KEYS, end, a.dim);
    }
    floatx16 s[NT], e[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        s[t][v] = table[bucket[t][v]];
        e[t][v] = -my_delta;
      }
#pragma unroll
    for (int c = 0; c < DP / 16; ++c)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        s[t] = product(keys.rows(t, c, lane), q[c], s[t]);
        e[t] = product(values.rows(t, c, lane), g[c], e[t]);
      }
    if (k0 + KEYS > last + 1) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (k0 + 16 * NT * h + 16 * t + v > last) s[t][v] = -INFINITY;
    }
    float ds[NT][16];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v)
        ds[t][v] = __builtin_amdgcn_exp2f(fmaf(s[t][v], a.scale2, -my_lse)) * e[t][v];
    if constexpr (COLUMNS > 0) {
#pragma unroll
      for (int turn = 0; turn < 64 / COLUMNS; ++turn) {
        if (lane / COLUMNS == turn) {
#pragma unroll
          for (int t = 0; t < NT; ++t) add_by_bucket<COLUMNS>(mine + lane % COLUMNS, bucket[t], a.buckets, ds[t]);
        }
        if (COLUMNS < 64) wave_order();   // the next turn's lanes read what these wrote
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const Operand<T> w = rounded<T>(ds[t] + 8 * half);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d) dq[d] = product(keys.columns(t, half, d, lane), w, dq[d]);
      }
  }
  if (a.dq && query < a.queries)
    store_columns<T, DP>((T*)a.dq + b * a.dqs[0] + head * a.dqs[1], a.dqs[2], query, a.dim, lane, dq, a.scale);
  if constexpr (COLUMNS > 0) {
    __syncthreads();
    for (int i = threadIdx.x; i < a.buckets; i += kThreads) {
      float x = 0.f;
      for (int w = 0; w < kWaves; ++w)
        for (int c = 0; c < COLUMNS; ++c)   // begun at the bucket's own column: other banks for other lanes
          x += sums[(w * (a.buckets + 1) + i) * COLUMNS + (c + i) % COLUMNS];
      table_parts[((int64_t)bh * tiles + tile) * a.buckets + i] = x;
    }
  }
}

// dT[head][bucket]: a workgroup an entry; the parts are added in an order of their own, in double.
template <typename T>
__global__ __launch_bounds__(256) void join_table(const Attention a, unsigned tiles, const float* parts) {
  __shared__ double sums[256];
  const int head = blockIdx.x / a.buckets, bucket = blockIdx.x % a.buckets;
  double x = 0;
  const int64_t count = (int64_t)a.batch * tiles;
  for (int64_t i = threadIdx.x; i < count; i += 256) {
    const int64_t b = i / tiles, tile = i % tiles;
    x += parts[((b * a.heads + head) * tiles + tile) * a.buckets + bucket];
  }
  sums[threadIdx.x] = x;
  __syncthreads();
  for (int n = 128; n > 0; n /= 2) {
    if ((int)threadIdx.x < n) sums[threadIdx.x] += sums[threadIdx.x + n];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const int64_t at = (int64_t)head * a.buckets + bucket;
    if (a.table_float)
      ((float*)a.dtable)[at] = (float)sums[0];
    else
      ((T*)a.dtable)[at] = (T)(float)sums[0];
  }
}

// dk and dv: a workgroup keeps 128 keys, 32 a wave, and walks the queries of every head that reads them:
// S = Q K^T has the keys in columns.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads, kBackwardWaves<DP>) void grad_keys(const Attention a, unsigned tiles, const float* delta,
                                                      const float* lse2, const uint8_t* turned, int64_t pitch) {
  constexpr int NT = kParts<T>, ROWS = 32 * NT;
  __shared__ __attribute__((aligned(16))) Tile<T, DP, NT> queries, grads;
  __shared__ float table[kTable];
  __shared__ __attribute__((aligned(16))) float row_lse[ROWS], row_delta[ROWS];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, h = lane / 32;
  const unsigned id = by_die(blockIdx.x, gridDim.x), tile = id % tiles, bh = id / tiles;
  const int shared_head = (int)(bh % (unsigned)a.key_heads), b = (int)(bh / (unsigned)a.key_heads);
  const int group = a.heads / a.key_heads;
  const int64_t first = (int64_t)tile * (32 * kWaves), key = first + wave * 32 + lane % 32;
  const int64_t len = a.length(b), shift = len - a.queries;
  const uint8_t* map = turned + ((a.ms[0] ? (int64_t)b * a.keys : 0) + std::min(key, a.keys - 1)) * pitch;

  Operand<T> k[DP / 16], v[DP / 16];
  load_columns<T, DP>(k, (const T*)a.k + b * a.ks[0] + shared_head * a.ks[1], a.ks[2], key, len, a.dim, lane);
  load_columns<T, DP>(v, (const T*)a.v + b * a.vs[0] + shared_head * a.vs[1], a.vs[2], key, len, a.dim, lane);
  floatx16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int d = 0; d < DP / 32; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[d][i] = dv[d][i] = 0.f;

  // queries that see some key of the workgroup
  int64_t from = 0;
  if (a.causal) from = std::max<int64_t>(0, first - shift) / ROWS * ROWS;
  if (first >= len) from = a.queries;
  const int64_t seen = a.causal ? key - shift : 0;   // this lane's first query
  for (int head = shared_head * group; head < (shared_head + 1) * group; ++head) {
    const T* qp = (const T*)a.q + b * a.qs[0] + head * a.qs[1];
    const T* gp = (const T*)a.grad + b * a.gs[0] + head * a.gs[1];
    const int64_t row = ((int64_t)b * a.heads + head) * a.queries;
    __syncthreads();
    table[threadIdx.x] = a.bias(head, threadIdx.x, __is_same(T, bf16));
    Carry<T, DP, NT, kThreads> next_q, next_g;
    next_q.load(qp, a.qs[2], from, a.queries, a.dim);
    next_g.load(gp, a.gs[2], from, a.queries, a.dim);
    for (int64_t q0 = from; q0 < a.queries; q0 += ROWS) {
      Buckets bucket[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) bucket[t].load(map, q0 + 16 * NT * h + 16 * t, pitch);
      __syncthreads();
      next_q.store(queries);
      next_g.store(grads);
      if (threadIdx.x < ROWS) {
        const int64_t q = q0 + threadIdx.x;
        row_lse[threadIdx.x] = q < a.queries ? -lse2[row + q] : -INFINITY;
        row_delta[threadIdx.x] = q < a.queries ? -delta[row + q] : 0.f;
      }
      __syncthreads();
      if (q0 + ROWS < a.queries) {
        next_q.load(qp, a.qs[2], q0 + ROWS, a.queries, a.dim);
        next_g.load(gp, a.gs[2], q0 + ROWS, a.queries, a.dim);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        floatx16 s, e;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          s[i] = table[bucket[t][i]];
          e[i] = row_delta[16 * NT * h + 16 * t + i];
        }
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
          s = product(queries.rows(t, c, lane), k[c], s);
          e = product(grads.rows(t, c, lane), v[c], e);
        }
        if (q0 < seen) {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (q0 + 16 * NT * h + 16 * t + i < seen) s[i] = -INFINITY;
        }
        float p[16], ds[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale2, row_lse[16 * NT * h + 16 * t + i]));
          ds[i] = p[i] * e[i];
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const Operand<T> w = rounded<T>(p + 8 * half), x = rounded<T>(ds + 8 * half);
#pragma unroll
          for (int d = 0; d < DP / 32; ++d) {
            dv[d] = product(grads.columns(t, half, d, lane), w, dv[d]);
            dk[d] = product(queries.columns(t, half, d, lane), x, dk[d]);
          }
        }
      }
    }
  }
  if (key >= a.keys) return;
  if (key >= len)   // columns of keys that do not count
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) dk[d][i] = dv[d][i] = 0.f;
  if (a.dk) store_columns<T, DP>((T*)a.dk + b * a.dks[0] + shared_head * a.dks[1], a.dks[2], key, a.dim, lane, dk, a.scale);
  if (a.dv) store_columns<T, DP>((T*)a.dv + b * a.dvs[0] + shared_head * a.dvs[1], a.dvs[2], key, a.dim, lane, dv, 1.f);
}

// ------------------------------------------------------------------------------------------ host
#define ATTENTION_DIM(dim, ...)                        \
  do {                                                  \
    if ((dim) <= 32) { constexpr int DP = 32; __VA_ARGS__; }   \
    else if ((dim) <= 64) { constexpr int DP = 64; __VA_ARGS__; } \
    else { constexpr int DP = 128; __VA_ARGS__; }              \
  } while (0)

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
  SDK_REQUIRE(a->scale > 0 && std::isfinite(a->scale), "scale must be positive and finite");
  SDK_REQUIRE(a->batch < 1 << 20 && a->heads < 1 << 20 && a->queries < (int64_t)1 << 31 && a->keys < (int64_t)1 << 31,
              "batch or heads of 2^20, or 2^31 tokens or more");
  const int64_t groups = a->batch * a->heads * std::max(ceil_div(a->queries, 128), ceil_div(a->keys, 128));
  SDK_REQUIRE(a->batch < 65536 && ceil_div(a->queries, 64) * ceil_div(a->keys, 64) < (int64_t)1 << 31,
              "a batch of 65536 or more, or a map of 2^43 pairs or more");
  SDK_REQUIRE(groups < (int64_t)1 << 24, "%lld tiles of 128 tokens are too many", (long long)groups);
  return SDK_OK;
}

int check_rows(const char* name, const void* p, const int64_t* strides, int dtype) {
  SDK_REQUIRE(p, "%s must not be NULL", name);
  bool ok = aligned16(p);
  for (int i = 0; i < 3; ++i) ok = ok && strides[i] % (16 / (int64_t)bytes_of(dtype)) == 0;
  SDK_REQUIRE(ok, "rows of %s must be 16-byte aligned", name);
  return SDK_OK;
}

Attention on_device(const sdk_bucket_attention* a) {
  Attention d = {};
  d.q = a->query, d.k = a->key, d.v = a->value, d.table = a->bias_table, d.out = a->output, d.grad = a->grad_output;
  d.map = a->bucket_map, d.lengths = a->key_lengths;
  d.dq = a->grad_query, d.dk = a->grad_key, d.dv = a->grad_value, d.dtable = a->grad_table, d.lse = a->lse;
  for (int i = 0; i < 3; ++i) {
    d.qs[i] = a->query_strides[i], d.ks[i] = a->key_strides[i], d.vs[i] = a->value_strides[i];
    d.os[i] = a->output_strides[i], d.gs[i] = a->grad_output_strides[i], d.dqs[i] = a->grad_query_strides[i];
    d.dks[i] = a->grad_key_strides[i], d.dvs[i] = a->grad_value_strides[i];
  }
  d.ms[0] = a->map_strides[0], d.ms[1] = a->map_strides[1];
  d.queries = a->queries, d.keys = a->keys, d.batch = (int)a->batch, d.heads = (int)a->heads;
  d.key_heads = (int)a->key_heads, d.dim = (int)a->dim, d.buckets = (int)a->buckets, d.causal = a->causal != 0;
  d.table_float = a->table_dtype == SDK_F32;
  d.scale = (float)a->scale, d.scale2 = (float)(a->scale * 1.4426950408889634);
  d.limit = (float)(0x1p100 / std::max(1.0, a->scale));
  return d;
}

// Whether a key head's rows go to attend_few.
bool few_rows(const sdk_bucket_attention* a) { return a->heads / a->key_heads * a->queries <= 32; }

// Parts that the keys are dealt to: enough workgroups for the 256 CUs, at least 256 keys each.
int splits_of(const sdk_bucket_attention* a) {
  const bool few = few_rows(a);
  const int64_t groups = few ? a->batch * a->key_heads : a->batch * a->heads * ceil_div(a->queries, 32 * kWaves);
  if (groups >= (few ? 512 : 256) || groups == 0) return 1;
  return (int)std::max<int64_t>(1, std::min(ceil_div(512, groups), a->keys / 256));
}

struct BackwardSpace {
  int64_t delta, lse2, parts, turned, pitch, total;
};
BackwardSpace backward_space(const sdk_bucket_attention* a) {
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  BackwardSpace w;
  const int64_t rows = a->batch * a->heads * a->queries;
  w.pitch = ceil_div(a->queries, 64) * 64;
  w.delta = 0;
  w.lse2 = w.delta + up(rows * 4);
  w.parts = w.lse2 + up(rows * 4);
  w.turned = w.parts + up(a->batch * a->heads * ceil_div(a->queries, 32 * kWaves) * a->buckets * 4);
  w.total = w.turned + up((a->map_strides[0] ? a->batch : 1) * a->keys * w.pitch);
  return w;
}

template <typename T, int DP, int COLUMNS>
int launch_grad_queries(const Attention& d, unsigned tiles, const float* delta, const float* lse2, float* parts,
                        hipStream_t s) {
  const size_t smem = (size_t)kWaves * (d.buckets + 1) * COLUMNS * sizeof(float);
  auto* kernel = grad_queries<T, DP, COLUMNS>;
  if (smem > (32 << 10)) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != hipSuccess) return fail(SDK_ERR_DEVICE, "LDS of %zu bytes: %s", smem, hipGetErrorString(e));
  }
  kernel<<<dim3(tiles * (unsigned)(d.batch * d.heads)), dim3(kThreads), smem, s>>>(d, tiles, delta, lse2, parts);
  return SDK_OK;
}

int check_inputs(const sdk_bucket_attention* a) {
  if (int rc = check_rows("query", a->query, a->query_strides, a->dtype)) return rc;
  if (int rc = check_rows("output", a->output, a->output_strides, a->dtype)) return rc;
  SDK_REQUIRE(a->bias_table, "bias_table must not be NULL");
  if (a->keys == 0) return SDK_OK;
  if (int rc = check_rows("key", a->key, a->key_strides, a->dtype)) return rc;
  if (int rc = check_rows("value", a->value, a->value_strides, a->dtype)) return rc;
  SDK_REQUIRE(a->bucket_map, "bucket_map must not be NULL");
  return SDK_OK;
}

}  // namespace
}  // namespace token
}  // namespace sdk

using namespace sdk;
using namespace sdk::token;

extern "C" {

size_t sdk_bucket_attention_workspace_bytes(const sdk_bucket_attention* a, int32_t backward) {
  if (check(a) != SDK_OK || a->batch == 0 || a->queries == 0) return 0;
  if (backward) return (size_t)backward_space(a).total;
  const int splits = splits_of(a);
  return splits == 1 ? 0 : (size_t)splits * a->batch * a->heads * a->queries * (a->dim + 1) * sizeof(float);
}

int sdk_bucket_attention_forward(const sdk_bucket_attention* a, void* workspace, size_t workspace_bytes,
                                 sdk_stream_t stream) {
  if (int rc = check(a)) return rc;
  if (a->batch == 0 || a->queries == 0) return SDK_OK;
  if (int rc = check_inputs(a)) return rc;
  const size_t need = sdk_bucket_attention_workspace_bytes(a, 0);
  if (need && (!workspace || workspace_bytes < need))
    return fail(SDK_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const Attention d = on_device(a);
  const int splits = splits_of(a);
  const unsigned tiles = (unsigned)ceil_div(a->queries, 32 * kWaves);
  const int64_t rows = a->batch * a->heads * a->queries;
  float* part_out = (float*)workspace;
  float* part_lse = part_out ? part_out + splits * rows * a->dim : nullptr;
  hipStream_t s = (hipStream_t)stream;
  SDK_DISPATCH_TOKEN_DTYPE(a->dtype, {
    if (few_rows(a)) {
      const int group = d.heads / d.key_heads;
      ATTENTION_DIM(a->dim, {
        attend_few<T, DP><<<dim3((unsigned)(a->batch * a->key_heads) * splits), dim3(kThreads),
                            group*(kTable + 1) * sizeof(float), s>>>(d, splits, part_out, part_lse);
      });
    } else
      ATTENTION_DIM(a->dim, launch(attend<T, DP>, dim3(tiles * (unsigned)(a->batch * a->heads) * splits),
                                 dim3(kThreads), s, d, splits, tiles, part_out, part_lse));
    if (splits > 1)
      launch(join<T>, dim3((unsigned)ceil_div(rows, 4)), dim3(256), s, d, splits, (const float*)part_out,
             (const float*)part_lse);
  });
  SDK_LAUNCH_CHECK("bucket_attention_forward");
  return SDK_OK;
}

int sdk_bucket_attention_backward(const sdk_bucket_attention* a, void* workspace, size_t workspace_bytes,
                                  sdk_stream_t stream) {
  if (int rc = check(a)) return rc;
  hipStream_t s = (hipStream_t)stream;
  const bool any = a->batch > 0 && a->queries > 0;
  if (any) {
    if (int rc = check_inputs(a)) return rc;
    if (int rc = check_rows("grad_output", a->grad_output, a->grad_output_strides, a->dtype)) return rc;
    SDK_REQUIRE(a->lse, "lse must not be NULL");
  }
  if (a->grad_query && any)
    if (int rc = check_rows("grad_query", a->grad_query, a->grad_query_strides, a->dtype)) return rc;
  if (a->grad_key && a->batch > 0 && a->keys > 0)
    if (int rc = check_rows("grad_key", a->grad_key, a->grad_key_strides, a->dtype)) return rc;
  if (a->grad_value && a->batch > 0 && a->keys > 0)
    if (int rc = check_rows("grad_value", a->grad_value, a->grad_value_strides, a->dtype)) return rc;
  const size_t need = sdk_bucket_attention_workspace_bytes(a, 1);
  if (need && (!workspace || workspace_bytes < need))
    return fail(SDK_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const Attention d = on_device(a);
  const BackwardSpace w = backward_space(a);
  char* ws = (char*)workspace;
  float *delta = (float*)(ws + w.delta), *lse2 = (float*)(ws + w.lse2), *parts = (float*)(ws + w.parts);
  uint8_t* turned = (uint8_t*)(ws + w.turned);
  const unsigned q_tiles = (unsigned)ceil_div(a->queries, 32 * kWaves), k_tiles = (unsigned)ceil_div(a->keys, 32 * kWaves);
  const int64_t rows = a->batch * a->heads * a->queries;
  const int columns = !a->grad_table ? 0 : a->buckets <= 64 ? 64 : a->buckets <= 128 ? 32 : 16;
  SDK_DISPATCH_TOKEN_DTYPE(a->dtype, {
    if (any) {
      launch(row_terms<T>, dim3((unsigned)ceil_div(rows, 4)), dim3(256), s, d, delta, lse2);
      if (a->grad_query || a->grad_table) {
        ATTENTION_DIM(a->dim, {
          int rc = columns == 0    ? launch_grad_queries<T, DP, 0>(d, q_tiles, delta, lse2, parts, s)
                   : columns == 64 ? launch_grad_queries<T, DP, 64>(d, q_tiles, delta, lse2, parts, s)
                   : columns == 32 ? launch_grad_queries<T, DP, 32>(d, q_tiles, delta, lse2, parts, s)
                                   : launch_grad_queries<T, DP, 16>(d, q_tiles, delta, lse2, parts, s);
          if (rc != SDK_OK) return rc;
        });
      }
    }
    if (a->grad_table)
      launch(join_table<T>, dim3((unsigned)(a->heads * a->buckets)), dim3(256), s, d, any ? q_tiles : 0u,
             (const float*)parts);
    if ((a->grad_key || a->grad_value) && a->batch > 0 && a->keys > 0) {
      if (any)
        launch(turn_map, dim3((unsigned)(w.pitch / 64 * ceil_div(a->keys, 64)), (unsigned)(a->map_strides[0] ? a->batch : 1)),
               dim3(256), s, d, turned, w.pitch);
      ATTENTION_DIM(a->dim, launch(grad_keys<T, DP>, dim3(k_tiles * (unsigned)(a->batch * a->key_heads)),
                                   dim3(kThreads), s, d, k_tiles, (const float*)delta, (const float*)lse2,
                                   (const uint8_t*)turned, w.pitch));
    }
  });
  SDK_LAUNCH_CHECK("bucket_attention_backward");
  return SDK_OK;
}

}  // extern "C"
