// Backward of attention with a bias for each bucket of relative positions (token_attention.hpp: operands and tiles).
//
//   p_ij = exp(s_ij - lse_i)      D_i = <do_i, o_i>      ds_ij = p_ij (<do_i, v_j> - D_i)
//   dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i      dv_j = sum_i p_ij do_i
//   dT[head][b] = sum of ds_ij over the pairs of bucket b
//
// The scores are formed again from the lse, once with the queries in registers (dq, dT) and once with the keys (dk,
// dv): seven products instead of five, and no sum whose order depends on scheduling.
//
// float16 has few exponents: p (about 1 / keys) and ds would fall among its subnormal numbers, or beyond its largest.
// There p is held times 2^8 and ds times a power of two of its own row (dq) or key (dk), so that rows and keys of any
// size keep their precision beside others; they are taken out of the sums, exactly.  dv takes do as it is.
#include "token_attention.hpp"

namespace sdk {
namespace token {
namespace {

// Waves of a SIMD: with two, accumulators lie among the 256 registers of a wave.  Heads of 96 in 16 bits spill 12 to 24
// bytes for it in grad_queries, once: 2 x 16 heads of 80, 2048 tokens, forward and backward 398 us for 460; heads of 128
// would spill 200 to 440.
template <typename T, int DP>
constexpr int kQueryWaves = DP <= (sizeof(T) == 2 ? 96 : 64) ? 2 : 1;
template <typename T, int DP>
constexpr int kKeyWaves = DP <= (sizeof(T) == 2 ? 64 : 32) ? 2 : 1;

template <typename T>
constexpr float kLift = __is_same(T, f16) ? 8.f : 0.f;   // log2 of what p is held times

// float16, dq: what p is held times (log2: lift) and what a row's do is (by).  With size = sum |do| of the row and value =
// the largest |v|, |ds| is at most p 2 size value: below 2^15 as held.  Values beyond 2^9 lower the lift instead of
// do, whose numbers would become subnormal.  p of far rows (Lse) reaches 2^10, not 2^lift.
struct Hold {
  float lift = kLift<f16>, by = 1.f;
  __device__ __forceinline__ Hold(float size, float value, bool far) {
    if (!(size > 0.f && size < INFINITY && value < INFINITY)) return;   // nothing to hold, or nothing finite
    const int s = (int)(__float_as_uint(size) >> 23) - 126;             // size < 2^s
    const int v = std::max((int)(__float_as_uint(value) >> 23) - 126, -8), up = 17 - std::max(v, 9);
    lift = (float)up;
    by = __uint_as_float((unsigned)(127 + 14 - (far ? 10 : up) - s - v) << 23);
  }
};

// A row's level and log2 of its sum as p = 2^(scale2 s - off) * factor, times 2^lift.  whole: off is a whole number, for
// weights that round as the forward's did; the factor is then between 1 and 2.  Else it is 1, but for levels (of rows
// that biases mask) that would swallow what is added to them.
__device__ __forceinline__ bool is_far(float level) { return fabsf(level) > 1024.f && fabsf(level) < INFINITY; }
struct Lse {
  float off, factor = 1.f;
  bool far;
  __device__ __forceinline__ Lse(float level, float part, bool whole, float lift) : off(level), far(is_far(level)) {
    const float up = whole ? ceilf(part) : part;
    if (far)
      factor = __builtin_amdgcn_exp2f(lift - part);
    else
      off += up - lift, factor = __builtin_amdgcn_exp2f(up - part);
  }
};

template <typename T>
__device__ __forceinline__ void flip(Operand<T>& x, bool odd) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 3; ++i) flip(x.piece[i], odd);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x.u[i] ^= odd ? 0x80008000u : 0u;
  }
}

// ------------------------------------------------------------------------------------------ terms of a row
// float16: the largest |v| among the keys that count of each key head, in `parts` parts of the keys.
constexpr int kMostParts = 64;   // a lane each where they are read
__global__ __launch_bounds__(256) void value_sizes(const Attention a, int parts, float* sizes) {
  __shared__ float slots[4];
  const int part = (int)(blockIdx.x % (unsigned)parts), bh = (int)(blockIdx.x / (unsigned)parts);
  const int head = bh % a.key_heads, b = bh / a.key_heads, d = 8 * (threadIdx.x % 16);
  const int len = a.length(b), to = split_at(len, part + 1, parts);
  const f16* v = (const f16*)a.v + b * a.vs[0] + head * a.vs[1] + d;
  float most = 0.f;
#pragma unroll 4
  for (int key = split_at(len, part, parts) + threadIdx.x / 16; key < to; key += 16) {
    if (d >= a.dim) continue;
    float x[8];
    load_pack<f16, 8>(v + key * a.vs[2], x);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = Largest::of(most, fabsf(x[e]));
  }
  most = over_group<Largest, 256>(most, slots);
  if (threadIdx.x == 0) sizes[blockIdx.x] = most;
}

// D_i and the row's level (+inf for a query without pairs: its p are zeros).  A row is read by LANES lanes, 16 bytes
// each.
template <typename T, int LANES>
__global__ __launch_bounds__(256) void row_terms(const Attention a, float* delta, float* lse2) {
  const int lane = threadIdx.x % LANES, d = kWide<T> * lane;
  const int64_t rows = (int64_t)a.batch * a.heads * a.queries;
  for (int64_t first = (int64_t)blockIdx.x * (256 / LANES); first < rows; first += (int64_t)gridDim.x * (256 / LANES)) {
    const int64_t row = first + threadIdx.x / LANES;
    float dot = 0.f;
    if (row < rows) {
      const int64_t query = row % a.queries, bh = row / a.queries;
      const int head = (int)(bh % a.heads), b = (int)(bh / a.heads);
      if (d < a.dim) {
        float x[kWide<T>], y[kWide<T>];
        const int64_t at = b * a.os[0] + head * a.os[1] + query * a.os[2] + d;
        load_pack<T, kWide<T>>((const T*)a.out + at, x);
        if (a.rest) {
          load_pack<T, kWide<T>>((const T*)a.rest + at, y);
#pragma unroll
          for (int e = 0; e < kWide<T>; ++e) x[e] += y[e];
        }
        load_pack<T, kWide<T>>((const T*)a.grad + b * a.gs[0] + head * a.gs[1] + query * a.gs[2] + d, y);
#pragma unroll
        for (int e = 0; e < kWide<T>; ++e) dot = fmaf(x[e], y[e], dot);
      }
    }
#pragma unroll
    for (int n = LANES / 2; n > 0; n /= 2) dot += __shfl_xor(dot, n);
    if (row < rows && lane == 0) {
      const float l = a.lse[row];
      delta[row] = dot;
      lse2[row] = l == -INFINITY ? INFINITY : l;
    }
  }
}

// map[query][key] to turned[key][query], rows of `pitch` bytes, 64 x 64 bytes a workgroup at a time.
__global__ __launch_bounds__(256) void turn_map(const Attention a, uint8_t* turned, int pitch, unsigned blocks) {
  __shared__ uint8_t block[64][65];
  const int across = pitch / 64, x = threadIdx.x % 64;
  const uint8_t* map = a.map + (int64_t)blockIdx.y * a.ms[0];
  uint8_t* to = turned + (int64_t)blockIdx.y * a.keys * pitch;
  for (unsigned i = blockIdx.x; i < blocks; i += gridDim.x) {
    const int q0 = (int)(i % across) * 64, k0 = (int)(i / across) * 64;
    for (int y = threadIdx.x / 64; y < 64; y += 4)
      block[y][x] = q0 + y < a.queries && k0 + x < a.keys ? map[(q0 + y) * a.ms[1] + k0 + x] : 255;
    __syncthreads();
    for (int y = threadIdx.x / 64; y < 64; y += 4)
      if (k0 + y < a.keys) to[(int64_t)(k0 + y) * pitch + q0 + x] = block[x][y];
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------ dq and the bias table
// Adds x * by to the sums of its buckets in one lane's column, two at a time: read, add, write, and where the two meet the
// second takes the first's sum.  (An LDS float add of 64 lanes takes 193 cycles of a CU whatever its addresses, this
// 13; by four or eight the comparisons cost more than the waits they save: 3 and 19 % more of the whole kernel.)
template <int COLUMNS>
__device__ __forceinline__ void add_by_bucket(float* column, const Buckets& bucket, int buckets, const float* x,
                                              float by) {
#pragma unroll
  for (int v = 0; v < 16; v += 2) {
    const int at = std::min((int)bucket[v], buckets) * COLUMNS, next = std::min((int)bucket[v + 1], buckets) * COLUMNS;
    const float sum = column[at] + x[v] * by, other = column[next];
    column[at] = sum;
    column[next] = (next == at ? sum : other) + x[v + 1] * by;
  }
}

// As the forward, a workgroup walks the keys (or a split of them) with 128 queries.  Each lane adds its ds to the
// bucket's sum in a column of its own (COLUMNS of them a wave: 64 up to 64 buckets, fewer beyond, then the lanes
// that share one take turns; 0: no table gradient), so that every sum has one order.
// Bound by vector instructions and LDS: 16 heads of 64, 8192 x 8192 pairs in bfloat16 take 704 us (585 TFLOP/s), 5 % of
// it the rounding of the weights.
// part: splits > 1: float32 sums of the splits, [split][row][dim].
template <typename T, int DP, int COLUMNS>
__global__ __launch_bounds__(kThreads, (kQueryWaves<T, DP>)) void grad_queries(
    const Attention a, int splits, int tiles, const float* delta, const float* lse2, const float* sizes, int size_parts,
    float* part, float* table_parts) {
  constexpr int NT = kParts<T>, KEYS = 32 * NT;
  __shared__ __attribute__((aligned(16))) struct {
    float table[kTable];   // at address zero: a lookup's address is four times the bucket
    Tile<T, DP, NT> keys, values;
  } lds;
  auto& table = lds.table;
  auto &keys = lds.keys, &values = lds.values;
  extern __shared__ float sums[];   // [wave][bucket, the last for pairs that do not count][column]
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, h = lane / 32;
  const Work work(tiles, a.batch * a.heads, splits, a.causal, false);
  const int head = work.head % a.heads, b = work.head / a.heads;
  const int shared_head = head / (a.heads / a.key_heads);
  const T* kp = (const T*)a.k + b * a.ks[0] + shared_head * a.ks[1];
  const T* vp = (const T*)a.v + b * a.vs[0] + shared_head * a.vs[1];
  table[threadIdx.x] = a.bias(head, threadIdx.x, __is_same(T, bf16));
  float* mine = sums + wave * (a.buckets + 1) * COLUMNS;
  for (int i = lane; i < (a.buckets + 1) * COLUMNS; i += 64) mine[i] = 0.f;

  const int first = work.tile * (32 * kWaves), query = first + wave * 32 + lane % 32;
  const int len = a.length(b), shift = len - a.queries;
  const int end = a.causal ? std::min(len, std::min(first + 32 * kWaves, a.queries) + shift) : len;
  const int blocks = end > 0 ? (end + KEYS - 1) / KEYS : 0;
  const int from = split_at(blocks, work.split, splits) * KEYS;
  const int to = std::min(end, split_at(blocks, work.split + 1, splits) * KEYS);
  const int clamped = std::min(query, a.queries - 1);
  const int64_t row = (int64_t)work.head * a.queries + clamped;
  const uint8_t* map = a.map + b * a.ms[0] + clamped * a.ms[1];
  const int last = a.causal ? std::min(len - 1, clamped + shift) : len - 1;
  const bool in = query < a.queries;
  const float level = in ? lse2[row] : INFINITY;

  Operand<T> q[DP / 16], g[DP / 16];
  load_columns<T, DP>(q, (const T*)a.q + b * a.qs[0] + head * a.qs[1], a.qs[2], query, in, a.dim, lane);
  load_columns<T, DP>(g, (const T*)a.grad + b * a.gs[0] + head * a.gs[1], a.gs[2], query, in, a.dim, lane);
  float lift = kLift<T>, held = 1.f;
  if constexpr (__is_same(T, f16)) {
    float size = 0.f;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const f16x8 x = __builtin_bit_cast(f16x8, g[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) size += fabsf((float)x[e]);
    }
    const int64_t at = ((int64_t)b * a.key_heads + shared_head) * size_parts;
    const float value = over_wave<Largest>(lane < size_parts ? sizes[at + lane] : 0.f);
    const Hold hold(size + other_half(size), value, is_far(level));
    lift = hold.lift, held = hold.by;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      f16x8 x = __builtin_bit_cast(f16x8, g[c]);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (f16)((float)x[e] * held);
      g[c] = __builtin_bit_cast(Operand<T>, x);
    }
  }
  const Lse lse(level, in ? a.lse[(int64_t)a.batch * a.heads * a.queries + row] : 0.f, true, lift);
  const float my_lse = lse.off;
  float my_delta = in ? delta[row] * held : 0.f;
  // Odd lanes work with -do and -D, so that ds has the other sign: what the matrix unit's rounding leaves to one side
  // would add up in the table's sums, which cancel over many rows.  A lane's row and column are all of one sign.
  const float sign = lane % 2 ? -1.f : 1.f;
  my_delta *= sign;
  // A factor of everything this lane sums.  16 columns hold two queries each, whose factors the table's sums take pair by
  // pair: float16's, which have any size, beside ds, the others with it (15 registers fewer).
  constexpr bool BESIDE = COLUMNS == 16 && __is_same(T, f16), WITHIN = COLUMNS == 16 && !BESIDE;
  const float back = exp2f(-lift) / held * sign * (WITHIN ? 1.f : lse.factor);
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) flip(g[c], lane % 2);
  floatx16 dq[DP / 32];
  clear(dq);

  Carry<T, DP, NT, kThreads> next_k(a.ks[2], a.dim), next_v(a.vs[2], a.dim);
  Buckets bucket[NT], next_bucket[NT];
  auto request = [&](int k0) {
    next_k.load(kp + k0 * a.ks[2], a.ks[2], to - k0, a.dim);
    next_v.load(vp + k0 * a.vs[2], a.vs[2], to - k0, a.dim);
    load_buckets<NT>(next_bucket, map, k0, a.keys, h);
  };
  const auto key_view = keys.view(lane), value_view = values.view(lane);
  if (from < to) request(from);
  landed();
  auto step = [&](int k0, auto edge) {   // edge: some key may be beyond a lane's last
    __syncthreads();
    next_k.store(keys);
    next_v.store(values);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) bucket[t] = next_bucket[t];
    request(k0 + KEYS);   // beyond the last tile nothing is read
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      floatx16 s = dot_tile<T, DP>(key_view, t, q, [&](int v) { return table[bucket[t][v]]; });
      const floatx16 e = dot_tile<T, DP>(value_view, t, g, [&](int) { return -my_delta; });
      if constexpr (edge)
        if (k0 + KEYS > last + 1) {
#pragma unroll
          for (int v = 0; v < 16; ++v)
            if (k0 + 16 * NT * h + 16 * t + v > last) s[v] = -INFINITY;
        }
      // The forward's own weights, rounded as they were: D is the mean of do v^T under these, so that a row's ds add up
      // to zero.  Unrounded ones miss it by 2^-9 of a weight, which a sum over many keys shows where the table's
      // entries, or keys with much in common, cancel.  ds then goes to the matrix unit in the inputs' type, here and for
      // dk: gradients are off by 2.9e-3 of their size in bfloat16 (3.5e-4 in float16), 1.7e-3 (2.1e-4) of it their own
      // rounding.  Weights and ds in two pieces everywhere leave that alone, and take 2241 us for a step of 1850.
      float ds[16];
#pragma unroll
      for (int v = 0; v < 16; ++v) ds[v] = __builtin_amdgcn_exp2f(fmaf(s[v], a.scale2, -my_lse));
      as_rounded<T>(ds);
#pragma unroll
      for (int v = 0; v < 16; ++v) ds[v] *= e[v];
      if constexpr (WITHIN) {
#pragma unroll
        for (int v = 0; v < 16; ++v) ds[v] *= lse.factor;
      }
      if constexpr (COLUMNS > 0) {
#pragma unroll
        for (int turn = 0; turn < 64 / COLUMNS; ++turn) {
          if (lane / COLUMNS == turn)
            add_by_bucket<COLUMNS>(mine + lane % COLUMNS, bucket[t], a.buckets, ds, BESIDE ? back : 1.f);
          if (COLUMNS < 64) wave_order();   // the next turn's lanes read what these wrote
        }
      }
      const Operand<T> w[2] = {rounded<T>(ds), rounded<T>(ds + 8)};
      add_columns<T>(dq, key_view, t, w);
    }
  };
  // whole tiles that every query of the workgroup sees, in a loop without branches
  const int whole = (a.causal ? std::max(0, std::min(len, first + shift + 1)) : len) / KEYS * KEYS;
  int k0 = from;
  if constexpr (sizeof(T) == 2)   // float32: the registers do not hold two loops (14 % more time than one)
    for (; k0 < std::min(to, whole); k0 += KEYS) step(k0, std::false_type());
  for (; k0 < to; k0 += KEYS) step(k0, std::true_type());
  if (in && splits > 1)
    store_columns<float, DP>(part + ((int64_t)work.split * a.batch * a.heads * a.queries + row) * a.dim, a.dim, 0, a.dim,
                             lane, dq, a.scale * back);
  else if (in && a.dq)
    store_columns<T, DP>((T*)a.dq + b * a.dqs[0] + head * a.dqs[1], a.dqs[2], query, a.dim, lane, dq,
                         a.scale * back);
  if constexpr (COLUMNS > 0) {
    __shared__ float column_back[kWaves][COLUMNS];
    if (lane < COLUMNS) column_back[wave][lane] = BESIDE ? 1.f : back;
    __syncthreads();
    for (int i = threadIdx.x; i < a.buckets; i += kThreads) {
      float x = 0.f;
      for (int w = 0; w < kWaves; ++w)
#pragma unroll 4
        for (int c = 0; c < COLUMNS; ++c) {   // begun at the bucket's own column: other banks for other lanes
          const int column = (c + i) % COLUMNS;
          x += sums[(w * (a.buckets + 1) + i) * COLUMNS + column] * column_back[w][column];
        }
      table_parts[(((int64_t)work.head * tiles + work.tile) * splits + work.split) * a.buckets + i] = x;
    }
  }
}

// dT[head][bucket]: a workgroup an entry at a time; the `each` parts of every batch element are added in an order of
// their own, in double.
template <typename T>
__global__ __launch_bounds__(256) void join_table(const Attention a, int each, const float* parts) {
  __shared__ double sums[256];
  const int64_t count = (int64_t)a.batch * each;
  for (int at = blockIdx.x; at < a.heads * a.buckets; at += gridDim.x) {   // fewer than 2^28
    const int head = at / a.buckets, bucket = at % a.buckets;
    double x = 0;
    for (int64_t i = threadIdx.x; i < count; i += 256)
      x += parts[((i / each * a.heads + head) * each + i % each) * a.buckets + bucket];
    sums[threadIdx.x] = x;
    __syncthreads();
    for (int n = 128; n > 0; n /= 2) {
      if ((int)threadIdx.x < n) sums[threadIdx.x] += sums[threadIdx.x + n];
      __syncthreads();
    }
    if (threadIdx.x == 0) {
      if (a.table_float)
        ((float*)a.dtable)[at] = (float)sums[0];
      else
        ((T*)a.dtable)[at] = (T)(float)sums[0];
    }
  }
}

// ------------------------------------------------------------------------------------------ dk and dv
// A workgroup keeps 128 keys, 32 a wave, and walks the queries of every head that reads them (or a split of these
// tiles): S = Q K^T has the keys in columns.  The next tile is requested while this one is worked on, into the
// other buffer.  Bound by LDS (both operands straight and turned) and what it does not overlap: 4 key heads of 16 heads
// of 64, 8192 x 8192 pairs in bfloat16 take 651 us, 845 TFLOP/s.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads, (kKeyWaves<T, DP>)) void grad_keys(
    const Attention a, int splits, int tiles, const float* delta, const float* lse2, const uint8_t* turned,
    int pitch, float* part) {
  constexpr int NT = kParts<T>, ROWS = 32 * NT;
  __shared__ __attribute__((aligned(16))) struct {
    float table[kTable];
    float row_lse[2][ROWS], row_delta[2][ROWS], row_factor[2][ROWS];
    Tile<T, DP, NT> queries[2], grads[2];   // 16-byte aligned
    int far[2];                             // whether some row of the tile has a factor
  } lds;
  auto& table = lds.table;
  auto &row_lse = lds.row_lse, &row_delta = lds.row_delta, &row_factor = lds.row_factor;
  auto &queries = lds.queries, &grads = lds.grads;
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, h = lane / 32;
  const Work work(tiles, a.batch * a.key_heads, splits, a.causal, true);
  const int shared_head = work.head % a.key_heads, b = work.head / a.key_heads;
  const int group = a.heads / a.key_heads;
  const int first = work.tile * (32 * kWaves), key = first + wave * 32 + lane % 32;
  const int len = a.length(b), shift = len - a.queries;
  const uint8_t* map = turned + ((a.ms[0] ? (int64_t)b * a.keys : 0) + std::min(key, a.keys - 1)) * pitch;

  Operand<T> k[DP / 16], v[DP / 16];
  load_columns<T, DP>(k, (const T*)a.k + b * a.ks[0] + shared_head * a.ks[1], a.ks[2], key, key < len, a.dim, lane);
  load_columns<T, DP>(v, (const T*)a.v + b * a.vs[0] + shared_head * a.vs[1], a.vs[2], key, key < len, a.dim, lane);
  floatx16 dk[DP / 32], dv[DP / 32];
  clear(dk);
  clear(dv);
  float held = __is_same(T, f16) ? 0x1p100f : 1.f;   // what this key's ds are held times

  // tiles of queries that see some key of the workgroup, head after head
  const int from = a.causal ? std::max(0, first - shift) / ROWS * ROWS : 0;
  const int each = first < len && from < a.queries ? (a.queries - from + ROWS - 1) / ROWS : 0;
  const int begin = split_at(group * each, work.split, splits), stop = split_at(group * each, work.split + 1, splits);
  const int seen = a.causal ? key - shift : 0;   // this lane's first query

  Carry<T, DP, NT, kThreads> next_q(a.qs[2], a.dim), next_g(a.gs[2], a.dim);
  Buckets bucket[NT], next_bucket[NT];
  float next_lse = 0.f, next_delta = 0.f, next_rest = 0.f;
  const float* rests = a.lse + (int64_t)a.batch * a.heads * a.queries;
  auto request = [&](int unit) {
    const int head = shared_head * group + unit / each, q0 = from + unit % each * ROWS;
    next_q.load((const T*)a.q + b * a.qs[0] + head * a.qs[1] + q0 * a.qs[2], a.qs[2], a.queries - q0, a.dim);
    next_g.load((const T*)a.grad + b * a.gs[0] + head * a.gs[1] + q0 * a.gs[2], a.gs[2], a.queries - q0, a.dim);
#pragma unroll
    for (int t = 0; t < NT; ++t)   // rows of the turned map are padded to whole tiles
      next_bucket[t].load(map + q0 + 16 * NT * h + 16 * t);
    if (threadIdx.x < ROWS) {
      const int q = q0 + threadIdx.x;
      const int64_t row = ((int64_t)b * a.heads + head) * a.queries + q;
      next_lse = INFINITY, next_delta = 0.f, next_rest = 0.f;
      // worked on in put: nothing waits here
      if (q < a.queries) next_lse = lse2[row], next_delta = delta[row], next_rest = rests[row];
    }
  };
  auto put = [&](int buffer) {
    next_q.store(queries[buffer]);
    next_g.store(grads[buffer]);
    if (threadIdx.x < ROWS) {   // lanes of the first wave
      const Lse lse(next_lse, next_rest, false, kLift<T>);
      row_lse[buffer][threadIdx.x] = -lse.off;
      row_delta[buffer][threadIdx.x] = -next_delta;
      row_factor[buffer][threadIdx.x] = lse.factor;
      const unsigned long long some = __ballot(lse.far);
      if (threadIdx.x == 0) lds.far[buffer] = some != 0;
    }
  };
  auto put_bias = [&](int unit) {
    table[threadIdx.x] = a.bias(shared_head * group + unit / each, threadIdx.x, __is_same(T, bf16));
  };
  if (begin < stop) {
    request(begin);
    put(0);
    put_bias(begin);
  }
  landed();
  __syncthreads();
  for (int unit = begin; unit < stop; ++unit) {
    const int now = (unit - begin) % 2, q0 = from + unit % each * ROWS;
    const bool more = unit + 1 < stop;
#pragma unroll
    for (int t = 0; t < NT; ++t) bucket[t] = next_bucket[t];
    request(more ? unit + 1 : unit);   // it has landed by `put`: until then no load is waited for
    const auto query_view = queries[now].view(lane), grad_view = grads[now].view(lane);
    const float *now_lse = row_lse[now] + 16 * NT * h, *now_delta = row_delta[now] + 16 * NT * h;
    const float* now_factor = row_factor[now] + 16 * NT * h;
    const bool some_far = __builtin_amdgcn_readfirstlane(lds.far[now]) != 0;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      floatx16 s = dot_tile<T, DP>(query_view, t, k, [&](int i) { return table[bucket[t][i]]; });
      const floatx16 e = dot_tile<T, DP>(grad_view, t, v, [&](int i) { return now_delta[16 * t + i]; });
      if (q0 < seen) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (q0 + 16 * NT * h + 16 * t + i < seen) s[i] = -INFINITY;
      }
      float p[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], a.scale2, now_lse[16 * t + i]));
      if (some_far) {
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] *= now_factor[16 * t + i];
      }
      {
        const Operand<T> w[2] = {rounded<T>(p), rounded<T>(p + 8)};
        add_columns<T>(dv, grad_view, t, w);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] *= e[i];   // ds
      if constexpr (__is_same(T, f16)) {
        // Held below 2: where a larger one comes, from there on below 2^-3, so that the sums seldom change theirs.
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(p[i]));
        if (__any(most * held >= 2.f)) {
          most = max_halves(most);   // the halves share the sums
          const unsigned exponent = std::min(__float_as_uint(most) >> 23, 240u);
          const float next = most * held >= 2.f ? __uint_as_float((250 - exponent) << 23) : held;
          const float by = next / held;
#pragma unroll
          for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) dk[d][i] *= by;
          held = next;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] *= held;
      }
      const Operand<T> w[2] = {rounded<T>(p), rounded<T>(p + 8)};
      add_columns<T>(dk, query_view, t, w);
    }
    if (more) put(1 - now);
    __syncthreads();
    if (more && (unit + 1) % each == 0) {   // the next tile is another head's
      put_bias(unit + 1);
      __syncthreads();
    }
  }
  if (key >= a.keys) return;
  if (key >= len) {   // columns of keys that do not count
    clear(dk);
    clear(dv);
  }
  const float back = exp2f(-kLift<T>), back_k = a.scale * (back / held);
  if (splits > 1) {
    const int64_t rows = (int64_t)a.batch * a.key_heads * a.keys, row = (int64_t)work.head * a.keys + key;
    float* to = part + ((int64_t)work.split * 2 * rows + row) * a.dim;
    store_columns<float, DP>(to, a.dim, 0, a.dim, lane, dk, back_k);
    store_columns<float, DP>(to + rows * a.dim, a.dim, 0, a.dim, lane, dv, back);
    return;
  }
  if (a.dk)
    store_columns<T, DP>((T*)a.dk + b * a.dks[0] + shared_head * a.dks[1], a.dks[2], key, a.dim, lane, dk, back_k);
  if (a.dv) store_columns<T, DP>((T*)a.dv + b * a.dvs[0] + shared_head * a.dvs[1], a.dvs[2], key, a.dim, lane, dv, back);
}

// ------------------------------------------------------------------------------------------ splits
// out[row] = sum of the splits' parts in their order, four values a thread; part [split][.. rows ..][dim], `pitch`
// values from split to split.
template <typename T>
__global__ __launch_bounds__(256) void join_splits(const float* part, int64_t pitch, int splits, T* out, int64_t s0,
                                                   int64_t s1, int64_t s2, int64_t rows, int tokens, int heads, int dim) {
  const int per_row = dim / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / per_row;
  if (row >= rows) return;
  const int d = (int)(i % per_row) * 4;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) {
    float y[4];
    load_pack<float, 4>(part + s * pitch + row * dim + d, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += y[e];
  }
  const int64_t bh = row / tokens, token = row % tokens;
  store_pack<T, 4>(out + bh / heads * s0 + bh % heads * s1 + token * s2 + d, x);
}

struct Space {
  int query_splits, key_splits, pitch, size_parts;
  int64_t sizes, delta, lse2, parts, turned, part, total;
};
Space space_of(const sdk_bucket_attention* a) {
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  Space w;
  const int64_t tile = 32 * (a->dtype == SDK_F32 ? kParts<float> : kParts<bf16>), rows = 32 * kWaves;
  const int64_t q_rows = a->batch * a->heads * a->queries, k_rows = a->batch * a->key_heads * a->keys;
  const int64_t q_groups = a->batch * a->heads * ceil_div(a->queries, rows);
  // workgroups that run at once, by the registers of their waves
  const bool wide = a->dtype == SDK_F32;
  const int64_t query_slots = a->dim <= (wide ? 64 : 96) ? 512 : 256, key_slots = a->dim <= (wide ? 32 : 64) ? 512 : 256;
  w.query_splits = parts_of(q_groups, ceil_div(a->keys, tile), query_slots, false);
  w.key_splits = parts_of(a->batch * a->key_heads * ceil_div(a->keys, rows),
                          a->heads / a->key_heads * ceil_div(a->queries, tile), key_slots, a->causal);
  w.pitch = (int)ceil_div(a->queries, 64) * 64;
  w.size_parts = (int)std::min<int64_t>(kMostParts, std::max<int64_t>(1, ceil_div(a->keys, 128)));
  w.sizes = 0;
  w.delta = a->dtype == SDK_F16 ? up(a->batch * a->key_heads * w.size_parts * 4) : 0;
  w.lse2 = w.delta + up(q_rows * 4);
  w.parts = w.lse2 + up(q_rows * 4);
  w.turned = w.parts + up(q_groups * w.query_splits * a->buckets * 4);
  w.part = w.turned + up((a->map_strides[0] ? a->batch : 1) * a->keys * w.pitch);
  // the parts of dq, then those of dk and dv, lie in the same place
  const int64_t q_part = w.query_splits > 1 ? w.query_splits * q_rows : 0;
  const int64_t k_part = w.key_splits > 1 ? w.key_splits * 2 * k_rows : 0;
  w.total = w.part + up(std::max(q_part, k_part) * a->dim * 4);
  return w;
}

template <typename T, int DP, int COLUMNS>
int launch_grad_queries(const Attention& d, const Space& w, char* ws, hipStream_t s) {
  const size_t smem = (size_t)kWaves * (d.buckets + 1) * COLUMNS * sizeof(float);
  const int tiles = (int)ceil_div(d.queries, 32 * kWaves);
  auto* kernel = grad_queries<T, DP, COLUMNS>;
  if (smem > (32 << 10)) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != hipSuccess) return fail(SDK_ERR_DEVICE, "LDS of %zu bytes: %s", smem, hipGetErrorString(e));
  }
  kernel<<<dim3((unsigned)tiles * (unsigned)(d.batch * d.heads) * w.query_splits), dim3(kThreads), smem, s>>>(
      d, w.query_splits, tiles, (const float*)(ws + w.delta), (const float*)(ws + w.lse2),
      (const float*)(ws + w.sizes), w.size_parts, (float*)(ws + w.part), (float*)(ws + w.parts));
  return SDK_OK;
}

template <typename T>
void launch_join(const Attention& d, const float* part, int64_t pitch, int splits, void* out, const int64_t (&st)[3],
                 int tokens, int heads, hipStream_t s) {
  const int64_t rows = (int64_t)d.batch * heads * tokens;
  launch(join_splits<T>, dim3((unsigned)ceil_div(rows * (d.dim / 4), 256)), dim3(256), s, part, pitch, splits, (T*)out,
         st[0], st[1], st[2], rows, tokens, heads, d.dim);
}

template <typename T>
int run(const sdk_bucket_attention* a, const Attention& d, char* ws, hipStream_t s) {
  const Space w = space_of(a);
  const bool any = a->batch > 0 && a->queries > 0;
  const int64_t rows = a->batch * a->heads * a->queries;
  float *delta = (float*)(ws + w.delta), *lse2 = (float*)(ws + w.lse2), *part = (float*)(ws + w.part);
  // As many columns as 66 KB hold.  Beside the tiles that leaves two workgroups a CU up to 59, 120 and 242 buckets with 64,
  // 32 and 16 columns (heads of 64 in 16 bits; 51, 104 and 210 padded to 96, 50, 102 and 206 in float32), one beyond, which
  // the slots that parts are planned with (space_of) do not know.  The backward of 16 heads of 64, 8192 x 8192 pairs: 48
  // buckets 1472 us, 59 1467, 60 1784, 64 1788, 65 1705, 120 1742, 121 2279, 129 2200, 242 2242, 243 3113; without the table
  // 1241 to 1345.
  const int columns = !a->grad_table ? 0 : a->buckets <= 64 ? 64 : a->buckets <= 128 ? 32 : 16;
  if (any) {
    constexpr int LANES = 128 / kWide<T>;
    const int64_t groups = std::min(ceil_div(rows, 256 / LANES), most_groups(256));
    launch(row_terms<T, LANES>, dim3((unsigned)groups), dim3(256), s, d, delta, lse2);
    if (a->grad_query || a->grad_table) {
      if (__is_same(T, f16))
        launch(value_sizes, dim3((unsigned)(a->batch * a->key_heads) * w.size_parts), dim3(256), s, d, w.size_parts,
               (float*)(ws + w.sizes));
      int rc = SDK_OK;
      ATTENTION_DIM(a->dim, rc = columns == 0    ? launch_grad_queries<T, DP, 0>(d, w, ws, s)
                                 : columns == 64 ? launch_grad_queries<T, DP, 64>(d, w, ws, s)
                                 : columns == 32 ? launch_grad_queries<T, DP, 32>(d, w, ws, s)
                                                 : launch_grad_queries<T, DP, 16>(d, w, ws, s));
      if (rc != SDK_OK) return rc;
      if (w.query_splits > 1 && a->grad_query)
        launch_join<T>(d, part, rows * a->dim, w.query_splits, d.dq, d.dqs, d.queries, d.heads, s);
    }
  }
  if (a->grad_table)
    launch(join_table<T>, dim3((unsigned)std::min(a->heads * a->buckets, most_groups(256))), dim3(256), s, d,
           any ? (int)ceil_div(a->queries, 32 * kWaves) * w.query_splits : 0, (const float*)(ws + w.parts));
  if ((a->grad_key || a->grad_value) && a->batch > 0 && a->keys > 0) {
    uint8_t* turned = (uint8_t*)(ws + w.turned);
    const int tiles = (int)ceil_div(a->keys, 32 * kWaves);
    if (any) {
      const int64_t blocks = w.pitch / 64 * ceil_div(a->keys, 64);   // fewer than 2^31
      launch(turn_map, dim3((unsigned)std::min(blocks, most_groups(256)), (unsigned)(a->map_strides[0] ? a->batch : 1)),
             dim3(256), s, d, turned, w.pitch, (unsigned)blocks);
    }
    ATTENTION_DIM(a->dim, launch(grad_keys<T, DP>, dim3((unsigned)(tiles * a->batch * a->key_heads) * w.key_splits),
                                 dim3(kThreads), s, d, w.key_splits, tiles, (const float*)delta, (const float*)lse2,
                                 (const uint8_t*)turned, w.pitch, part));
    if (w.key_splits > 1) {
      const int64_t values = a->batch * a->key_heads * a->keys * a->dim;
      if (a->grad_key) launch_join<T>(d, part, 2 * values, w.key_splits, d.dk, d.dks, d.keys, d.key_heads, s);
      if (a->grad_value)
        launch_join<T>(d, part + values, 2 * values, w.key_splits, d.dv, d.dvs, d.keys, d.key_heads, s);
    }
  }
  SDK_LAUNCH_CHECK("bucket_attention_backward");
  return SDK_OK;
}

}  // namespace

size_t backward_bytes(const sdk_bucket_attention* a) { return (size_t)space_of(a).total; }

int run_backward(const sdk_bucket_attention* a, void* workspace, hipStream_t s) {
  const Attention d = on_device(a);
  SDK_DISPATCH_TOKEN_DTYPE(a->dtype, return run<T>(a, d, (char*)workspace, s));
}

}  // namespace token
}  // namespace sdk
