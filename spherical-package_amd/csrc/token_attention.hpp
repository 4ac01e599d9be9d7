// Matrix operands, tiles in LDS and addressing of the attention kernels.
//
// One product computes D[i][j] += sum_k A[i][k] B[k][j] for a 32 x 32 tile and 16 values of k.  Lane l of the
// wave supplies 8 values of k of row i = l % 32 of A and of column j = l % 32 of B, and holds
// D[8 (v / 4) + 4 (l / 32) + v % 4][l % 32], v = 0 .. 15.  What B's columns are stays in registers (queries in
// the kernels that walk the keys, keys in the one that walks the queries); rows of A come from LDS.
//
// Rows are placed so that a lane's 16 values of a tile are 16 consecutive tokens: of a tile of ROWS = 32 NT
// tokens, lane half h has in part t the tokens 16 NT h + 16 t + (0 .. 15).  Token k of the tile therefore lies in
// row `row_of(k)`.  A lane reads the buckets of its 16 pairs as 16 consecutive bytes, and the values it holds are
// the next product's B operand as they are: the sum's index may be permuted if A's rows are named alike.
#pragma once
#include <algorithm>
#include <type_traits>

#include "sdk_mfma.hpp"
#include "token_types.hpp"

namespace sdk {
namespace token {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Eight values of k of an operand.  float32 runs on the bf16 matrix unit: a float is the exact sum of three bf16
// pieces (hi, mid, lo), and six of the nine products of pieces, all but those below 2^-26 of the product, are added
// in float32.  (The unit's own float32 product takes 512 cycles for 16 values of k, these six 192.)
template <typename T>
struct Operand {
  unsigned u[4];
};
template <>
struct Operand<float> {
  Operand<bf16> piece[3];
};

__device__ __forceinline__ floatx16 product(const Operand<bf16>& a, const Operand<bf16>& b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}
__device__ __forceinline__ floatx16 product(const Operand<f16>& a, const Operand<f16>& b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                0);
}
__device__ __forceinline__ floatx16 product(const Operand<float>& a, const Operand<float>& b, floatx16 c) {
  c = product(a.piece[2], b.piece[0], c);
  c = product(a.piece[0], b.piece[2], c);
  c = product(a.piece[1], b.piece[1], c);
  c = product(a.piece[1], b.piece[0], c);
  c = product(a.piece[0], b.piece[1], c);
  return product(a.piece[0], b.piece[0], c);
}

// Two floats' pieces, packed.  Each piece is rounded to nearest, so what is left out has either sign.
__device__ __forceinline__ void split_pair(float x, float y, unsigned& hi, unsigned& mid, unsigned& lo) {
  hi = pack_bf16x2(x, y);
  x -= __uint_as_float(hi << 16), y -= __uint_as_float(hi & 0xffff0000u);
  mid = pack_bf16x2(x, y);
  x -= __uint_as_float(mid << 16), y -= __uint_as_float(mid & 0xffff0000u);
  lo = pack_bf16x2(x, y);
}

template <typename T>
__device__ __forceinline__ Operand<T> rounded(const float* f) {
  Operand<T> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      split_pair(f[2 * i], f[2 * i + 1], r.piece[0].u[i], r.piece[1].u[i], r.piece[2].u[i]);
    } else if constexpr (__is_same(T, bf16)) {
      r.u[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    } else {
      const f32x2 v = {f[2 * i], f[2 * i + 1]};
      r.u[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, f16x2));
    }
  }
  return r;
}

// Eight consecutive values in memory, 16-byte aligned; `in` false: zeros, not read.
template <typename T>
__device__ __forceinline__ Operand<T> load_operand(const T* p, bool in) {
  Operand<T> r = {};
  if (in) {
    if constexpr (sizeof(T) == 4) {
      float f[8];
      load_pack<float, 4>(p, *reinterpret_cast<float(*)[4]>(f));
      load_pack<float, 4>(p + 4, *reinterpret_cast<float(*)[4]>(f + 4));
      r = rounded<T>(f);
    } else {
      r = *reinterpret_cast<const Operand<T>*>(__builtin_assume_aligned(p, 16));
    }
  }
  return r;
}

template <int NT>
__device__ __forceinline__ int row_of(int token) {
  const int h = token / (16 * NT), t = token / 16 % NT, v = token % 16;
  return 32 * t + 8 * (v / 4) + 4 * h + v % 4;
}

// A tile of 32 NT tokens, DP values each, in LDS; float32 as three planes of pieces.  16 bytes beside each row
// spread rows over the banks.
template <typename T, int DP, int NT>
struct Tile {
  using Half = std::conditional_t<sizeof(T) == 4, bf16, T>;
  static constexpr int kRows = 32 * NT, kStride = DP + 8, kPlanes = sizeof(T) == 4 ? 3 : 1;
  Half v[kPlanes][kRows * kStride];

  // What a lane reads of a tile, by its own addresses: everything but the lane's part is a constant offset.
  struct View {
    const Half *row, *column;

    // rows of A, values 16 c + 8 h .. + 7
    __device__ __forceinline__ Operand<T> rows(int t, int c) const {
      const int at = 32 * t * kStride + 16 * c;
      Operand<T> r;
      if constexpr (kPlanes == 3) {
#pragma unroll
        for (int i = 0; i < 3; ++i) r.piece[i] = straight<bf16>(row + i * kRows * kStride + at);
      } else {
        r = straight<T>(row + at);
      }
      return r;
    }
    // the first piece of float32 rows alone
    __device__ __forceinline__ Operand<bf16> first_piece(int t, int c) const {
      return straight<bf16>(row + 32 * t * kStride + 16 * c);
    }
    // columns of the tile as A: row i of A = column 32 d + i, k = the 16 tokens that registers 8 half .. 8 half + 7
    // of part t hold
    __device__ __forceinline__ Operand<T> columns(int t, int half, int d) const {
      const int at = (32 * t + 16 * half) * kStride + 32 * d;
      Operand<T> r;
      if constexpr (kPlanes == 3) {
#pragma unroll
        for (int i = 0; i < 3; ++i) r.piece[i] = turned<bf16>(column + i * kRows * kStride + at);
      } else {
        r = turned<T>(column + at);
      }
      return r;
    }
  };
  __device__ __forceinline__ View view(int lane) const {
    return {v[0] + (lane % 32) * kStride + 8 * (lane / 32),
            v[0] + (4 * (lane / 32) + lane % 16 / 4) * kStride + 16 * (lane / 16 % 2) + 4 * (lane % 4)};
  }
  // kWide values of a token from d on
  __device__ __forceinline__ void store(int token, int d, const Pack<T, kWide<T>>& x) {
    const int at = row_of<NT>(token) * kStride + d;
    if constexpr (kPlanes == 3) {
      unsigned p[3][2];
      split_pair(x.v[0], x.v[1], p[0][0], p[1][0], p[2][0]);
      split_pair(x.v[2], x.v[3], p[0][1], p[1][1], p[2][1]);
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<uint2*>(v[i] + at) = make_uint2(p[i][0], p[i][1]);
    } else {
      *reinterpret_cast<Pack<T, kWide<T>>*>(v[0] + at) = x;
    }
  }

 private:
  template <typename H>
  __device__ static __forceinline__ Operand<H> straight(const Half* p) {
    return *reinterpret_cast<const Operand<H>*>(__builtin_assume_aligned(p, 16));
  }
  template <typename H>
  __device__ static __forceinline__ Operand<H> turned(const Half* p) {
    const Bf16Frag f = tr_frag((const char*)p, (const char*)(p + 8 * kStride));
    Operand<H> r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.u[i] = f.u[i];
    return r;
  }
};

// begin(v) plus the products of the tile's rows with x.  float32: the five small products of each pair first, from
// zero, and `begin` last: the unit drops what falls below the sum's last bit, which adds up over the steps.  The
// rows' first pieces are read twice for it (the fence keeps them from staying in registers).
template <typename T, int DP, typename View, typename Begin>
__device__ __forceinline__ floatx16 dot_tile(const View& view, int t, const Operand<T> (&x)[DP / 16], Begin begin) {
  floatx16 c;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int v = 0; v < 16; ++v) c[v] = 0.f;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const Operand<T> a = view.rows(t, i);
      c = product(a.piece[2], x[i].piece[0], c);
      c = product(a.piece[0], x[i].piece[2], c);
      c = product(a.piece[1], x[i].piece[1], c);
      c = product(a.piece[1], x[i].piece[0], c);
      c = product(a.piece[0], x[i].piece[1], c);
    }
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) c = product(view.first_piece(t, i), x[i].piece[0], c);
#pragma unroll
    for (int v = 0; v < 16; ++v) c[v] += begin(v);
  } else {
#pragma unroll
    for (int v = 0; v < 16; ++v) c[v] = begin(v);
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) c = product(view.rows(t, i), x[i], c);
  }
  return c;
}

// acc += the tile's columns times the 16 weights of part t.  float32: summed apart for each tile, the small products
// first, and then added: a chain of two roundings a tile instead of twelve.
template <typename T, int D, typename View>
__device__ __forceinline__ void add_columns(floatx16 (&acc)[D], const View& view, int t, const Operand<T> (&w)[2]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      floatx16 c;
#pragma unroll
      for (int v = 0; v < 16; ++v) c[v] = 0.f;
      Operand<T> a[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        a[half] = view.columns(t, half, d);
        c = product(a[half].piece[2], w[half].piece[0], c);
        c = product(a[half].piece[0], w[half].piece[2], c);
        c = product(a[half].piece[1], w[half].piece[1], c);
        c = product(a[half].piece[1], w[half].piece[0], c);
        c = product(a[half].piece[0], w[half].piece[1], c);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) c = product(a[half].piece[0], w[half].piece[0], c);
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[d][v] += c[v];
    }
  } else {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int d = 0; d < D; ++d) acc[d] = product(view.columns(t, half, d), w[half], acc[d]);
  }
}

// A tile on its way from memory to LDS, in the registers of the workgroup's THREADS threads.  The tile's `left`
// tokens and `dim` values are read, zeros stand for the others: a buffer descriptor that ends with the last token
// tells them apart, and a thread's vectors lie at the same 32-bit offsets of every tile (the host checks that 64
// tokens span less than 2^31 bytes).  Tile and descriptor are the workgroup's own, in scalar registers.
template <typename T, int DP, int NT, int THREADS>
struct Carry {
  static constexpr int kVectors = DP / kWide<T>, kCount = 32 * NT * kVectors / THREADS;
  static_assert(32 * NT * kVectors % THREADS == 0, "every thread carries as many vectors");
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  u32x4 v[kCount];
  unsigned at[kCount];

  __device__ __forceinline__ Carry(int64_t stride, int dim) {
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int i = n * THREADS + threadIdx.x, d = i % kVectors * kWide<T>;
      at[n] = d < dim ? (unsigned)((i / kVectors) * (int)stride + d) * (unsigned)sizeof(T) : 0xfffffff0u;
    }
  }
  __device__ __forceinline__ void load(const T* tile, int64_t stride, int left, int dim) {
    const int rows = std::min(left, 32 * NT);
    const unsigned bytes = rows > 0 ? (unsigned)((rows - 1) * (int)stride + dim) * (unsigned)sizeof(T) : 0u;
    const __amdgpu_buffer_rsrc_t all = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(tile), 0, bytes, 0x00020000);
#pragma unroll
    for (int n = 0; n < kCount; ++n) v[n] = __builtin_amdgcn_raw_buffer_load_b128(all, at[n], 0, 0);
  }
  __device__ __forceinline__ void store(Tile<T, DP, NT>& tile) const {
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int i = n * THREADS + threadIdx.x;
      tile.store(i / kVectors, i % kVectors * kWide<T>, __builtin_bit_cast(Pack<T, kWide<T>>, v[n]));
    }
  }
};

// The buckets of a lane's 16 pairs: 16 bytes at any address; near the map's end byte by byte.
struct Buckets {
  unsigned w[4];
  __device__ __forceinline__ void load(const uint8_t* row) { __builtin_memcpy(w, row, 16); }
  __device__ __forceinline__ void load(const uint8_t* row, int left) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = 0;
#pragma unroll 1
    for (int i = 0; i < 16 && i < left; ++i) {
      const unsigned x = (unsigned)row[i] << (8 * (i % 4));
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] |= i / 4 == k ? x : 0u;
    }
  }
  __device__ __forceinline__ unsigned operator[](int v) const { return w[v / 4] >> (8 * (v % 4)) & 255u; }
};
// The buckets of a tile's parts from key `first` on.
template <int NT>
__device__ __forceinline__ void load_buckets(Buckets (&b)[NT], const uint8_t* row, int first, int count, int h) {
  if (first + 32 * NT <= count) {
#pragma unroll
    for (int t = 0; t < NT; ++t) b[t].load(row + first + 16 * NT * h + 16 * t);
  } else {
#pragma unroll
    for (int t = 0; t < NT; ++t)
      b[t].load(row + first + 16 * NT * h + 16 * t, count - (first + 16 * NT * h + 16 * t));
  }
}

// The value of the lane 32 away.
__device__ __forceinline__ float other_half(float x) {
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(threadIdx.x % 64 < 32 ? r[1] : r[0]);
}
// Largest of the lane's and the other half's value (NaN: the other one).
__device__ __forceinline__ float max_halves(float x) {
  const unsigned u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// sum + the eight weights f, as the product takes them (16-bit: rounded, two at a time).
template <typename T>
__device__ __forceinline__ float add_weights(const Operand<T>& w, const float* f, float sum) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += f[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (__is_same(T, bf16)) {
        const bf16x2 one = {(__bf16)1.f, (__bf16)1.f};
        sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w.u[i]), one, sum, false);
      } else {
        const f16x2 one = {(_Float16)1.f, (_Float16)1.f};
        sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w.u[i]), one, sum, false);
      }
    }
  }
  return sum;
}

// A row's sum of exponentials is 2^level * sum.  The level is a whole number at or above (or little below) the largest
// score in powers of two: weights against two levels differ by a power of two, so that they round to 16 bits alike in
// every part of the keys and in the backward.  Kept as (level, log2 sum); a row without pairs: (-inf, 0).
__device__ __forceinline__ float2 lse_of(float level, float sum) {
  return sum > 0.f || sum != sum ? make_float2(level, log2f(sum)) : make_float2(-INFINITY, 0.f);
}

// The weights of a row as the product takes them, as floats again.
template <typename T>
__device__ __forceinline__ void as_rounded(float (&p)[16]) {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const Operand<T> w = rounded<T>(p + 8 * half);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (__is_same(T, bf16)) {
          p[8 * half + 2 * i] = __uint_as_float(w.u[i] << 16);
          p[8 * half + 2 * i + 1] = __uint_as_float(w.u[i] & 0xffff0000u);
        } else {
          const f16x2 x = __builtin_bit_cast(f16x2, w.u[i]);
          p[8 * half + 2 * i] = (float)x[0];
          p[8 * half + 2 * i + 1] = (float)x[1];
        }
      }
    }
  }
}

// What the kernels take of sdk_bucket_attention; scale2 = scale * log2(e).
struct Attention {
  const void *q, *k, *v, *table, *out, *grad;
  void* rest;
  const uint8_t* map;
  const int32_t* lengths;
  void *dq, *dk, *dv, *dtable;
  float* lse;
  int64_t qs[3], ks[3], vs[3], os[3], gs[3], dqs[3], dks[3], dvs[3], ms[2];
  int queries, keys, batch, heads, key_heads, dim, buckets, causal, table_float;
  float scale, scale2, limit;

  __device__ __forceinline__ int length(int b) const {
    if (!lengths) return keys;
    const int n = __builtin_amdgcn_readfirstlane(lengths[b]);
    return n < 0 ? 0 : n > keys ? keys : n;
  }
  // bias / scale of a bucket: scores enter the softmax as scale2 * (q k + bias / scale).  Finite biases of 2^20 powers
  // of two or more, as masks have them, become one value +-limit, a power of two: limit * scale2 is exact, so that
  // the level of a row of nothing else is too, and its pairs weigh the same.
  __device__ __forceinline__ float bias(int head, int bucket, bool half_is_bf16) const {
    if (bucket >= buckets) return -INFINITY;
    const int64_t at = (int64_t)head * buckets + bucket;
    const float x = table_float ? ((const float*)table)[at]
                                : half_is_bf16 ? (float)((const bf16*)table)[at] : (float)((const f16*)table)[at];
    if (fabsf(x) < INFINITY && fabsf(x) > 0x1p20f * 0.6931472f) return x < 0.f ? -limit : limit;
    return x / scale;
  }
};

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kTable = 256;

template <typename T>
constexpr int kParts = sizeof(T) == 4 ? 1 : 2;   // 32-token parts of a tile

// A wave's 32 columns of B: row `row` of a tensor, values 16 c + 8 h .. + 7 in operand c; zeros unless `in`.
template <typename T, int DP>
__device__ __forceinline__ void load_columns(Operand<T> (&x)[DP / 16], const T* base, int64_t stride, int row, bool in,
                                             int dim, int lane) {
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
    const int d = 16 * c + 8 * (lane / 32);
    x[c] = load_operand<T>(base + row * stride + d, in && d < dim);
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

// The same for the output: rounded, and, where `rest` is not NULL, what the rounding took.
template <typename T, int DP>
__device__ __forceinline__ void store_output(T* base, T* rest, int64_t stride, int64_t row, int dim, int lane,
                                             floatx16 (&acc)[DP / 32], float by) {
  store_columns<T, DP>(base, stride, row, dim, lane, acc, by);
  if constexpr (sizeof(T) == 2)
    if (rest) {
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const float x = acc[d][v] * by;
          acc[d][v] = x - (float)(T)x;
        }
      store_columns<T, DP>(rest, stride, row, dim, lane, acc, 1.f);
    }
}

template <int N>
__device__ __forceinline__ void clear(floatx16 (&x)[N]) {
#pragma unroll
  for (int d = 0; d < N; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) x[d][v] = 0.f;
}

// Waits for every load so far.  Before a loop: the compiler, which cannot tell a first step from a later one, would
// otherwise wait in each step for what the loop uses of before it, and with it for the step's own requests.
__device__ __forceinline__ void landed() { __builtin_amdgcn_s_waitcnt(0x0f70); }   // vmcnt(0) alone

// Where split `split` of `splits` begins among `tiles`.
__device__ __forceinline__ int split_at(int tiles, int split, int splits) {
  return (int)((int64_t)tiles * split / splits);
}

// Which tile of which head (counted with the batch) and which split of it a workgroup takes.  In causal calls
// the tiles differ in work: the longest ones first (`ascending`: those with small numbers), all heads' together.
struct Work {
  int tile, head, split;
  __device__ __forceinline__ Work(int tiles, int heads, int splits, bool causal, bool ascending) {
    if (causal) {
      unsigned id = blockIdx.x;
      head = (int)(id % (unsigned)heads);
      id /= (unsigned)heads;
      split = (int)(id % (unsigned)splits);
      tile = (int)(id / (unsigned)splits);
      if (!ascending) tile = tiles - 1 - tile;
    } else {
      unsigned id = by_die(blockIdx.x, gridDim.x);
      split = (int)(id % (unsigned)splits);
      id /= (unsigned)splits;
      tile = (int)(id % (unsigned)tiles);
      head = (int)(id / (unsigned)tiles);
    }
  }
};

// host
// Parts that a walk of `steps` tiles is dealt to, for `groups` workgroups without and `slots` that run at once: the
// fewest rounds of workgroups times the tiles of a round; a part costs about four tiles more (its operands, its sums
// in memory), and has four at least.  More workgroups than that stay whole: 1152 of the forward at 4608 x 4608 pairs
// as two parts each took 284 us and a join for 265.  balance: two parts at least where all run at once (causal walks
// differ in length: 256 workgroups of dk and dv take 1.54 times as long whole as in two parts, in four 1.15 times).
inline int parts_of(int64_t groups, int64_t steps, int64_t slots, bool balance) {
  if (groups == 0 || groups > slots || (groups == slots && !balance)) return 1;
  int64_t best = 1, least = INT64_MAX;
  for (int64_t s = balance && steps >= 8 ? 2 : 1; s <= 16 && (s <= 2 || s * 4 <= steps); ++s) {
    const int64_t cost = ceil_div(groups * s, slots) * (ceil_div(steps, s) + 4);
    if (cost < least) least = cost, best = s;
  }
  return (int)best;
}

Attention on_device(const sdk_bucket_attention* a);
bool few_rows(const sdk_bucket_attention* a);       // whether a key head's rows go to the kernel of few queries
int forward_splits(const sdk_bucket_attention* a);
size_t backward_bytes(const sdk_bucket_attention* a);
int run_forward(const sdk_bucket_attention* a, void* workspace, hipStream_t s);
int run_backward(const sdk_bucket_attention* a, void* workspace, hipStream_t s);

// Runs the statement with DP, the padded dim, a multiple of the products' 32 columns.  96 beside 128: 2 x 16 heads of 80,
// 2048 tokens, 75 us for 93 forward and 398 for 525 with gradients in bfloat16; 1024 tokens in float32 411 for 617, whose
// registers of three pieces then fit.
#define ATTENTION_DIM(dim, ...)                                  \
  do {                                                           \
    if ((dim) <= 32) { constexpr int DP = 32; __VA_ARGS__; }     \
    else if ((dim) <= 64) { constexpr int DP = 64; __VA_ARGS__; } \
    else if ((dim) <= 96) { constexpr int DP = 96; __VA_ARGS__; } \
    else { constexpr int DP = 128; __VA_ARGS__; }                \
  } while (0)

}  // namespace token
}  // namespace sdk
