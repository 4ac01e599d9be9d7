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
#include "sdk_mfma.hpp"
#include "token_types.hpp"

namespace sdk {
namespace token {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Eight values of k of an operand.
template <typename T>
struct Operand {
  unsigned u[4];
};
template <>
struct Operand<float> {
  float u[8];
};

__device__ __forceinline__ floatx16 product(const Operand<bf16>& a, const Operand<bf16>& b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}
__device__ __forceinline__ floatx16 product(const Operand<f16>& a, const Operand<f16>& b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                0);
}
// float32: eight products of two values of k each, value s of both lane halves in product s.
__device__ __forceinline__ floatx16 product(const Operand<float>& a, const Operand<float>& b, floatx16 c) {
#pragma unroll
  for (int s = 0; s < 8; ++s) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.u[s], b.u[s], c, 0, 0, 0);
  return c;
}

template <typename T>
__device__ __forceinline__ Operand<T> rounded(const float* f) {
  Operand<T> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.u[i] = f[i];
  } else if constexpr (__is_same(T, bf16)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.u[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x2 v = {f[2 * i], f[2 * i + 1]};
      r.u[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, f16x2));
    }
  }
  return r;
}

template <typename T>
__device__ __forceinline__ Operand<T> zeros() {
  Operand<T> r;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(r.u) / 4); ++i) r.u[i] = 0;
  return r;
}

// Eight consecutive values, 16-byte aligned (in memory or LDS).
template <typename T>
__device__ __forceinline__ Operand<T> load_operand(const T* p) {
  return *reinterpret_cast<const Operand<T>*>(__builtin_assume_aligned(p, 16));
}

template <int NT>
__device__ __forceinline__ int row_of(int token) {
  const int h = token / (16 * NT), t = token / 16 % NT, v = token % 16;
  return 32 * t + 8 * (v / 4) + 4 * h + v % 4;
}

// A tile of 32 NT tokens, DP values each, in LDS.  16 bytes beside each row spread rows over the banks.
template <typename T, int DP, int NT>
struct Tile {
  static constexpr int kRows = 32 * NT, kStride = DP + 16 / (int)sizeof(T);
  T v[kRows * kStride];

  // rows of A, values 16 c + 8 h .. + 7
  __device__ __forceinline__ Operand<T> rows(int t, int c, int lane) const {
    return load_operand<T>(v + (32 * t + lane % 32) * kStride + 16 * c + 8 * (lane / 32));
  }
  // columns of the tile as A: row i of A = column 32 d + i, k = the 16 tokens that registers 8 half .. 8 half + 7 of
  // part t hold
  __device__ __forceinline__ Operand<T> columns(int t, int half, int d, int lane) const {
    const int first = 32 * t + 16 * half + 4 * (lane / 32);
    Operand<T> r;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int s = 0; s < 8; ++s) r.u[s] = v[(first + s % 4 + 8 * (s / 4)) * kStride + 32 * d + lane % 32];
    } else {
      const T* p = v + (first + lane % 16 / 4) * kStride + 32 * d + 16 * (lane / 16 % 2) + 4 * (lane % 4);
      const Bf16Frag f = tr_frag((const char*)p, (const char*)(p + 8 * kStride));
#pragma unroll
      for (int i = 0; i < 4; ++i) r.u[i] = f.u[i];
    }
    return r;
  }
};

// A tile on its way from memory to LDS, in the registers of the workgroup's THREADS threads.  Tokens at or
// beyond `end` and values at or beyond `dim` are zeros and are not read.
template <typename T, int DP, int NT, int THREADS>
struct Carry {
  static constexpr int kVectors = DP / kWide<T>, kCount = 32 * NT * kVectors / THREADS;
  static_assert(32 * NT * kVectors % THREADS == 0, "every thread carries as many vectors");
  Pack<T, kWide<T>> v[kCount];

  __device__ __forceinline__ void load(const T* base, int64_t stride, int64_t first, int64_t end, int dim) {
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int at = n * THREADS + threadIdx.x, token = at / kVectors, d = at % kVectors * kWide<T>;
      if (first + token < end && d < dim) {
        v[n] = *reinterpret_cast<const Pack<T, kWide<T>>*>(base + (first + token) * stride + d);
      } else {
#pragma unroll
        for (int e = 0; e < kWide<T>; ++e) v[n].v[e] = (T)0.f;
      }
    }
  }
  __device__ __forceinline__ void store(Tile<T, DP, NT>& tile) const {
#pragma unroll
    for (int n = 0; n < kCount; ++n) {
      const int at = n * THREADS + threadIdx.x, token = at / kVectors, d = at % kVectors * kWide<T>;
      *reinterpret_cast<Pack<T, kWide<T>>*>(&tile.v[row_of<NT>(token) * Tile<T, DP, NT>::kStride + d]) = v[n];
    }
  }
};

// The buckets of a lane's 16 pairs: 16 bytes at any address; at the map's end byte by byte.
struct Buckets {
  unsigned w[4];
  __device__ __forceinline__ void load(const uint8_t* row, int64_t first, int64_t count) {
    if (first + 16 <= count) {
      __builtin_memcpy(w, row + first, 16);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (first + i < count) w[i / 4] |= (unsigned)row[first + i] << (8 * (i % 4));
    }
  }
  __device__ __forceinline__ unsigned operator[](int v) const { return w[v / 4] >> (8 * (v % 4)) & 255u; }
};

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

// Workgroups follow each other round the eight dies; consecutive tiles of one head share its keys and values, so
// each die gets a consecutive range of tiles.
__device__ __forceinline__ unsigned by_die(unsigned id, unsigned count) {
  const unsigned die = id % 8, each = count / 8, more = count % 8;
  return die * each + (die < more ? die : more) + id / 8;
}

// What the kernels take of sdk_bucket_attention; scale2 = scale * log2(e).
struct Attention {
  const void *q, *k, *v, *table, *out, *grad;
  const uint8_t* map;
  const int32_t* lengths;
  void *dq, *dk, *dv, *dtable;
  float* lse;
  int64_t qs[3], ks[3], vs[3], os[3], gs[3], dqs[3], dks[3], dvs[3], ms[2];
  int64_t queries, keys;
  int batch, heads, key_heads, dim, buckets, causal, table_float;
  float scale, scale2, limit;

  __device__ __forceinline__ int64_t length(int b) const {
    if (!lengths) return keys;
    const int64_t n = lengths[b];
    return n < 0 ? 0 : n > keys ? keys : n;
  }
  // bias / scale of a bucket: scores enter the softmax as scale2 * (q k + bias / scale)
  __device__ __forceinline__ float bias(int head, int bucket, bool half_is_bf16) const {
    if (bucket >= buckets) return -INFINITY;
    const int64_t at = (int64_t)head * buckets + bucket;
    const float x = table_float ? ((const float*)table)[at]
                                : half_is_bf16 ? (float)((const bf16*)table)[at] : (float)((const f16*)table)[at];
    const float y = x / scale;
    return fabsf(x) < INFINITY ? fminf(fmaxf(y, -limit), limit) : x;
  }
};

}  // namespace token
}  // namespace sdk
