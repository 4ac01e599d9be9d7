// Matrices made orthogonal by Newton-Schulz steps, alone and as the update of a Muon step over many parameters.
//
//   X_0 = U / (|U|_F + eps), smaller side first (k x l, k <= l)
//   S = X X^T      P = a I + b S + c S S^T      X' = P X          (odd polynomial of the singular values, S = S^T)
//   Muon: m = mu m + (1 - mu) g,  U = mu m + (1 - mu) g (nesterov) or m,
//         p = p (1 - lr decay) - lr sqrt(max(1, rows / columns)) X_steps
//
// Bound by the matrix unit: k^2 l + k^3 + 2 k^2 l operations a step, where of the symmetric S and P only the tiles on and
// above the diagonal are formed and written twice.
//
// Operands are float16 times 2^12.  float32 and float16 matrices take two pieces a value, v = hi + lo, and three products
// hi hi + hi lo + lo hi: 22 bits, 1.2e-6 of the result (701 x 1100) where float32 products leave 3.2e-6, at a third
// of the float16 rate where the float32 unit runs at an eighth.  bfloat16 matrices take one piece, but for the diagonals of S
// and P, whose rests are kept: they weigh whole rows, so their roundings add up where others average out (34 x 1855 would be
// 3.1e-3 off for 1.7e-3, 400 x 4000 2.6e-3 for 1.8e-3; of these the result's own rounding is 1.66e-3).  With D the rests of S,
// S S is formed as S S + D S + S D; with D those of P, X' = P X + D X.
//
// Entries of X, S and P have to stay below 16: no entry is larger than the largest singular value, which the coefficients
// alone bound (check_coefficients).  Sums are float32, of the norm double.
//
// 32 matrices of 640 x 640 to 640 x 2560, 39 million values, a step in float32: 1.81 to 1.88 ms, as cards differ.  S takes
// 110 us (820 TFLOP/s of products of pieces; its workgroups' sums are 640 to 2560 long), P 43 (710), X' 165 (910), momentum
// and norm 77, X_0 85, the last X' into the parameters 190.  A large library product of float16 reaches 1165.  bfloat16: 0.84
// to 0.90 ms (S 43 to 46, P 20 to 23, X' 68 to 74, 61, 78 and 100; without the diagonals' rests X' 65 to 70).
//
// All matrices of a call go through a stage in one launch; their table is a kernel argument.  Small ones go through all
// stages in a workgroup of their own, those of up to 16 rows on S alone, in 64 bits, where the steps are few.
#include <algorithm>
#include <cmath>
#include <functional>
#include <memory>
#include <new>
#include <type_traits>

#include "sdk_mfma.hpp"
#include "token_types.hpp"

namespace sdk {
namespace token {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kMatrices = 64;            // of a launch
constexpr float kScale = 4096.f, kDown = 1.f / 4096.f;
constexpr int kPad = 64;                 // sides in the workspace are multiples of it
constexpr int kPerGroup = 4096;          // values of a workgroup of the norm

struct Table {
  void* p[kMatrices];        // parameter, or result
  const void* g[kMatrices];  // gradient, or input
  float* m[kMatrices];       // momentum, or NULL
  int64_t at[kMatrices];     // byte offset of the matrix in the workspace
  int rows[kMatrices], columns[kMatrices];
  float rate[kMatrices];
  unsigned start[kMatrices]; // first workgroup of each matrix; beyond the last: more than the grid
};

struct Settings {
  float a, b, c, eps, mu, rest, keep;   // rest: 1 - mu; keep: 1 - lr decay
  int nesterov;
  int thin;                             // whether matrices of up to 16 rows go by S alone
  double a64, b64, c64;                 // a, b, c as they were given
};
static_assert(sizeof(Table) + sizeof(Settings) + 64 <= 4096, "kernel arguments are limited to 4 KB");

// The matrix of a workgroup.  Every lane reads one matrix's entries before the workgroup knows which is its own: one trip
// to the arguments where one for the index and one for the entries would follow each other (65 x 65: 85 us for 90).
struct Mine {
  int rows, columns;
  int64_t at, id;     // place in the workspace; which workgroup of the matrix
  char* p;
  const char* g;
  float* m;
  float rate;
};
__device__ __forceinline__ int64_t lane_of(int64_t x, int lane) {
  const unsigned low = __builtin_amdgcn_readlane((int)x, lane);
  return (int64_t)__builtin_amdgcn_readlane((int)(x >> 32), lane) << 32 | low;
}
__device__ __forceinline__ Mine matrix_of(const Table& t, unsigned group) {
  const int lane = threadIdx.x & 63;
  const unsigned start = t.start[lane];
  const int rows = t.rows[lane], columns = t.columns[lane];
  const int64_t at = t.at[lane], p = (int64_t)t.p[lane], g = (int64_t)t.g[lane], m = (int64_t)t.m[lane];
  const float rate = t.rate[lane];
  const int i = __builtin_amdgcn_readfirstlane(__popcll(__ballot(start <= group)) - 1);
  Mine mine;
  mine.rows = __builtin_amdgcn_readlane(rows, i), mine.columns = __builtin_amdgcn_readlane(columns, i);
  mine.at = lane_of(at, i), mine.id = group - (unsigned)__builtin_amdgcn_readlane((int)start, i);
  mine.p = (char*)lane_of(p, i), mine.g = (const char*)lane_of(g, i), mine.m = (float*)lane_of(m, i);
  mine.rate = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, rate), i));
  return mine;
}

// A row of an operand is a sequence of lines of 128 bytes: 64 values, or 32 values' hi and then their lo pieces.
template <bool SPLIT>
constexpr int kLine = SPLIT ? 32 : 64;

// Where the buffers of a matrix lie; sides padded with zeros to multiples of kPad.
struct Layout {
  int64_t k, l, kp, lp, x0, x1, s, p, s_rest, p_rest, sums, end;   // byte offsets from the matrix's place; X of even and
                                                                   // odd steps
  int64_t k_row, l_row;                             // bytes of a row of k and of l values
  __host__ __device__ Layout(int64_t rows, int64_t columns, bool split) {
    k = rows < columns ? rows : columns, l = rows < columns ? columns : rows;
    kp = (k + kPad - 1) / kPad * kPad, lp = (l + kPad - 1) / kPad * kPad;
    k_row = kp * (split ? 4 : 2), l_row = lp * (split ? 4 : 2);
    x0 = 0, x1 = x0 + kp * l_row, s = x1 + kp * l_row, p = s + kp * k_row;
    s_rest = p + kp * k_row, p_rest = s_rest + (split ? 0 : kp * 4), sums = p_rest + (split ? 0 : kp * 4);
    end = sums + ((rows * columns + kPerGroup - 1) / kPerGroup * 8 + 127) / 128 * 128;
  }
};

template <bool SPLIT>
__device__ __forceinline__ char* place_of(char* row, int64_t at) {
  return row + at / kLine<SPLIT> * 128 + at % kLine<SPLIT> * 2;
}

// v = hi + lo.  The value is kept from the compiler's view: it would form hi of a product twice, for the store from the
// rounded product and for lo by one fused rounding, and where the two differ lo misses a half of hi's last place (1e-5 of a
// matrix instead of 2e-7).
__device__ __forceinline__ void split_f16(float v, f16& hi, f16& lo) {
  asm("" : "+v"(v));
  hi = (f16)v;
  lo = (f16)(v - (float)hi);
}

// N consecutive values (a power of two up to 8, at a multiple of N) into or out of a row.
template <bool SPLIT, int N>
__device__ __forceinline__ void write_values(char* row, int64_t at, const float (&v)[N]) {
  char* to = place_of<SPLIT>(row, at);
  Pack<f16, N> hi, lo;
#pragma unroll
  for (int e = 0; e < N; ++e) split_f16(v[e], hi.v[e], lo.v[e]);
  *reinterpret_cast<Pack<f16, N>*>(to) = hi;
  if constexpr (SPLIT) *reinterpret_cast<Pack<f16, N>*>(to + 64) = lo;
}
template <bool SPLIT, int N>
__device__ __forceinline__ void read_values(const char* row, int64_t at, float (&v)[N]) {
  const char* from = place_of<SPLIT>(const_cast<char*>(row), at);
  const Pack<f16, N> hi = *reinterpret_cast<const Pack<f16, N>*>(from);
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = (float)hi.v[e];
  if constexpr (SPLIT) {
    const Pack<f16, N> lo = *reinterpret_cast<const Pack<f16, N>*>(from + 64);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] += (float)lo.v[e];
  }
}

// kScale / (norm + eps) for the sum of squares `sum`.  The norm may be beyond float32's largest value, so it and eps are
// taken down by a power of two, which changes no bit of the others.
__device__ __forceinline__ float scale_of(double sum, float eps) {
  constexpr float kNear = 0x1p-24f;
  return kScale * kNear / ((float)(sqrt(sum) * kNear) + eps * kNear);
}

__device__ __forceinline__ float update_of(bool momentum, float g, float m, const Settings& s) {
  if (!momentum) return g;
  return s.nesterov ? s.mu * m + s.rest * g : m;
}

// The momentum and the sum of squares of kPerGroup values, four beside each other a thread; all are requested before the
// first is used.  WHOLE: all are in the matrix, and 16-byte vectors fit the addresses.
template <typename T, bool WHOLE>
__device__ __forceinline__ double squares_of(const T* g, float* m, int64_t left, const Settings& s) {
  constexpr int N = kPerGroup / 1024;
  float from[N][4], held[N][4];
#pragma unroll
  for (int r = 0; r < N; ++r) {
    const int at = r * 1024 + threadIdx.x * 4;
    const int here = (int)(left - at < 4 ? left - at : 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) from[r][e] = held[r][e] = 0.f;
    if (WHOLE || here > 0) {
      get<T, 4, WHOLE>(g + at, from[r], here);
      if (m) get<float, 4, WHOLE>(m + at, held[r], here);
    }
  }
  double sum = 0;
#pragma unroll
  for (int r = 0; r < N; ++r) {
    const int at = r * 1024 + threadIdx.x * 4;
    const int here = (int)(left - at < 4 ? left - at : 4);
    if (m) {
#pragma unroll
      for (int e = 0; e < 4; ++e) held[r][e] = s.mu * held[r][e] + s.rest * from[r][e];
      if (WHOLE || here > 0) put<float, 4, WHOLE>(m + at, held[r], here);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const double u = update_of(m != nullptr, from[r][e], held[r][e], s);
      sum += u * u;
    }
  }
  return sum;
}
template <typename T>
__global__ __launch_bounds__(256) void squares(const Table t, const Settings s, char* workspace, int split) {
  __shared__ double sums[4];
  const Mine mine = matrix_of(t, blockIdx.x);
  const int64_t n = (int64_t)mine.rows * mine.columns, first = mine.id * kPerGroup;
  const T* g = (const T*)mine.g + first;
  float* m = mine.m ? mine.m + first : nullptr;
  const bool whole = first + kPerGroup <= n && (uintptr_t)g % 16 == 0 && (uintptr_t)m % 16 == 0;
  double sum = whole ? squares_of<T, true>(g, m, n - first, s) : squares_of<T, false>(g, m, n - first, s);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    const Layout at(mine.rows, mine.columns, split);
    ((double*)(workspace + mine.at + at.sums))[mine.id] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
}

// The normalised update as X, 64 x 64 values a workgroup.
template <typename T, bool SPLIT>
__global__ __launch_bounds__(256) void lay_out(const Table t, const Settings s, char* workspace) {
  __shared__ float tile[64][65];
  __shared__ double sums[4];
  const unsigned group = gridDim.x - 1 - blockIdx.x;   // last first: what squares() touched last is still in the caches
  const Mine mine = matrix_of(t, group);
  const int rows = mine.rows, columns = mine.columns;
  const Layout at(rows, columns, SPLIT);
  char* place = workspace + mine.at;
  const T* g = (const T*)mine.g;
  const float* m = mine.m;
  // the tile as it lies in the matrix
  const bool tall = rows > columns;
  const int64_t cp = tall ? at.kp : at.lp, id = mine.id;
  const int64_t r0 = id / (cp / 64) * 64, c0 = id % (cp / 64) * 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float from[16], held[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const bool there = r0 + 4 * r + wave < rows && c0 + lane < columns;
    const int64_t i = (r0 + 4 * r + wave) * columns + c0 + lane;
    from[r] = there ? (float)g[i] : 0.f;
    held[r] = there && m ? m[i] : 0.f;
  }
  const double* parts = (const double*)(place + at.sums);
  const int64_t count = ((int64_t)rows * columns + kPerGroup - 1) / kPerGroup;
  double sum = 0;
  for (int64_t j = threadIdx.x; j < count; j += 256) sum += parts[j];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) sums[wave] = sum;
#pragma unroll
  for (int r = 0; r < 16; ++r) tile[4 * r + wave][lane] = update_of(m != nullptr, from[r], held[r], s);
  __syncthreads();
  const float up = scale_of((sums[0] + sums[1]) + (sums[2] + sums[3]), s.eps);
  const int64_t k0 = tall ? c0 : r0, l0 = tall ? r0 : c0;
  for (int c = threadIdx.x; c < 64 * 8; c += 256) {
    const int r = c / 8, from = c % 8 * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (tall ? tile[from + e][r] : tile[r][from + e]) * up;
    write_values<SPLIT, 8>(place + at.x0 + (k0 + r) * at.l_row, l0 + from, v);
  }
}

typedef const __attribute__((address_space(1))) void* Global;
typedef __attribute__((address_space(3))) void* Lds;

// Between the steps of a product: all but the wave's last LEFT requests have landed, its reads are done, and so have every
// other wave's.
template <int LEFT>
__device__ __forceinline__ void step_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((LEFT & 15) | 7 << 4 | (LEFT >> 4) << 14);   // vmcnt(LEFT) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The lanes' columns of 16 KK rows of ROW bytes: KK operands, from the lane's place in the first four rows.  Waits for them
// itself.
template <int KK, int ROW>
__device__ __forceinline__ void turned_reads(const char* first, f16x8 (&operands)[KK]) {
  typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
  const unsigned at = (unsigned)(uintptr_t)(Lds)(first);
  u32x2_t lo[KK], hi[KK];
  if constexpr (KK == 2) {
    asm volatile("ds_read_b64_tr_b16 %0, %4\n\t"
                 "ds_read_b64_tr_b16 %1, %4 offset:%5\n\t"
                 "ds_read_b64_tr_b16 %2, %4 offset:%6\n\t"
                 "ds_read_b64_tr_b16 %3, %4 offset:%7\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1])
                 : "v"(at), "i"(4 * ROW), "i"(16 * ROW), "i"(20 * ROW)
                 : "memory");
  } else {
    static_assert(KK == 4, "lines of 32 or 64 values");
    asm volatile("ds_read_b64_tr_b16 %0, %8\n\t"
                 "ds_read_b64_tr_b16 %1, %8 offset:%9\n\t"
                 "ds_read_b64_tr_b16 %2, %8 offset:%10\n\t"
                 "ds_read_b64_tr_b16 %3, %8 offset:%11\n\t"
                 "ds_read_b64_tr_b16 %4, %8 offset:%12\n\t"
                 "ds_read_b64_tr_b16 %5, %8 offset:%13\n\t"
                 "ds_read_b64_tr_b16 %6, %8 offset:%14\n\t"
                 "ds_read_b64_tr_b16 %7, %8 offset:%15\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(lo[0]), "=&v"(hi[0]), "=&v"(lo[1]), "=&v"(hi[1]), "=&v"(lo[2]), "=&v"(hi[2]), "=&v"(lo[3]),
                   "=&v"(hi[3])
                 : "v"(at), "i"(4 * ROW), "i"(16 * ROW), "i"(20 * ROW), "i"(32 * ROW), "i"(36 * ROW), "i"(48 * ROW),
                   "i"(52 * ROW)
                 : "memory");
  }
#pragma unroll
  for (int k = 0; k < KK; ++k) {
    typedef unsigned u32x4_t __attribute__((ext_vector_type(4)));
    operands[k] = __builtin_bit_cast(f16x8, u32x4_t{lo[k].x, lo[k].y, hi[k].x, hi[k].y});
  }
}

constexpr int kGram = 0, kPolynomial = 1, kNext = 2, kLast = 3;

// A workgroup's block of F rows of the first operand and G of the second, dealt to waves of at most 64 x 64.
// LINES: of 128 bytes of each row that a step takes, by as many groups of waves, each with a sum of its own.
template <int F_, int G_, int ACROSS_, int LINES_, int STAGES_>
struct Shape {
  static constexpr int F = F_, G = G_, DOWN = F_ < 64 ? 1 : 2, ACROSS = ACROSS_, LINES = LINES_;
  static constexpr int WAVES = DOWN * ACROSS, THREADS = 64 * WAVES * LINES;
  static constexpr int Y = F / 32 / DOWN, X = G / 32 / ACROSS;   // 32 x 32 blocks of a wave
  static constexpr int STAGES = STAGES_;                         // steps in LDS
  static constexpr int F_LOADS = F * 8 / (64 * WAVES), LOADS = (F + G) * 8 / (64 * WAVES);   // 16-byte requests of a thread
                                                                                              // and step
  static constexpr int LINE_BYTES = (F + G) * 128, STEP = LINES * LINE_BYTES;                // in LDS
};

// A wave's 32 x 32 block on its way to memory: in LDS as rows of 128 bytes whose 16-byte chunks are exchanged by the row's
// number, so that neither the lanes' columns nor the rows meet in one bank.
__device__ __forceinline__ int chunk_at(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) * 16); }

// From the lanes (column lane % 32, rows 8 q + 4 (lane / 32) + e of value 4 q + e) to lines of memory: its rows to `rows`, its
// columns to `columns` (NULL: not written); without ROWS_TOO to `columns` alone.
template <bool SPLIT, bool ROWS_TOO>
__device__ __forceinline__ void write_block(const floatx16& v, char* scratch, int lane, char* rows, int64_t rows_bytes,
                                            char* columns, int64_t columns_bytes) {
  constexpr int PIECES = SPLIT ? 2 : 1;
  const int half = lane / 32, c = lane % 32;
  f16 piece[2][16];
#pragma unroll
  for (int e = 0; e < 16; ++e) split_f16(v[e], piece[0][e], piece[1][e]);
#pragma unroll
  for (int p = 0; p < PIECES; ++p)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (ROWS_TOO) *(f16*)(scratch + chunk_at(8 * q + 4 * half + e, p * 4 + c / 8) + c % 8 * 2) = piece[p][4 * q + e];
      if (!ROWS_TOO || columns) {
        Pack<f16, 4> four;
#pragma unroll
        for (int e = 0; e < 4; ++e) four.v[e] = piece[p][4 * q + e];
        *reinterpret_cast<Pack<f16, 4>*>(scratch + 4096 + chunk_at(c, p * 4 + q) + half * 8) = four;
      }
    }
  wave_order();
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  constexpr int CHUNKS = 4 * PIECES, ROWS = 64 / CHUNKS;   // chunks of a row; rows of a store
#pragma unroll
  for (int r = 0; r < 32; r += ROWS) {
    const int row = r + lane / CHUNKS, chunk = lane % CHUNKS;
    if (ROWS_TOO) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(scratch + chunk_at(row, chunk));
      *reinterpret_cast<u32x4*>(rows + row * rows_bytes + chunk * 16) = x;
    }
    if (!ROWS_TOO || columns) {
      const u32x4 y = *reinterpret_cast<const u32x4*>(scratch + 4096 + chunk_at(row, chunk));
      *reinterpret_cast<u32x4*>(columns + row * columns_bytes + chunk * 16) = y;
    }
  }
  wave_order();
}

// What a block on a diagonal keeps beside its float16 values: of each column the rest of its diagonal's value.
__device__ __forceinline__ void keep_rest(const floatx16& v, int lane, float* to) {
  const int c = lane % 32;
  float own = v[0];
#pragma unroll
  for (int e = 1; e < 16; ++e) own = e == c / 8 * 4 + c % 4 ? v[e] : own;
  if (c / 4 % 2 == lane / 32) to[c] = own - (float)(f16)own;
}

// The diagonal of 32 rests, one of each lane's column, as two operands of 16.
struct Rests {
  f16x8 v[2];
  __device__ __forceinline__ Rests() = default;
  __device__ __forceinline__ Rests(float rest, int lane) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[kk][e] = kk * 16 + lane / 32 * 8 + e == lane % 32 ? (f16)rest : (f16)0.f;
  }
};

// Where the last product goes: element (row, column) at p[row * columns + column], alone or as a parameter's step.
template <typename T>
struct Result {
  T* p;
  int64_t rows, columns;
  bool turned;               // the block's columns are the matrix's rows
  bool step, wide;           // wide: rows of whole 16-byte vectors
  float keep, rate;

  static constexpr int V = kWide<T>, PARTS = 32 / V, ROWS = 64 / PARTS, N = 32 / ROWS;   // vectors of a block's row, rows of
                                                                                         // a wave's request, requests
  typedef Pack<T, V> Old[N];

  __device__ __forceinline__ bool there(int64_t row0, int64_t column0, int lane, int n, int64_t& at) const {
    const int64_t row = row0 + n * ROWS + lane / PARTS, column = column0 + lane % PARTS * V;
    at = row * columns + column;
    return row < rows && column < columns;
  }
  // The parameters of a block, requested before the block is worked on.
  __device__ __forceinline__ void load(Old& old, int lane, int64_t row0, int64_t column0) const {
    if (!wide || !step) return;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      int64_t at;
      if (there(row0, column0, lane, n, at)) old[n] = *reinterpret_cast<const Pack<T, V>*>(p + at);
    }
  }
  __device__ __forceinline__ T value(T old, float x) const { return (T)(step ? (float)old * keep - rate * x : x); }

  // The block through LDS: memory's rows in rows there.
  __device__ __forceinline__ void store(const floatx16& v, const Old& old, char* scratch, int lane, int64_t row0,
                                        int64_t column0) const {
    const int half = lane / 32, c = lane % 32;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (turned) {
        const float4 four = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        *reinterpret_cast<float4*>(scratch + chunk_at(c, 2 * q + half)) = four;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) *(float*)(scratch + chunk_at(8 * q + 4 * half + e, c / 4) + c % 4 * 4) = v[4 * q + e];
      }
    }
    wave_order();
    if (wide) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        int64_t at;
        const bool inside = there(row0, column0, lane, n, at);
        const int row = n * ROWS + lane / PARTS, chunk = lane % PARTS * V / 4;
        Pack<T, V> out;
#pragma unroll
        for (int e = 0; e < V; e += 4) {
          const float4 x = *reinterpret_cast<const float4*>(scratch + chunk_at(row, chunk + e / 4));
          out.v[e] = value(old[n].v[e], x.x), out.v[e + 1] = value(old[n].v[e + 1], x.y);
          out.v[e + 2] = value(old[n].v[e + 2], x.z), out.v[e + 3] = value(old[n].v[e + 3], x.w);
        }
        if (inside) *reinterpret_cast<Pack<T, V>*>(p + at) = out;
      }
    } else {
      T one[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t row = row0 + 2 * e + half;
        if (step && row < rows && column0 + c < columns) one[e] = p[row * columns + column0 + c];
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t row = row0 + 2 * e + half;
        const float x = *(const float*)(scratch + chunk_at(2 * e + half, c / 4) + c % 4 * 4);
        if (row < rows && column0 + c < columns) p[row * columns + column0 + c] = value(one[e], x);
      }
    }
    wave_order();
  }
};

// One product of F x G values a workgroup, of which a step has 128 bytes of each of the F + G rows in LDS, brought there
// without registers on the way while the steps before are multiplied.
//   S, P: rows i of X (of S) with rows j of it, tiles i <= j, written both ways.
//   X':   columns j of X with rows i of P: the block's rows are X's columns, so that a lane has four of a row of X' beside
//         each other.  X lies with its columns beside each other: those operands are transposed on the way out of LDS.
// The 16-byte chunks of a row are exchanged by its number, so that the lanes of a read meet no bank twice: of rows of 128
// bytes by row % 8, of the steps of X by 4 (row % 4) (rows of 128 bytes: by half of that).
template <bool SPLIT, typename S, int STAGE, typename T>
__global__ __launch_bounds__(S::THREADS, 2) void product(const Table t, const Settings s, char* workspace, int turn) {
  constexpr bool SQUARE = STAGE <= kPolynomial;
  static_assert(!SQUARE || S::F == S::G, "tiles on the diagonal");
  constexpr int CHUNKS = S::F * (SPLIT ? 4 : 2) / 16;       // of a row of X's step
  constexpr int LINE = kLine<SPLIT>, KK = LINE / 16, PIECES = SPLIT ? 2 : 1;
  __shared__ __attribute__((aligned(128))) char lds[S::STAGES * S::STEP];
  const unsigned group = by_die(blockIdx.x, gridDim.x);
  const Mine mine = matrix_of(t, group);
  const Layout at(mine.rows, mine.columns, SPLIT);
  char* place = workspace + mine.at;
  const int64_t id = mine.id;
  int64_t ti, tj;                             // tile of the block's rows, of its columns
  if constexpr (SQUARE) {                     // ti <= tj, counted column by column
    tj = (int64_t)((sqrtf(8.f * (float)id + 1.f) - 1.f) * 0.5f);
    while (tj * (tj + 1) / 2 > id) --tj;
    while ((tj + 1) * (tj + 2) / 2 <= id) ++tj;
    ti = id - tj * (tj + 1) / 2;
  } else {
    const int64_t across = (at.kp + S::G - 1) / S::G;
    tj = id % across, ti = id / across;
  }
  const char* X = place + (turn ? at.x1 : at.x0);
  const char* rows_of = STAGE == kGram ? X : place + (STAGE == kPolynomial ? at.s : at.p);   // of 128 bytes a step
  const int64_t row_bytes = STAGE == kGram ? at.l_row : at.k_row;
  const int lines = (int)(row_bytes / 128), steps = (lines + S::LINES - 1) / S::LINES;

  // a group of waves takes every LINES-th line of the rows
  const int any_wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, wave = any_wave % S::WAVES, line = any_wave / S::WAVES;
  const int thread = threadIdx.x % (64 * S::WAVES);
  const char* from[S::LOADS];
#pragma unroll
  for (int r = 0; r < S::LOADS; ++r) {
    const bool first = r < S::F_LOADS;
    const int chunk = (first ? r : r - S::F_LOADS) * 64 * S::WAVES + thread;   // of its operand's part of the line
    if (SQUARE || !first) {
      const int row = chunk / 8;
      int64_t global = first ? ti * S::F + row : tj * S::G + row;
      global = global < at.kp ? global : at.kp - 1;   // tiles that pass the end: the last row again, not written
      from[r] = rows_of + global * row_bytes + ((chunk % 8) ^ (row & 7)) * 16;
    } else {
      const int row = chunk / CHUNKS, turned = CHUNKS >= 16 ? row % 4 * 4 : row / 2 % 2 * 4;
      int64_t byte = ti * (CHUNKS * 16) + ((chunk % CHUNKS) ^ turned) * 16;
      byte = byte < at.l_row ? byte : at.l_row - 16;
      from[r] = X + row * at.l_row + byte;
    }
  }
  const int64_t first_line = SQUARE ? 128 : LINE * at.l_row;
  auto request = [&](int step) {   // of lines behind the rows' end: the last one, not used
    char* to = lds + step % S::STAGES * S::STEP + line * S::LINE_BYTES + wave * 1024;
    int64_t here = step * S::LINES + line;
    if constexpr (S::LINES > 1) here = here < lines ? here : lines - 1;
#pragma unroll
    for (int r = 0; r < S::LOADS; ++r)
      __builtin_amdgcn_global_load_lds((Global)(from[r] + here * (r < S::F_LOADS ? first_line : 128)),
                                       (Lds)(to + r * S::WAVES * 1024), 16, 0, 0);
  };

  floatx16 acc[S::Y][S::X];
#pragma unroll
  for (int y = 0; y < S::Y; ++y)
#pragma unroll
    for (int x = 0; x < S::X; ++x)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[y][x][v] = 0.f;

  const int half = lane / 32, wy = wave / S::ACROSS * S::Y * 32, wx = wave % S::ACROSS * S::X * 32;
  // the rests of the diagonals of S and, as operands that are zero beside it, of the blocks' rows of P
  constexpr bool DIAGONAL = !SPLIT && !SQUARE;
  float *s_rest = (float*)(place + at.s_rest), *p_rest = (float*)(place + at.p_rest);
  Rests rest[DIAGONAL ? S::X : 1];
  if constexpr (DIAGONAL) {
#pragma unroll
    for (int x = 0; x < S::X; ++x) {
      const int64_t j = tj * S::G + wx + x * 32 + lane % 32;
      rest[x] = Rests(j < at.kp ? p_rest[j] : 0.f, lane);
    }
  }
#pragma unroll
  for (int step = 0; step < S::STAGES - 1; ++step)
    if (step < steps) request(step);
  for (int step = 0; step < steps; ++step) {
    if (step + S::STAGES - 1 <= steps)   // as many steps requested as there is room for
      step_barrier<(S::STAGES - 2) * S::LOADS>();
    else
      step_barrier<0>();
    const bool more = step + S::STAGES - 1 < steps;
    const char* buffer = lds + step % S::STAGES * S::STEP + line * S::LINE_BYTES;
    auto operand = [&](int row, int chunk) { return *reinterpret_cast<const f16x8*>(buffer + chunk_at(row, chunk)); };
    // columns first .. first + 31 of 16 rows of X from row `row` on
    auto turned_at = [&](int first, int row, int piece) {
      const int r = row + 8 * half + lane % 16 / 4;   // and r + 4, whose chunks lie alike
      const int column = first + lane / 16 % 2 * 16;
      const int chunk = column / LINE * 8 + piece * 4 + column % LINE / 8 + lane % 4 / 2;
      return buffer + r * (CHUNKS * 16) + ((chunk ^ (CHUNKS >= 16 ? r % 4 * 4 : r / 2 % 2 * 4)) * 16) + lane % 2 * 8;
    };
    f16x8 a[KK][S::Y][PIECES];
    if constexpr (SQUARE) {
      if (more) request(step + S::STAGES - 1);
    } else if constexpr (S::STAGES == 2) {
      // the compiler waits for every request in flight before a transposing read: these come first
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int y = 0; y < S::Y; ++y)
#pragma unroll
          for (int piece = 0; piece < PIECES; ++piece) {
            const char* lo = turned_at(wy + y * 32, kk * 16, piece);
            a[kk][y][piece] = __builtin_bit_cast(f16x8, tr_frag(lo, lo + 4 * CHUNKS * 16).v);
          }
      asm volatile("" ::: "memory");
      if (more) request(step + S::STAGES - 1);
      asm volatile("" ::: "memory");
    } else {
      if (more) request(step + S::STAGES - 1);
#pragma unroll
      for (int y = 0; y < S::Y; ++y)
#pragma unroll
        for (int piece = 0; piece < PIECES; ++piece) {
          f16x8 all[KK];
          turned_reads<KK, CHUNKS * 16>(turned_at(wy + y * 32, 0, piece), all);
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) a[kk][y][piece] = all[kk];
        }
    }
    if (S::LINES > 1 && step * S::LINES + line >= lines) continue;
    f16x8 b[KK][S::X][PIECES];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int piece = 0; piece < PIECES; ++piece) {
#pragma unroll
        for (int x = 0; x < S::X; ++x) b[kk][x][piece] = operand(S::F + wx + x * 32 + lane % 32, piece * 4 + kk * 2 + half);
        if constexpr (SQUARE) {
#pragma unroll
          for (int y = 0; y < S::Y; ++y) a[kk][y][piece] = operand(wy + y * 32 + lane % 32, piece * 4 + kk * 2 + half);
        }
      }
    if constexpr (S::LINES > 1) __builtin_amdgcn_sched_barrier(0);   // few products: all reads before the first
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
#pragma unroll
      for (int y = 0; y < S::Y; ++y)
#pragma unroll
        for (int x = 0; x < S::X; ++x) {
          if constexpr (SPLIT) {
            acc[y][x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[kk][y][1], b[kk][x][0], acc[y][x], 0, 0, 0);
            acc[y][x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[kk][y][0], b[kk][x][1], acc[y][x], 0, 0, 0);
          }
          acc[y][x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[kk][y][0], b[kk][x][0], acc[y][x], 0, 0, 0);
        }
    if constexpr (DIAGONAL) {
#pragma unroll
      for (int x = 0; x < S::X; ++x) {
        const int64_t j0 = tj * S::G + wx + x * 32;
        if (j0 / LINE != step * S::LINES + line) continue;
        auto add = [&](auto first) {   // its 32 of the line's rows of X
#pragma unroll
          for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int y = 0; y < S::Y; ++y)
              acc[y][x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[decltype(first)::value + kk][y][0], rest[x].v[kk], acc[y][x],
                                                                 0, 0, 0);
        };
        if (j0 % LINE == 0)
          add(std::integral_constant<int, 0>());
        else
          add(std::integral_constant<int, 2>());
      }
    }
  }
  step_barrier<0>();   // the buffers are free

  if constexpr (S::LINES > 1) {   // the groups' sums, in their order
    float* sums = (float*)lds;
    if (line > 0) {
#pragma unroll
      for (int y = 0; y < S::Y; ++y)
#pragma unroll
        for (int x = 0; x < S::X; ++x)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            sums[((((line - 1) * S::Y + y) * S::X + x) * 16 + v) * (64 * S::WAVES) + thread] = acc[y][x][v];
    }
    __syncthreads();
    if (line > 0) return;
#pragma unroll
    for (int more = 0; more < S::LINES - 1; ++more)
#pragma unroll
      for (int y = 0; y < S::Y; ++y)
#pragma unroll
        for (int x = 0; x < S::X; ++x)
#pragma unroll
          for (int v = 0; v < 16; ++v)
            acc[y][x][v] += sums[(((more * S::Y + y) * S::X + x) * 16 + v) * (64 * S::WAVES) + thread];
  }
  // behind the sums that were just read
  char* scratch = lds + (S::LINES - 1) * S::F * S::G * 4 + wave * 8192;
  static_assert((S::LINES - 1) * S::F * S::G * 4 + S::WAVES * 8192 <= S::STAGES * S::STEP, "scratch lies in the buffers");
  const int64_t i_end = SQUARE ? at.kp : at.lp;
  auto scaled = [&](int y, int x) {
    floatx16 v;
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = acc[y][x][e] * (STAGE == kLast ? kDown * kDown : kDown);
    return v;
  };
  if constexpr (STAGE == kLast) {
    const bool tall = mine.rows > mine.columns;
    T* p = (T*)mine.p;
    const int64_t columns = tall ? at.k : at.l;
    const Result<T> result = {p, tall ? at.l : at.k, columns, !tall, mine.m != nullptr,
                              columns % kWide<T> == 0 && (uintptr_t)p % 16 == 0, s.keep, mine.rate};
#pragma unroll
    for (int y = 0; y < S::Y; ++y) {
      typename Result<T>::Old old[S::X];
      const int64_t i0 = ti * S::F + wy + y * 32;
#pragma unroll
      for (int x = 0; x < S::X; ++x) {
        const int64_t j0 = tj * S::G + wx + x * 32;
        result.load(old[x], lane, tall ? i0 : j0, tall ? j0 : i0);
      }
#pragma unroll
      for (int x = 0; x < S::X; ++x) {
        const int64_t j0 = tj * S::G + wx + x * 32;
        if (i0 < i_end && j0 < at.kp)
          result.store(scaled(y, x), old[x], scratch, lane, tall ? i0 : j0, tall ? j0 : i0);
      }
    }
    return;
  }
#pragma unroll
  for (int y = 0; y < S::Y; ++y)
#pragma unroll
    for (int x = 0; x < S::X; ++x) {
      const int64_t i0 = ti * S::F + wy + y * 32, j0 = tj * S::G + wx + x * 32;
      if (i0 >= i_end || j0 >= at.kp) continue;
      floatx16 v = scaled(y, x);
      if (!SPLIT && STAGE == kGram && i0 == j0) keep_rest(v, lane, s_rest + i0);
      if constexpr (STAGE == kPolynomial) {   // a I + b S + c S S; S is its own transpose
        const int64_t j = j0 + lane % 32;
        const float own_rest = SPLIT ? 0.f : s_rest[j];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t row = i0 + 8 * q + 4 * half;
          float old[4];
          read_values<SPLIT, 4>(place + at.s + j * at.k_row, row, old);
          if constexpr (!SPLIT) {
            const float4 rests = *reinterpret_cast<const float4*>(s_rest + row);
            const float d[4] = {rests.x, rests.y, rests.z, rests.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              v[4 * q + e] = fmaf((d[e] + own_rest) * kDown, old[e], v[4 * q + e]);
              old[e] += row + e == j ? own_rest : 0.f;
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[4 * q + e] = fmaf(s.c, v[4 * q + e], s.b * old[e]) + (row + e == j ? s.a * kScale : 0.f);
        }
        if (!SPLIT && i0 == j0) keep_rest(v, lane, p_rest + i0);
      }
      if constexpr (SQUARE) {
        char* to = place + (STAGE == kGram ? at.s : at.p);
        write_block<SPLIT, true>(v, scratch, lane, place_of<SPLIT>(to + i0 * at.k_row, j0), at.k_row,
                           ti == tj ? nullptr : place_of<SPLIT>(to + j0 * at.k_row, i0), at.k_row);
      } else {
        char* to = place + (turn ? at.x0 : at.x1);
        write_block<SPLIT, false>(v, scratch, lane, nullptr, 0, place_of<SPLIT>(to + j0 * at.l_row, i0), at.l_row);
      }
    }
}

// Matrices of up to 16 rows (or columns): the steps on S alone, in 64 bits, where squares of small singular values keep 1e-16
// of the largest.  All matrices of a step are polynomials of S, so they commute and are symmetric, and with Q the product
// of all P so far
//   Q = P Q    S = P S P = P P S        X_steps = Q X_0
// reads the matrix twice however many steps there are: one workgroup, in float64 products of 16 x 16 x 4.  A lane's four
// values of a product are rows 4 i + lane / 16 of column lane % 16, which is how it takes the second operand, and of a
// symmetric matrix the first: products follow each other in registers, in every wave by itself.
//
// X is not read again, so nothing takes back what rounding does to S.  A step makes of an eigenvalue s the value f(s) = s q(s)^2,
// and of an error E of S, in S's eigenvectors, the differences of f: E_ij (f(s_i) - f(s_j)) / (s_i - s_j), at most max |f'|
// times E.  (For that S has to be symmetric, and is made so in each step: a product taken by its transpose moves the rest of an
// S that is not by more, 16 x 27 2e-6 off after 12 steps of the default coefficients for 3e-15.)  Where f' is not small the
// error grows, and once an eigenvalue of zero is rounded to less, it leaves for minus infinity: equal rows are 3e-13 off after
// 5 steps, 4e-11 after 8, and infinite after 20.  So this is the way of as many steps as keep the product of
// max |f'| below 2^24 (check_coefficients), which leaves 16 roundings of 2^-53 below 2^-25 of S: six steps of the default
// coefficients, thirteen of 1.875, -1.25, 0.375.  More go by X, whose S is a sum of squares anew in each step.
typedef double f64x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f64x4 product_of(const f64x4& a, const f64x4& b) {
  f64x4 sum = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_mfma_f64_16x16x4f64(a[i], b[i], sum, 0, 0, 0);
  return sum;
}

// Five steps against those of X in LDS or through the launches, float32, 16 rows of 17 values 11 us for 18, of 400 16 for 78,
// of 1000 24 for 86, of 4096 70 for 134, of 16384 257 for 340, of 131072 1.76 ms for 2.27; 64 of 16 x 16384 at once 268 us for
// 1160; 3 rows of 1000 18 for 86, of 131072 1.21 ms for 2.28; 2.5e-8 off for 1e-6.  In one piece the launches read half as
// much: bfloat16, 16 rows of 1000 25 us for 76, of 4096 79 for 101, but of 8192 140 for 131.
constexpr int kThin = 16, kThinWaves = 8;
constexpr double kMostGrowth = 1 << 24;
__host__ __device__ inline bool is_thin(int64_t rows, int64_t columns, bool split) {
  const int64_t k = rows < columns ? rows : columns, l = rows < columns ? columns : rows;
  return k <= kThin && (split || l <= 4096);
}

template <typename T>
__device__ void thin_matrix(const T* g, float* m, T* p, int rows, int columns, float rate, const Settings& s, int steps,
                            double (*parts)[4][64]) {
  constexpr int TILES = 4, STRIDE = 16 * kThinWaves;   // tiles of 16 columns of a wave that are requested at once; to its next
  const bool tall = rows > columns;
  const int k = tall ? columns : rows, l = tall ? rows : columns;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, across = lane % 16, down = lane / 16;
  auto place = [&](int row, int column) { return tall ? column * k + row : row * l + column; };

  // the momentum, and S: a lane has row `across` of four columns
  f64x4 S = {0, 0, 0, 0};
  for (int base = wave * 16; base < l; base += TILES * STRIDE) {
    float u[TILES][4], held[TILES][4];
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int column = base + n * STRIDE + 4 * e + down;
        const bool there = across < k && column < l;
        u[n][e] = there ? (float)g[place(across, column)] : 0.f;
        held[n][e] = there && m ? m[place(across, column)] : 0.f;
      }
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int column = base + n * STRIDE + 4 * e + down;
        if (m) {
          held[n][e] = s.mu * held[n][e] + s.rest * u[n][e];
          if (across < k && column < l) m[place(across, column)] = held[n][e];
        }
        const double x = update_of(m != nullptr, u[n][e], held[n][e], s);
        S = __builtin_amdgcn_mfma_f64_16x16x4f64(x, x, S, 0, 0, 0);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) parts[wave][i][lane] = S[i];
  __syncthreads();
  double norm = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    S[i] = parts[0][i][lane];
#pragma unroll
    for (int w = 1; w < kThinWaves; ++w) S[i] += parts[w][i][lane];
    if (4 * i + down == across) norm += S[i];
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) norm += __shfl_xor(norm, d);
  const double scale = 1. / (sqrt(norm) + (double)s.eps);
  f64x4 Q, P, unit;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unit[i] = 4 * i + down == across ? 1. : 0.;
    S[i] *= scale * scale, Q[i] = unit[i] * scale;
  }
  for (int step = 0; step < steps; ++step) {
    const f64x4 turned = product_of(S, unit);   // S's transpose, exactly
#pragma unroll
    for (int i = 0; i < 4; ++i) S[i] = 0.5 * (S[i] + turned[i]);
    const f64x4 square = product_of(S, S);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      P[i] = unit[i] * s.a64 + s.b64 * S[i] + s.c64 * square[i];
    Q = product_of(P, Q);
    if (step + 1 < steps) S = product_of(P, product_of(P, S));
  }

  // Q X_0: a lane has four rows of column `across`
  for (int base = wave * 16; base < l; base += TILES * STRIDE) {
    float u[TILES][4], held[TILES][4], old[TILES][4];
#pragma unroll
    for (int n = 0; n < TILES; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 4 * i + down, column = base + n * STRIDE + across;
        const bool there = row < k && column < l;
        u[n][i] = there ? (float)g[place(row, column)] : 0.f;
        held[n][i] = there && m ? m[place(row, column)] : 0.f;
        old[n][i] = there && m ? (float)p[place(row, column)] : 0.f;
      }
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
      f64x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = update_of(m != nullptr, u[n][i], held[n][i], s);
      x = product_of(Q, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 4 * i + down, column = base + n * STRIDE + across;
        const float out = (float)x[i];
        if (row < k && column < l) p[place(row, column)] = (T)(m ? old[n][i] * s.keep - rate * out : out);
      }
    }
  }
}

// Small matrices, k up to 64: one workgroup takes a matrix through all steps, in LDS throughout.  X, S and P lie there as
// lines of 128 bytes, a row after the other, their chunks exchanged by the row's number.  Thin ones of few steps are steps
// of S alone.
template <bool SPLIT>
struct Small {
  static constexpr int THREADS = 512, LP = SPLIT ? 384 : 640;   // and l up to LP
  static constexpr int SQUARE = 64 * (64 / kLine<SPLIT>) * 128, X = SQUARE / 64 * LP;
  static constexpr int BYTES = X + SQUARE + 16384;              // X, S, P; from P's place on sums of S in float32
};

// 16 bytes of a row's line.
__device__ __forceinline__ char* line_at(char* base, int row, int pitch, int line, int chunk) {
  return base + row * pitch + line * 128 + ((chunk ^ (row & 7)) * 16);
}

// A block's columns into lines: value 4 q + e of a lane is row 8 q + 4 (lane / 32) + e, column lane % 32; its column goes to
// row `row0` + column of `base`, from value `at` of the row on (a multiple of 32).
template <bool SPLIT>
__device__ __forceinline__ void keep_block(const floatx16& v, int lane, char* base, int pitch, int row0, int at) {
  const int half = lane / 32, row = row0 + lane % 32, line = at / kLine<SPLIT>, first = at % kLine<SPLIT> / 8;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    Pack<f16, 4> hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) split_f16(v[4 * q + e], hi.v[e], lo.v[e]);
    *reinterpret_cast<Pack<f16, 4>*>(line_at(base, row, pitch, line, first + q) + half * 8) = hi;
    if constexpr (SPLIT) *reinterpret_cast<Pack<f16, 4>*>(line_at(base, row, pitch, line, 4 + q) + half * 8) = lo;
  }
}

// acc += the products of two operands' pieces
template <bool SPLIT>
__device__ __forceinline__ void add_product(floatx16& acc, const f16x8 (&a)[2], const f16x8 (&b)[2]) {
  if constexpr (SPLIT) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[1], b[0], acc, 0, 0, 0);
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[1], acc, 0, 0, 0);
  }
  acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[0], b[0], acc, 0, 0, 0);
}

template <typename T>
__global__ __launch_bounds__(512) void small_matrix(const Table t, const Settings s, int steps) {
  constexpr bool SPLIT = !std::is_same<T, bf16>::value;
  constexpr int LINE = kLine<SPLIT>, KK = LINE / 16, PIECES = SPLIT ? 2 : 1, SQUARE_PITCH = 64 / LINE * 128;
  using Z = Small<SPLIT>;
  __shared__ __attribute__((aligned(128))) char lds[Z::BYTES];
  __shared__ double sums[8];
  __shared__ __attribute__((aligned(16))) float s_rest[SPLIT ? 4 : 64], p_rest[SPLIT ? 4 : 64];   // of the diagonals
  const int i = blockIdx.x, rows = t.rows[i], columns = t.columns[i];
  if (s.thin && is_thin(rows, columns, SPLIT)) {
    static_assert(Z::THREADS == 64 * kThinWaves && Z::BYTES >= kThinWaves * 4 * 64 * 8, "threads and LDS of both");
    thin_matrix((const T*)t.g[i], t.m[i], (T*)t.p[i], rows, columns, t.rate[i], s, steps, (double (*)[4][64])lds);
    return;
  }
  const bool tall = rows > columns;
  const int k = tall ? columns : rows, l = tall ? rows : columns, lp = (l + 63) / 64 * 64, pitch = lp / LINE * 128;
  const T* g = (const T*)t.g[i];
  float* m = t.m[i];
  char *X = lds, *S = lds + Z::X, *P = S + Z::SQUARE;
  float* blocks = (float*)P;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane / 32;

  // momentum and norm; the update stays in registers, X begins as zeros
  // four columns of a row at once, a thread's vectors THREADS apart
  constexpr int EACH = Z::LP * 64 / 4 / Z::THREADS;
  const int vectors = (columns + 3) / 4, rows_on = Z::THREADS / vectors, vectors_on = Z::THREADS % vectors;
  const int row0 = (int)threadIdx.x / vectors, vector0 = (int)threadIdx.x % vectors;
  auto next_vector = [&](int& row, int& vector) {
    row += rows_on, vector += vectors_on;
    if (vector >= vectors) vector -= vectors, ++row;
  };
  float u[EACH][4], old[EACH][4];
  int row = row0, vector = vector0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
#pragma unroll
    for (int c = 0; c < 4; ++c) u[e][c] = old[e][c] = 0.f;
    if (row < rows) {
      load_part<T, 4>(g + row * columns + vector * 4, u[e], columns - vector * 4);
      if (m) load_part<float, 4>(m + row * columns + vector * 4, old[e], columns - vector * 4);
    }
    next_vector(row, vector);
  }
  double sum = 0;
  row = row0, vector = vector0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (m && row < rows) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float grad = u[e][c];
        old[e][c] = s.mu * old[e][c] + s.rest * grad;
        u[e][c] = s.nesterov ? s.mu * old[e][c] + s.rest * grad : old[e][c];
      }
      store_part<float, 4>(m + row * columns + vector * 4, old[e], columns - vector * 4);
    }
    // four squares in double: float32's range would not do
    sum += ((double)u[e][0] * u[e][0] + (double)u[e][1] * u[e][1]) + ((double)u[e][2] * u[e][2] + (double)u[e][3] * u[e][3]);
    next_vector(row, vector);
  }
  for (int at = threadIdx.x * 16; at < 64 * pitch; at += Z::THREADS * 16) *(float4*)(X + at) = float4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) sum += sums[w];
  const float up = scale_of(sum, s.eps);
  row = row0, vector = vector0;
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    if (row < rows) {
      Pack<f16, 4> hi, lo;
#pragma unroll
      for (int c = 0; c < 4; ++c) split_f16(u[e][c] * up, hi.v[c], lo.v[c]);
      if (tall) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {   // up to three rows behind the matrix's: zeros
          const int y = vector * 4 + c;
          *(f16*)(line_at(X, y, pitch, row / LINE, row % LINE / 8) + row % 8 * 2) = hi.v[c];
          if constexpr (SPLIT) *(f16*)(line_at(X, y, pitch, row / LINE, 4 + row % LINE / 8) + row % 8 * 2) = lo.v[c];
        }
      } else {
        const int x = vector * 4;
        *reinterpret_cast<Pack<f16, 4>*>(line_at(X, row, pitch, x / LINE, x % LINE / 8) + x % 8 * 2) = hi;
        if constexpr (SPLIT)
          *reinterpret_cast<Pack<f16, 4>*>(line_at(X, row, pitch, x / LINE, 4 + x % LINE / 8) + x % 8 * 2) = lo;
      }
    }
    next_vector(row, vector);
  }
  __syncthreads();

  auto operand = [&](char* base, int row_pitch, int row, int line, int kk, f16x8 (&x)[2]) {
#pragma unroll
    for (int piece = 0; piece < PIECES; ++piece)
      x[piece] = *reinterpret_cast<const f16x8*>(line_at(base, row + lane % 32, row_pitch, line, piece * 4 + kk * 2 + half));
  };
  Rests rest[2];   // of P's diagonal
  // columns j .. j + 31 of P X times `down`, as rows: the rows of P in two halves
  auto multiply = [&](int j, floatx16 (&next)[2], float down) {
#pragma unroll
    for (int v = 0; v < 16; ++v) next[0][v] = next[1][v] = 0.f;
    f16x8 x[4][2];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int piece = 0; piece < PIECES; ++piece) {
        const int row = kk * 16 + 8 * half + lane % 16 / 4, column = j + lane / 16 % 2 * 16;
        const int chunk = piece * 4 + column % LINE / 8 + lane % 4 / 2;
        const char* lo = line_at(X, row, pitch, column / LINE, chunk) + lane % 2 * 8;
        const char* hi = line_at(X, row + 4, pitch, column / LINE, chunk) + lane % 2 * 8;
        x[kk][piece] = __builtin_bit_cast(f16x8, tr_frag(lo, hi).v);
      }
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        f16x8 p[2];
        operand(P, SQUARE_PITCH, y * 32, kk / KK, kk % KK, p);
        add_product<SPLIT>(next[y], x[kk], p);
      }
    if constexpr (!SPLIT) {   // the rests of P's diagonal
#pragma unroll
      for (int y = 0; y < 2; ++y)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
          next[y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x[2 * y + kk][0], rest[y].v[kk], next[y], 0, 0, 0);
    }
#pragma unroll
    for (int v = 0; v < 16; ++v) next[0][v] *= down, next[1][v] *= down;
  };
  const int by = wave / 2 % 2 * 32, bx = wave % 2 * 32;   // of S and P, by waves 0 to 3
  for (int step = 0; step < steps; ++step) {
    floatx16 acc;
#pragma unroll
    for (int v = 0; v < 16; ++v) acc[v] = 0.f;
    // S: four waves take even lines, four odd ones
    for (int line = wave / 4; line < lp / LINE; line += 2) {
      f16x8 a[KK][2], b[KK][2];
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) operand(X, pitch, by, line, kk, a[kk]), operand(X, pitch, bx, line, kk, b[kk]);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) add_product<SPLIT>(acc, a[kk], b[kk]);
    }
    float* part = blocks + wave % 4 * 1024 + lane;
    if (wave >= 4) {
#pragma unroll
      for (int v = 0; v < 16; ++v) part[v * 64] = acc[v];
    }
    __syncthreads();
    if (wave < 4) {
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[v] = (acc[v] + part[v * 64]) * kDown;
      keep_block<SPLIT>(acc, lane, S, SQUARE_PITCH, bx, by);   // S is its own transpose
      if (!SPLIT && by == bx) keep_rest(acc, lane, s_rest + bx);
    }
    __syncthreads();
    if (wave < 4) {
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[v] = 0.f;
#pragma unroll
      for (int line = 0; line < 64 / LINE; ++line)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          f16x8 a[2], b[2];
          operand(S, SQUARE_PITCH, by, line, kk, a), operand(S, SQUARE_PITCH, bx, line, kk, b);
          add_product<SPLIT>(acc, a, b);
        }
      const int row = bx + lane % 32;   // where this lane's column of S lies
      const float own_rest = SPLIT ? 0.f : s_rest[row];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int line = by / LINE, chunk = by % LINE / 8 + q;
        const Pack<f16, 4> hi = *reinterpret_cast<const Pack<f16, 4>*>(line_at(S, row, SQUARE_PITCH, line, chunk) + half * 8);
        Pack<f16, 4> lo;
        if constexpr (SPLIT)
          lo = *reinterpret_cast<const Pack<f16, 4>*>(line_at(S, row, SQUARE_PITCH, line, 4 + q) + half * 8);
        float4 rests = {0.f, 0.f, 0.f, 0.f};
        if constexpr (!SPLIT) rests = *reinterpret_cast<const float4*>(s_rest + by + 8 * q + 4 * half);
        const float d[4] = {rests.x, rests.y, rests.z, rests.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float old = (float)hi.v[e] + (SPLIT ? (float)lo.v[e] : 0.f);
          if constexpr (!SPLIT) {
            acc[4 * q + e] = fmaf(d[e] + own_rest, old, acc[4 * q + e]);
            old += by + 8 * q + 4 * half + e == row ? own_rest : 0.f;
          }
          acc[4 * q + e] = fmaf(s.c, acc[4 * q + e] * kDown, s.b * old) +
                           (by + 8 * q + 4 * half + e == row ? s.a * kScale : 0.f);
        }
      }
      keep_block<SPLIT>(acc, lane, P, SQUARE_PITCH, bx, by);
      if (!SPLIT && by == bx) keep_rest(acc, lane, p_rest + bx);
    }
    __syncthreads();
    if constexpr (!SPLIT) {
#pragma unroll
      for (int y = 0; y < 2; ++y) rest[y] = Rests(p_rest[y * 32 + lane % 32], lane);
    }
    if (step + 1 == steps) break;
    // X' = P X in place: a wave has 32 columns of X to itself
    for (int j = wave * 32; j < lp; j += Z::THREADS / 2) {
      floatx16 next[2];
      multiply(j, next, kDown);
#pragma unroll
      for (int y = 0; y < 2; ++y) keep_block<SPLIT>(next[y], lane, X, pitch, y * 32, j);
    }
    __syncthreads();
  }
  T* p = (T*)t.p[i];
  const float keep = m ? s.keep : 0.f, rate = m ? -t.rate[i] : 1.f;
  for (int j = wave * 32; j < lp; j += Z::THREADS / 2) {
    floatx16 next[2];
    multiply(j, next, kDown * kDown);
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int row = y * 32 + lane % 32, left = row < k ? l - j - 4 * half : 0;   // columns of this lane's from its first on
      float old[4][4];
      if (left <= 0) continue;
      if (tall) {
        T* to = p + row + (j + 4 * half) * k;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int column = 8 * (v / 4) + v % 4;
          old[v / 4][v % 4] = m && column < left ? (float)to[column * k] : 0.f;
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int column = 8 * (v / 4) + v % 4;
          if (column < left) to[column * k] = (T)(old[v / 4][v % 4] * keep + rate * next[y][v]);
        }
      } else {
        T* to = p + row * l + j + 4 * half;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
          for (int c = 0; c < 4; ++c) old[q][c] = 0.f;
          if (m && 8 * q < left) load_part<T, 4>(to + 8 * q, old[q], left - 8 * q);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
          for (int c = 0; c < 4; ++c) old[q][c] = old[q][c] * keep + rate * next[y][4 * q + c];
          if (8 * q < left) store_part<T, 4>(to + 8 * q, old[q], left - 8 * q);
        }
      }
    }
  }
}

// ------------------------------------------------------------------------------------------ host
struct Matrix {
  void* p;
  const void* g;
  float* m;
  int64_t rows, columns;
  float rate;
};

// float16's 11 bits are more than bfloat16 has, and no more than float16 has.
bool split(int dtype) { return dtype != SDK_BF16; }

// Fills the table's starts with the workgroups that `of` names for each matrix; their sum.
template <typename Of>
int64_t deal(Table& t, int used, Of of) {
  int64_t groups = 0;
  for (int i = 0; i < kMatrices; ++i) {
    t.start[i] = i < used ? (unsigned)groups : 0xffffffffu;
    if (i < used) groups += of(Layout(t.rows[i], t.columns[i], true));
  }
  return groups;
}

int64_t triangle(int64_t n) { return n * (n + 1) / 2; }

template <int STAGE, typename S>
int64_t groups_of(Table& t, int used) {
  return deal(t, used, [](const Layout& at) {
    const int64_t across = ceil_div(at.kp, S::G);
    return STAGE <= kPolynomial ? triangle(across) : across * ceil_div(at.lp, S::F);
  });
}

template <bool SPLIT, typename S, int STAGE, typename T>
void multiply(Table& t, int used, const Settings& s, char* workspace, int turn, hipStream_t stream) {
  const int64_t groups = groups_of<STAGE, S>(t, used);
  launch(product<SPLIT, S, STAGE, T>, dim3((unsigned)groups), dim3(S::THREADS), stream, t, s, workspace, turn);
}

// Tiles of 128 x 128 where they make a workgroup a CU, of 64 x 64 otherwise.  Eight waves a tile keep the matrix unit busier
// than four (S of 32 matrices of up to 640 x 2560 in bfloat16 45 us for 48, X' 67 for 71), but leave too few registers for
// the last stage's parameters (247 us for 190 in float32).  S and P of so few tiles that those of 32 x 32 still make one
// workgroup a CU, take them, eight waves along the sums (five steps of 701 x 1100 in float32 153 us for 184, 400 x 4000 214
// for 289; with two workgroups for some CUs 900 x 1000 226 for 199).
template <bool SPLIT, int STAGE, typename T>
void stage(Table& t, int used, const Settings& s, char* workspace, int turn, hipStream_t stream) {
  using Large = Shape<128, 128, STAGE == kLast ? 2 : 4, 1, 2>;
  using Middle = Shape<64, 64, 2, 2, 4>;
  using Little = std::conditional_t<(STAGE <= kPolynomial), Shape<32, 32, 1, 8, 2>, Middle>;
  if (groups_of<STAGE, Large>(t, used) >= 256)
    multiply<SPLIT, Large, STAGE, T>(t, used, s, workspace, turn, stream);
  else if (STAGE <= kPolynomial && groups_of<STAGE, Little>(t, used) <= 256)
    multiply<SPLIT, Little, STAGE, T>(t, used, s, workspace, turn, stream);
  else
    multiply<SPLIT, Middle, STAGE, T>(t, used, s, workspace, turn, stream);
}

template <typename T>
void run_group(Table& t, int used, const Settings& s, int steps, char* workspace, hipStream_t stream) {
  constexpr bool SPLIT = !std::is_same<T, bf16>::value;
  int64_t groups = deal(t, used, [](const Layout& at) { return ceil_div(at.k * at.l, kPerGroup); });
  launch(squares<T>, dim3((unsigned)groups), dim3(256), stream, t, s, workspace, (int)SPLIT);
  groups = deal(t, used, [](const Layout& at) { return at.kp / 64 * (at.lp / 64); });
  launch(lay_out<T, SPLIT>, dim3((unsigned)groups), dim3(256), stream, t, s, workspace);
  for (int step = 0; step < steps; ++step) {
    const int turn = step & 1;
    stage<SPLIT, kGram, f16>(t, used, s, workspace, turn, stream);
    stage<SPLIT, kPolynomial, f16>(t, used, s, workspace, turn, stream);
    if (step + 1 < steps)
      stage<SPLIT, kNext, f16>(t, used, s, workspace, turn, stream);
    else
      stage<SPLIT, kLast, T>(t, used, s, workspace, turn, stream);
  }
}

// Whether one workgroup takes the matrix.  Three matrices of 16 x 27 to 64 x 288 in float32, a step of each, 43 us for 110
// through the launches.  thin: whether the steps may go by S alone.
bool is_small(int64_t rows, int64_t columns, int dtype, bool thin) {
  const int64_t k = std::min(rows, columns), l = std::max(rows, columns);
  return (thin && is_thin(rows, columns, split(dtype))) ||
         (k <= 64 && l <= (split(dtype) ? Small<true>::LP : Small<false>::LP));
}

// Deals the matrices to groups that share the workspace one after another: 64 at most, and as many workgroups as a
// launch holds.  `run` gets a table and how many it holds; returns the bytes of the largest group.
// small: those that a workgroup takes alone, or the others.
template <typename Get, typename Run>
size_t in_groups(int64_t count, int dtype, bool thin, bool small, Get get, Run run) {
  Table t = {};
  int used = 0;
  int64_t bytes = 0, most = 0, tiles = 0;
  auto done = [&] {
    if (used) run(t, used);
    most = std::max(most, bytes);
    used = 0, bytes = 0, tiles = 0;
  };
  for (int64_t i = 0; i < count; ++i) {
    const Matrix x = get(i);
    if (x.rows < 1 || x.columns < 1 || is_small(x.rows, x.columns, dtype, thin) != small) continue;
    const Layout at(x.rows, x.columns, split(dtype));
    const int64_t mine = std::max(at.kp / 64 * (at.lp / 64), ceil_div(x.rows * x.columns, kPerGroup));
    if (used == kMatrices || tiles + mine > most_groups(256)) done();
    t.p[used] = x.p, t.g[used] = x.g, t.m[used] = x.m, t.rate[used] = x.rate;
    t.rows[used] = (int)x.rows, t.columns[used] = (int)x.columns, t.at[used] = bytes;
    bytes += at.end, tiles += mine;
    ++used;
  }
  done();
  return (size_t)most;
}

// The workspace that is enough for any steps and coefficients.
template <typename Get>
size_t most_bytes(int64_t count, int dtype, Get get) {
  const auto none = [](Table&, int) {};
  return std::max(in_groups(count, dtype, true, false, get, none), in_groups(count, dtype, false, false, get, none));
}

constexpr int64_t kMostSide = 1 << 17;

int check_matrix(int64_t rows, int64_t columns) {
  SDK_REQUIRE(rows >= 0 && columns >= 0 && rows <= kMostSide && columns <= kMostSide &&
                  rows * columns <= (int64_t)1 << 31,
              "a matrix of %lld x %lld: sides up to 131072, 2^31 values", (long long)rows, (long long)columns);
  return SDK_OK;
}

// X begins with a norm of 1 at most, and a step makes of a singular value x the value x q(x^2), q(s) = a + b s + c s^2.
// Followed from 1 on, no value may pass 3.8, so that S stays below 15, and no q of one 15.  Roundings take values further, in
// pieces of 11 bits by up to about three times 2^-12 of them a step, and where the polynomial is steep behind its largest
// value they do not come back: 3 x - x^3 stays within 2 and left float16 after 6 steps.  So 2^-10 goes on top in each step.
// thin: whether errors of S grow little enough for the steps to go by S alone: f(s) = s q(s)^2 has the slope q(s) r(s),
// r(s) = a + 3 b s + 5 c s^2.
int check_coefficients(int64_t steps, const double* k, bool& thin) {
  const double a = k[0], b = k[1], c = k[2];
  auto q = [&](double s) { return std::fabs(a + (b + c * s) * s); };
  auto r = [&](double s) { return std::fabs(a + (3 * b + 5 * c * s) * s); };
  constexpr double kMore = 1 + 0x1p-10;
  double most = kMore, growth = 1;
  for (int64_t step = 0; step < steps; ++step) {
    const double end = most * most;
    double of_q = std::max(q(0), q(end)), next = most * q(end);
    auto inside = [&](double s, bool of_product) {   // where q's or x q(x^2)'s slope is zero
      if (!(s > 0 && s < end)) return;
      if (of_product)
        next = std::max(next, std::sqrt(s) * q(s));
      else
        of_q = std::max(of_q, q(s));
    };
    inside(-b / (2 * c), false);   // c = 0: no number, or none inside
    const double root = 9 * b * b - 20 * a * c;
    if (root >= 0) {   // of r; the second from their product, where -3 b less a root of nearly 3 b would leave nothing
      const double sum = -3 * b - std::copysign(std::sqrt(root), b);
      inside(sum / (10 * c), true), inside(2 * a / sum, true);
    }
    SDK_REQUIRE(of_q <= 15 && next <= 3.8,
                "coefficients %g, %g, %g let singular values or the polynomial grow too far (3.8 and 15) in step %lld", a, b, c,
                (long long)step + 1);
    const double turn = -3 * b / (10 * c);   // c = 0: no number, or none inside
    const double of_r = std::max({r(0), r(end), turn > 0 && turn < end ? r(turn) : 0.});
    growth = std::min(growth * std::max(1., of_q * of_r), 2 * kMostGrowth);
    most = std::max(1e-30, next * kMore);
  }
  thin = growth <= kMostGrowth;
  return SDK_OK;
}

int check_settings(int64_t count, int64_t steps, const double* coefficients, double eps, int dtype, bool& thin) {
  SDK_REQUIRE(known(dtype), "unknown dtype %d (float32, bfloat16 and float16 only)", dtype);
  SDK_REQUIRE(count >= 0, "count must not be negative");
  SDK_REQUIRE(steps >= 1 && steps <= 100, "steps = %lld must be between 1 and 100", (long long)steps);
  SDK_REQUIRE(coefficients, "coefficients must not be NULL");
  for (int i = 0; i < 3; ++i)
    SDK_REQUIRE(std::fabs(coefficients[i]) <= 100, "coefficients must be numbers up to 100 in magnitude");
  SDK_REQUIRE(eps >= 0x1p-100 && eps <= 1, "eps = %g must be between 2^-100 and 1", eps);
  return check_coefficients(steps, coefficients, thin);
}

Settings settings_of(const double* c, double eps, bool thin) {
  Settings s = {};
  s.a = (float)c[0], s.b = (float)c[1], s.c = (float)c[2], s.eps = (float)eps;
  s.a64 = c[0], s.b64 = c[1], s.c64 = c[2], s.thin = thin;
  return s;
}

int run_all(int64_t count, int steps, const Settings& s, void* workspace, size_t workspace_bytes, int dtype,
            sdk_stream_t stream, Matrix (*get)(const void*, int64_t), const void* context) {
  auto of = [&](int64_t i) { return get(context, i); };
  const bool thin = s.thin;
  const size_t need = in_groups(count, dtype, thin, false, of, [](Table&, int) {});
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 128))
    return fail(SDK_ERR_WORKSPACE, "workspace of %zu bytes at a multiple of 128, %zu needed", workspace_bytes, need);
  in_groups(count, dtype, thin, true, of, [&](Table& t, int used) {
    SDK_DISPATCH_TOKEN_DTYPE(dtype, launch(small_matrix<T>, dim3(used), dim3(512), (hipStream_t)stream, t, s, steps));
  });
  in_groups(count, dtype, thin, false, of, [&](Table& t, int used) {
    SDK_DISPATCH_TOKEN_DTYPE(dtype, run_group<T>(t, used, s, steps, (char*)workspace, (hipStream_t)stream));
  });
  return SDK_OK;
}

struct Stack {
  const char* x;
  char* out;
  int64_t rows, columns, bytes;
};
struct Lists {
  void* const* p;
  const void* const* g;
  float* const* m;
  const int64_t *rows, *columns;
  double lr;
};

// A parameter or momentum that is in the lists twice would be changed by two workgroups at once.
int check_once(const Lists& l, int64_t count) {
  std::unique_ptr<const void*[]> written(new (std::nothrow) const void*[2 * count]);
  SDK_REQUIRE(written, "no memory for the addresses of %lld matrices", (long long)count);
  const void** end = written.get();
  for (int64_t i = 0; i < count; ++i)
    if (l.rows[i] && l.columns[i]) *end++ = l.p[i], *end++ = l.m[i];
  std::sort(written.get(), end, std::less<const void*>());
  SDK_REQUIRE(std::adjacent_find(written.get(), end) == end, "a parameter or momentum is in the lists twice");
  for (int64_t i = 0; i < count; ++i)
    SDK_REQUIRE(!l.rows[i] || !l.columns[i] || !std::binary_search(written.get(), end, l.g[i], std::less<const void*>()),
                "gradient %lld is a parameter or a momentum too", (long long)i);
  return SDK_OK;
}

}  // namespace
}  // namespace token
}  // namespace sdk

using namespace sdk;
using namespace sdk::token;

extern "C" {

size_t sdk_orthogonalize_workspace_bytes(int64_t rows, int64_t columns, int64_t count, int32_t dtype) {
  if (check_matrix(rows, columns) != SDK_OK || !known(dtype) || count < 0) return 0;
  count = std::min<int64_t>(count, kMatrices);
  return most_bytes(count, dtype, [&](int64_t) { return Matrix{nullptr, nullptr, nullptr, rows, columns, 0.f}; });
}

int sdk_orthogonalize(const void* x, void* out, int64_t rows, int64_t columns, int64_t count, int32_t steps,
                      const double* coefficients, double eps, void* workspace, size_t workspace_bytes, int32_t dtype,
                      sdk_stream_t stream) {
  bool thin = false;
  if (int rc = check_settings(count, steps, coefficients, eps, dtype, thin)) return rc;
  if (int rc = check_matrix(rows, columns)) return rc;
  if (!count || !rows || !columns) return SDK_OK;
  SDK_REQUIRE(x && out, "x and out must not be NULL");
  const Stack stack = {(const char*)x, (char*)out, rows, columns, rows * columns * (int64_t)bytes_of(dtype)};
  const int rc = run_all(count, steps, settings_of(coefficients, eps, thin), workspace, workspace_bytes, dtype, stream,
                         [](const void* context, int64_t i) {
                           const Stack& s = *(const Stack*)context;
                           return Matrix{s.out + i * s.bytes, s.x + i * s.bytes, nullptr, s.rows, s.columns, 0.f};
                         },
                         &stack);
  if (rc != SDK_OK) return rc;
  SDK_LAUNCH_CHECK("orthogonalize");
  return SDK_OK;
}

size_t sdk_muon_step_workspace_bytes(const int64_t* rows, const int64_t* columns, int64_t count, int32_t dtype) {
  if (!known(dtype) || count < 1 || !rows || !columns) return 0;
  for (int64_t i = 0; i < count; ++i)
    if (check_matrix(rows[i], columns[i]) != SDK_OK) return 0;
  return most_bytes(count, dtype, [&](int64_t i) { return Matrix{nullptr, nullptr, nullptr, rows[i], columns[i], 0.f}; });
}

int sdk_muon_step(void* const* params, const void* const* grads, float* const* momenta, const int64_t* rows,
                  const int64_t* columns, int64_t count, double lr, double momentum, int32_t nesterov,
                  double weight_decay, int32_t steps, const double* coefficients, double eps, void* workspace,
                  size_t workspace_bytes, int32_t dtype, sdk_stream_t stream) {
  bool thin = false;
  if (int rc = check_settings(count, steps, coefficients, eps, dtype, thin)) return rc;
  SDK_REQUIRE(lr >= 0 && weight_decay >= 0 && momentum >= 0 && momentum < 1 && lr <= 1e30 && weight_decay <= 1e30,
              "lr and weight_decay must not be negative, momentum in [0, 1)");
  if (!count) return SDK_OK;
  SDK_REQUIRE(params && grads && momenta && rows && columns, "the lists must not be NULL");
  bool any = false;
  for (int64_t i = 0; i < count; ++i) {
    if (int rc = check_matrix(rows[i], columns[i])) return rc;
    if (!rows[i] || !columns[i]) continue;
    SDK_REQUIRE(params[i] && grads[i] && momenta[i], "matrix %lld: a tensor is NULL", (long long)i);
    any = true;
  }
  if (!any) return SDK_OK;
  Settings s = settings_of(coefficients, eps, thin);
  s.mu = (float)momentum, s.rest = (float)(1 - momentum), s.keep = (float)(1 - lr * weight_decay);
  s.nesterov = nesterov != 0;
  const Lists lists = {params, grads, momenta, rows, columns, lr};
  if (int rc = check_once(lists, count)) return rc;
  const int rc = run_all(count, steps, s, workspace, workspace_bytes, dtype, stream,
                         [](const void* context, int64_t i) {
                           const Lists& l = *(const Lists*)context;
                           const double wide = l.columns[i] ? (double)l.rows[i] / (double)l.columns[i] : 1.0;
                           return Matrix{l.p[i], l.g[i], l.m[i], l.rows[i], l.columns[i],
                                         (float)(l.lr * std::sqrt(std::max(1.0, wide)))};
                         },
                         &lists);
  if (rc != SDK_OK) return rc;
  SDK_LAUNCH_CHECK("muon_step");
  return SDK_OK;
}

}  // extern "C"
