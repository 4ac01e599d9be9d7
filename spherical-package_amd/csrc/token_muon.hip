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
// hi hi + hi lo + lo hi: 22 bits, 2.5e-7 of the result, below what float32 products leave (2e-6), at a third of the
// float16 rate where the float32 unit runs at an eighth.  bfloat16 matrices take one piece: 1.3e-3 of the result, beside
// the 1.7e-3 of its own rounding.  Every singular value stays below about 1.2 on its way with the usual coefficients, so
// entries of X and S are at most 1.5; up to 15 fit.  Sums are float32, of the norm double.
//
// All matrices of a call go through a stage in one launch; their table is a kernel argument.
#include <algorithm>
#include <cmath>
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
};
static_assert(sizeof(Table) + sizeof(Settings) + 64 <= 4096, "kernel arguments are limited to 4 KB");

__device__ __forceinline__ int matrix_of(const unsigned* start, unsigned group) {
  const unsigned long long before = __ballot(start[threadIdx.x & 63] <= group);
  return __builtin_amdgcn_readfirstlane(__popcll(before) - 1);
}

// A row of an operand is a sequence of lines of 128 bytes: 64 values, or 32 values' hi and then their lo pieces.
template <bool SPLIT>
constexpr int kLine = SPLIT ? 32 : 64;

// Where the buffers of a matrix lie; sides padded with zeros to multiples of kPad.
struct Layout {
  int64_t k, l, kp, lp, x, xt[2], s, p, sums, end;   // byte offsets from the matrix's place
  int64_t k_row, l_row;                             // bytes of a row of k and of l values
  __host__ __device__ Layout(int64_t rows, int64_t columns, bool split) {
    k = rows < columns ? rows : columns, l = rows < columns ? columns : rows;
    kp = (k + kPad - 1) / kPad * kPad, lp = (l + kPad - 1) / kPad * kPad;
    k_row = kp * (split ? 4 : 2), l_row = lp * (split ? 4 : 2);
    x = 0, xt[0] = x + kp * l_row, xt[1] = xt[0] + lp * k_row, s = xt[1] + lp * k_row, p = s + kp * k_row;
    sums = p + kp * k_row;
    end = sums + ((rows * columns + kPerGroup - 1) / kPerGroup * 8 + 127) / 128 * 128;
  }
};

template <bool SPLIT>
__device__ __forceinline__ char* place_of(char* row, int64_t at) {
  return row + at / kLine<SPLIT> * 128 + at % kLine<SPLIT> * 2;
}

// N consecutive values (a power of two up to 8, at a multiple of N) into or out of a row.
template <bool SPLIT, int N>
__device__ __forceinline__ void write_values(char* row, int64_t at, const float (&v)[N]) {
  char* to = place_of<SPLIT>(row, at);
  Pack<f16, N> hi, lo;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    hi.v[e] = (f16)v[e];
    lo.v[e] = (f16)(v[e] - (float)hi.v[e]);
  }
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

template <typename T>
__device__ __forceinline__ float update_of(const T* g, const float* m, int64_t i, const Settings& s) {
  if (!m) return (float)g[i];
  return s.nesterov ? s.mu * m[i] + s.rest * (float)g[i] : m[i];
}

// The momentum, and the sum of squares of the update, 4096 values a workgroup.
template <typename T>
__global__ __launch_bounds__(256) void squares(const Table t, const Settings s, char* workspace, int split) {
  __shared__ double sums[4];
  const int i = matrix_of(t.start, blockIdx.x);
  const int64_t n = (int64_t)t.rows[i] * t.columns[i], group = blockIdx.x - t.start[i];
  const T* g = (const T*)t.g[i];
  float* m = t.m[i];
  double sum = 0;
#pragma unroll 4
  for (int r = 0; r < kPerGroup / 256; ++r) {
    const int64_t at = group * kPerGroup + r * 256 + threadIdx.x;
    if (at < n) {
      if (m) m[at] = s.mu * m[at] + s.rest * (float)g[at];
      const double u = update_of(g, m, at, s);
      sum += u * u;
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    const Layout at(t.rows[i], t.columns[i], split);
    ((double*)(workspace + t.at[i] + at.sums))[group] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  }
}

// The normalised update as operands, 64 x 64 values of X and of its transpose a workgroup.
template <typename T, bool SPLIT>
__global__ __launch_bounds__(256) void lay_out(const Table t, const Settings s, char* workspace) {
  __shared__ float tile[64][65];
  __shared__ double sums[4];
  const int i = matrix_of(t.start, blockIdx.x), rows = t.rows[i], columns = t.columns[i];
  const Layout at(rows, columns, SPLIT);
  char* place = workspace + t.at[i];
  const T* g = (const T*)t.g[i];
  const float* m = t.m[i];
  const double* parts = (const double*)(place + at.sums);
  const int64_t count = ((int64_t)rows * columns + kPerGroup - 1) / kPerGroup;
  double sum = 0;
  for (int64_t j = threadIdx.x; j < count; j += 256) sum += parts[j];
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = sum;
  __syncthreads();
  const float up = kScale / ((float)sqrt((sums[0] + sums[1]) + (sums[2] + sums[3])) + s.eps);
  // the tile as it lies in the matrix
  const bool tall = rows > columns;
  const int64_t cp = tall ? at.kp : at.lp, id = blockIdx.x - t.start[i];
  const int64_t r0 = id / (cp / 64) * 64, c0 = id % (cp / 64) * 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll 4
  for (int r = wave; r < 64; r += 4) {
    const bool there = r0 + r < rows && c0 + lane < columns;
    tile[r][lane] = there ? update_of(g, m, (r0 + r) * columns + c0 + lane, s) * up : 0.f;
  }
  __syncthreads();
  char* by_row = place + (tall ? at.xt[0] : at.x);
  char* by_column = place + (tall ? at.x : at.xt[0]);
  const int64_t row_bytes = tall ? at.k_row : at.l_row, column_bytes = tall ? at.l_row : at.k_row;
  for (int c = threadIdx.x; c < 64 * 8; c += 256) {
    const int r = c / 8, from = c % 8 * 8;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[r][from + e];
    write_values<SPLIT, 8>(by_row + (r0 + r) * row_bytes, c0 + from, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = tile[from + e][r];
    write_values<SPLIT, 8>(by_column + (c0 + r) * column_bytes, r0 + from, v);
  }
}

typedef const __attribute__((address_space(1))) void* Global;
typedef __attribute__((address_space(3))) void* Lds;

// Between the steps of a product: every wave's requests have landed and its reads are done.
__device__ __forceinline__ void step_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

constexpr int kGram = 0, kPolynomial = 1, kNext = 2, kLast = 3;

// Waves of a workgroup, down and across, and 32 x 32 blocks of a wave.
template <int TILE>
struct Shape {
  static constexpr int DOWN = 2, ACROSS = TILE == 256 ? 4 : 2, THREADS = 64 * DOWN * ACROSS;
  static constexpr int Y = TILE / 32 / DOWN, X = TILE / 32 / ACROSS;
  static constexpr int LOADS = 2 * TILE * 128 / 16 / THREADS;   // 16-byte requests of a thread and step
};

// A wave's 32 x 32 block on its way to memory: in LDS as rows of 128 bytes whose 16-byte chunks are exchanged by the row's
// number, so that neither the lanes' columns nor the rows meet in one bank.
__device__ __forceinline__ int chunk_at(int row, int chunk) { return row * 128 + ((chunk ^ (row & 7)) * 16); }

// From the lanes (column lane % 32, rows 8 q + 4 (lane / 32) + e of value 4 q + e) to the lines of `rows` and `columns`
// (NULL: not written), rows of the matrix in rows of operands and in columns of them.
template <bool SPLIT>
__device__ __forceinline__ void write_block(const floatx16& v, char* scratch, int lane, char* rows, int64_t rows_bytes,
                                            char* columns, int64_t columns_bytes) {
  constexpr int PIECES = SPLIT ? 2 : 1;
  const int half = lane / 32, c = lane % 32;
  f16 piece[2][16];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    piece[0][e] = (f16)v[e];
    piece[1][e] = (f16)(v[e] - (float)piece[0][e]);
  }
#pragma unroll
  for (int p = 0; p < PIECES; ++p)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *(f16*)(scratch + chunk_at(8 * q + 4 * half + e, p * 4 + c / 8) + c % 8 * 2) = piece[p][4 * q + e];
      if (columns) {
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
    const u32x4 x = *reinterpret_cast<const u32x4*>(scratch + chunk_at(row, chunk));
    *reinterpret_cast<u32x4*>(rows + row * rows_bytes + chunk * 16) = x;
    if (columns) {
      const u32x4 y = *reinterpret_cast<const u32x4*>(scratch + 4096 + chunk_at(row, chunk));
      *reinterpret_cast<u32x4*>(columns + row * columns_bytes + chunk * 16) = y;
    }
  }
  wave_order();
}

// A block of the last product into the matrix: element (row, column) at p[row * stride + column]; `turned`: the block's
// columns are the matrix's rows.
template <typename T>
__device__ __forceinline__ void write_result(const floatx16& v, char* scratch, int lane, T* p, int64_t stride, bool turned,
                                             int64_t row0, int64_t column0, int64_t rows, int64_t columns, bool step,
                                             float keep, float rate) {
  const int half = lane / 32, c = lane % 32;
  float x[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = v[e];
  if (turned) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 four = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
      *reinterpret_cast<float4*>(scratch + chunk_at(c, 2 * q + half)) = four;
    }
    wave_order();
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = *(const float*)(scratch + chunk_at(2 * e + half, c / 4) + c % 4 * 4);
    wave_order();
  }
  T old[16];
  bool there[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int row = turned ? 2 * e + half : 8 * (e / 4) + 4 * half + e % 4;
    there[e] = row0 + row < rows && column0 + c < columns;
    if (step && there[e]) old[e] = p[(row0 + row) * stride + column0 + c];
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int row = turned ? 2 * e + half : 8 * (e / 4) + 4 * half + e % 4;
    if (there[e]) p[(row0 + row) * stride + column0 + c] = (T)(step ? (float)old[e] * keep - rate * x[e] : x[e]);
  }
}

// One product of TILE x TILE values a workgroup, rows i of A with rows j of B, of which step k has 128 bytes each in LDS,
// brought there without registers on the way while the step before is multiplied.  A row's eight 16-byte chunks are
// exchanged by its number, so that the lanes of a read meet no bank twice.
template <bool SPLIT, int TILE, int STAGE, typename T>
__global__ __launch_bounds__(Shape<TILE>::THREADS, TILE == 64 ? 4 : 2) void product(const Table t, const Settings s, char* workspace, int turn) {
  using S = Shape<TILE>;
  __shared__ __attribute__((aligned(128))) char lds[2][2 * TILE * 128];
  const unsigned group = by_die(blockIdx.x, gridDim.x);
  const int i = matrix_of(t.start, group);
  const Layout at(t.rows[i], t.columns[i], SPLIT);
  char* place = workspace + t.at[i];
  const int64_t id = group - t.start[i];
  int64_t ti, tj;
  if constexpr (STAGE <= kPolynomial) {      // tiles ti <= tj, counted column by column
    tj = (int64_t)((sqrtf(8.f * (float)id + 1.f) - 1.f) * 0.5f);
    while (tj * (tj + 1) / 2 > id) --tj;
    while ((tj + 1) * (tj + 2) / 2 <= id) ++tj;
    ti = id - tj * (tj + 1) / 2;
  } else {
    const int64_t down = (at.kp + TILE - 1) / TILE;
    ti = id % down, tj = id / down;
  }
  const char* A = place + (STAGE == kGram ? at.x : STAGE == kPolynomial ? at.s : at.p);
  const char* B = place + (STAGE == kGram ? at.x : STAGE == kPolynomial ? at.s : at.xt[turn]);
  const int64_t row_bytes = STAGE == kGram ? at.l_row : at.k_row;
  const int64_t b_rows = STAGE <= kPolynomial ? at.kp : at.lp;
  const int steps = (int)(row_bytes / 128);

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const char* from[S::LOADS];
#pragma unroll
  for (int r = 0; r < S::LOADS; ++r) {
    const int row = r * (S::THREADS / 8) + wave * 8 + lane / 8;   // of A's rows, then B's
    const bool second = r >= S::LOADS / 2;
    int64_t global = second ? tj * TILE + row - TILE : ti * TILE + row;
    const int64_t most = (second ? b_rows : at.kp) - 1;
    global = global < most ? global : most;         // tiles that pass the end: their last rows again, not written
    from[r] = (second ? B : A) + global * row_bytes + ((lane % 8) ^ (lane / 8)) * 16;
  }
  auto request = [&](int step) {
    char* to = lds[step & 1] + wave * 8 * 128;
#pragma unroll
    for (int r = 0; r < S::LOADS; ++r)
      __builtin_amdgcn_global_load_lds((Global)(from[r] + (int64_t)step * 128), (Lds)(to + r * S::THREADS * 16), 16, 0, 0);
  };

  floatx16 acc[S::Y][S::X];
#pragma unroll
  for (int y = 0; y < S::Y; ++y)
#pragma unroll
    for (int x = 0; x < S::X; ++x)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[y][x][v] = 0.f;

  const int half = lane / 32, wy = wave / S::ACROSS * S::Y * 32, wx = wave % S::ACROSS * S::X * 32;
  request(0);
  for (int step = 0; step < steps; ++step) {
    step_barrier();
    if (step + 1 < steps) request(step + 1);
    const char* buffer = lds[step & 1];
    auto operand = [&](int row, int chunk) { return *reinterpret_cast<const f16x8*>(buffer + chunk_at(row, chunk)); };
#pragma unroll
    for (int kk = 0; kk < (SPLIT ? 2 : 4); ++kk) {
      f16x8 a[S::Y][2], b[S::X][2];
#pragma unroll
      for (int piece = 0; piece < (SPLIT ? 2 : 1); ++piece) {
#pragma unroll
        for (int x = 0; x < S::X; ++x) b[x][piece] = operand(TILE + wx + x * 32 + lane % 32, piece * 4 + kk * 2 + half);
#pragma unroll
        for (int y = 0; y < S::Y; ++y) a[y][piece] = operand(wy + y * 32 + lane % 32, piece * 4 + kk * 2 + half);
      }
#pragma unroll
      for (int y = 0; y < S::Y; ++y)
#pragma unroll
        for (int x = 0; x < S::X; ++x) {
          if constexpr (SPLIT) {
            acc[y][x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[y][1], b[x][0], acc[y][x], 0, 0, 0);
            acc[y][x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[y][0], b[x][1], acc[y][x], 0, 0, 0);
          }
          acc[y][x] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[y][0], b[x][0], acc[y][x], 0, 0, 0);
        }
    }
  }
  step_barrier();   // the buffers are free

  char* scratch = &lds[0][0] + wave * 8192;
  const bool mirrored = STAGE <= kPolynomial && ti == tj;
#pragma unroll
  for (int y = 0; y < S::Y; ++y)
#pragma unroll
    for (int x = 0; x < S::X; ++x) {
      const int64_t i0 = ti * TILE + wy + y * 32, j0 = tj * TILE + wx + x * 32;
      if (i0 >= at.kp || j0 >= b_rows) continue;
      floatx16 v;
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = acc[y][x][e] * (STAGE == kLast ? kDown * kDown : kDown);
      if constexpr (STAGE == kPolynomial) {   // a I + b S + c S S; S is its own transpose
        const int64_t j = j0 + lane % 32;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t row = i0 + 8 * q + 4 * half;
          float old[4];
          read_values<SPLIT, 4>(place + at.s + j * at.k_row, row, old);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[4 * q + e] = fmaf(s.c, v[4 * q + e], s.b * old[e]) + (row + e == j ? s.a * kScale : 0.f);
        }
      }
      if constexpr (STAGE == kLast) {
        const bool tall = t.rows[i] > t.columns[i];
        write_result<T>(v, scratch, lane, (T*)t.p[i], tall ? at.k : at.l, tall, tall ? j0 : i0, tall ? i0 : j0,
                        tall ? at.l : at.k, tall ? at.k : at.l, t.m[i] != nullptr, s.keep, t.rate[i]);
      } else {
        char* rows_to = place + (STAGE == kGram ? at.s : STAGE == kPolynomial ? at.p : at.x);
        char* columns_to = STAGE == kNext ? place + at.xt[turn ^ 1] : rows_to;
        const int64_t rows_bytes = STAGE == kNext ? at.l_row : at.k_row;
        write_block<SPLIT>(v, scratch, lane, place_of<SPLIT>(rows_to + i0 * rows_bytes, j0), rows_bytes,
                           mirrored ? nullptr : place_of<SPLIT>(columns_to + j0 * at.k_row, i0), at.k_row);
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

template <bool SPLIT, int TILE, int STAGE, typename T>
void multiply(Table& t, int used, const Settings& s, char* workspace, int turn, hipStream_t stream) {
  const int64_t groups = deal(t, used, [](const Layout& at) {
    const int64_t down = ceil_div(at.kp, TILE);
    return STAGE <= kPolynomial ? triangle(down) : down * ceil_div(at.lp, TILE);
  });
  launch(product<SPLIT, TILE, STAGE, T>, dim3((unsigned)groups), dim3(Shape<TILE>::THREADS), stream, t, s, workspace, turn);
}

template <bool SPLIT, int STAGE, typename T>
void stage(Table& t, int used, const Settings& s, char* workspace, int turn, hipStream_t stream, int tile) {
  if (tile == 128)
    multiply<SPLIT, 128, STAGE, T>(t, used, s, workspace, turn, stream);
  else
    multiply<SPLIT, 64, STAGE, T>(t, used, s, workspace, turn, stream);
}

template <typename T>
void run_group(Table& t, int used, const Settings& s, int steps, char* workspace, hipStream_t stream) {
  constexpr bool SPLIT = !std::is_same<T, bf16>::value;
  int64_t groups = deal(t, used, [](const Layout& at) { return ceil_div(at.k * at.l, kPerGroup); });
  launch(squares<T>, dim3((unsigned)groups), dim3(256), stream, t, s, workspace, (int)SPLIT);
  groups = deal(t, used, [](const Layout& at) { return at.kp / 64 * (at.lp / 64); });
  launch(lay_out<T, SPLIT>, dim3((unsigned)groups), dim3(256), stream, t, s, workspace);
  // tiles of 128 where they fill the GPU
  const int tile = groups >= 1024 ? 128 : 64;
  for (int step = 0; step < steps; ++step) {
    const int turn = step & 1;
    stage<SPLIT, kGram, f16>(t, used, s, workspace, turn, stream, tile);
    stage<SPLIT, kPolynomial, f16>(t, used, s, workspace, turn, stream, tile);
    if (step + 1 < steps)
      stage<SPLIT, kNext, f16>(t, used, s, workspace, turn, stream, tile);
    else
      stage<SPLIT, kLast, T>(t, used, s, workspace, turn, stream, tile);
  }
}

// Deals the matrices to groups that share the workspace one after another: 64 at most, and as many workgroups as a
// launch holds.  `run` gets a table and how many it holds; returns the bytes of the largest group.
template <typename Get, typename Run>
size_t in_groups(int64_t count, int dtype, Get get, Run run) {
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
    if (x.rows < 1 || x.columns < 1) continue;
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

constexpr int64_t kMostSide = 1 << 17;

int check_matrix(int64_t rows, int64_t columns) {
  SDK_REQUIRE(rows >= 0 && columns >= 0 && rows <= kMostSide && columns <= kMostSide &&
                  rows * columns <= (int64_t)1 << 31,
              "a matrix of %lld x %lld: sides up to 131072, 2^31 values", (long long)rows, (long long)columns);
  return SDK_OK;
}

int check_settings(int64_t count, int64_t steps, const double* coefficients, double eps, int dtype) {
  SDK_REQUIRE(known(dtype), "unknown dtype %d (float32, bfloat16 and float16 only)", dtype);
  SDK_REQUIRE(count >= 0, "count must not be negative");
  SDK_REQUIRE(steps >= 1 && steps <= 100, "steps = %lld must be between 1 and 100", (long long)steps);
  SDK_REQUIRE(coefficients, "coefficients must not be NULL");
  for (int i = 0; i < 3; ++i)
    SDK_REQUIRE(std::fabs(coefficients[i]) <= 100, "coefficients must be numbers up to 100 in magnitude");
  SDK_REQUIRE(eps >= 0x1p-100 && eps <= 1, "eps = %g must be between 2^-100 and 1", eps);
  return SDK_OK;
}

Settings settings_of(const double* c, double eps) {
  Settings s = {};
  s.a = (float)c[0], s.b = (float)c[1], s.c = (float)c[2], s.eps = (float)eps;
  return s;
}

int run_all(int64_t count, int steps, const Settings& s, void* workspace, size_t workspace_bytes, int dtype,
            sdk_stream_t stream, Matrix (*get)(const void*, int64_t), const void* context) {
  auto of = [&](int64_t i) { return get(context, i); };
  const size_t need = in_groups(count, dtype, of, [](Table&, int) {});
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 128))
    return fail(SDK_ERR_WORKSPACE, "workspace of %zu bytes at a multiple of 128, %zu needed", workspace_bytes, need);
  in_groups(count, dtype, of, [&](Table& t, int used) {
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

}  // namespace
}  // namespace token
}  // namespace sdk

using namespace sdk;
using namespace sdk::token;

extern "C" {

size_t sdk_orthogonalize_workspace_bytes(int64_t rows, int64_t columns, int64_t count, int32_t dtype) {
  if (check_matrix(rows, columns) != SDK_OK || !known(dtype) || count < 0) return 0;
  count = std::min<int64_t>(count, kMatrices);
  return in_groups(count, dtype, [&](int64_t) { return Matrix{nullptr, nullptr, nullptr, rows, columns, 0.f}; },
                   [](Table&, int) {});
}

int sdk_orthogonalize(const void* x, void* out, int64_t rows, int64_t columns, int64_t count, int32_t steps,
                      const double* coefficients, double eps, void* workspace, size_t workspace_bytes, int32_t dtype,
                      sdk_stream_t stream) {
  if (int rc = check_settings(count, steps, coefficients, eps, dtype)) return rc;
  if (int rc = check_matrix(rows, columns)) return rc;
  if (!count || !rows || !columns) return SDK_OK;
  SDK_REQUIRE(x && out, "x and out must not be NULL");
  const Stack stack = {(const char*)x, (char*)out, rows, columns, rows * columns * (int64_t)bytes_of(dtype)};
  const int rc = run_all(count, steps, settings_of(coefficients, eps), workspace, workspace_bytes, dtype, stream,
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
  return in_groups(count, dtype, [&](int64_t i) { return Matrix{nullptr, nullptr, nullptr, rows[i], columns[i], 0.f}; },
                   [](Table&, int) {});
}

int sdk_muon_step(void* const* params, const void* const* grads, float* const* momenta, const int64_t* rows,
                  const int64_t* columns, int64_t count, double lr, double momentum, int32_t nesterov,
                  double weight_decay, int32_t steps, const double* coefficients, double eps, void* workspace,
                  size_t workspace_bytes, int32_t dtype, sdk_stream_t stream) {
  if (int rc = check_settings(count, steps, coefficients, eps, dtype)) return rc;
  SDK_REQUIRE(lr >= 0 && weight_decay >= 0 && momentum >= 0 && momentum < 1 && lr <= 1e30 && weight_decay <= 1e30,
              "lr and weight_decay must not be negative, momentum in [0, 1)");
  if (!count) return SDK_OK;
  SDK_REQUIRE(params && grads && momenta && rows && columns, "the lists must not be NULL");
  for (int64_t i = 0; i < count; ++i) {
    if (int rc = check_matrix(rows[i], columns[i])) return rc;
    SDK_REQUIRE(!rows[i] || !columns[i] || (params[i] && grads[i] && momenta[i]), "matrix %lld: a tensor is NULL",
                (long long)i);
  }
  Settings s = settings_of(coefficients, eps);
  s.mu = (float)momentum, s.rest = (float)(1 - momentum), s.keep = (float)(1 - lr * weight_decay);
  s.nesterov = nesterov != 0;
  const Lists lists = {params, grads, momenta, rows, columns, lr};
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
