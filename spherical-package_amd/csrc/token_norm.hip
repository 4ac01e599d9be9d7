// Addition of the residual and root-mean-square norm of rows, with gradients, and the same with rows in
// 8 bits and a scale each.
//
//   h = x + r            y_j = w_j h_j inv,  inv = 1 / sqrt(mean_j h_j^2 + eps)
//   dh_j = inv (w_j g_j - h_j inv^2 mean_i(w_i g_i h_i)) + s_j      (g, s: the gradients of y and h)
//   dw_j = sum over rows of g_j h_j inv
//
// All of it is bound by memory: a row is read once, held in registers, and every sum over it (squares,
// largest magnitude, w g h) is formed there.  Sums are float32.  The forward normalises the sum before it is
// rounded to the tensors' type; the backward reads the rounded h, which the forward wrote (2 bytes a value less than
// float32 sums): gradients are off by 2.5e-3 of their size in bfloat16, 1.7e-3 of it their own rounding.
#include <algorithm>

#include "token_types.hpp"

namespace sdk {
namespace token {
namespace {

// A row is dealt to THREADS threads, N chunks of V elements each: chunk k of thread t begins at
// (k * THREADS + t) * V, so that a wave reads consecutive memory.  Workgroups of at least 256 threads:
// narrow rows share one.
// 65536 rows of 1024 bfloat16 values: forward 87 us (6.2 TB/s of rows read and written), backward 110 us (4.9 TB/s), of
// which the weight's sum over 1024 workgroups is 4.  Rows of fewer 16-byte vectors than 64 leave lanes without work: 2^26
// bfloat16 values in rows of 64, 128 and 256 take 384, 211 and 126 us forward, of 512 90.
template <int THREADS>
constexpr int kGroup = THREADS < 256 ? 256 : THREADS;

constexpr int kPlain = 0, kInt8 = 1, kFp8 = 2;
constexpr float kSmallestRow = 0x1p-100f;   // rows below it are zeros in 8 bits: 1 / scale stays finite

template <typename T, int V, int N, int THREADS, bool ALIGNED>
__global__ __launch_bounds__(kGroup<THREADS>) void norm_forward(
    const T* x, const T* residual, const void* weight, int weight_float, void* out, float* scales,
    T* summed, float* inverse, int64_t rows, int width, float eps, int codes) {
  __shared__ float slots[kGroup<THREADS> / 64];
  const int t = threadIdx.x % THREADS;
  const int64_t row = (int64_t)blockIdx.x * (kGroup<THREADS> / THREADS) + threadIdx.x / THREADS;
  const bool live = row < rows;
  const int64_t base = row * width;
  float h[N][V];
  float sq = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int j = (k * THREADS + t) * V;
    if (live && j < width) {
      get<T, V, ALIGNED>(x + base + j, h[k], width - j);
      if (residual) {
        float r[V];
        get<T, V, ALIGNED>(residual + base + j, r, width - j);
#pragma unroll
        for (int e = 0; e < V; ++e) h[k][e] += r[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) h[k][e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) sq += h[k][e] * h[k][e];
  }
  if (summed) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int j = (k * THREADS + t) * V;
      if (live && j < width) put<T, V, ALIGNED>(summed + base + j, h[k], width - j);
    }
  }
  sq = over_group<Add, THREADS>(sq, slots);
  const float inv = 1.f / sqrtf(sq / (float)width + eps);
  if (inverse && live && t == 0) inverse[row] = inv;
  float largest = 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int j = (k * THREADS + t) * V;
    if (j < width) {
      float w[V];
      load_weight<T, V, ALIGNED>(weight, weight_float, j, w, width - j);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        h[k][e] = h[k][e] * inv * w[e];
        if (codes != kPlain) largest = Largest::of(largest, fabsf(h[k][e]));
      }
      if (codes == kPlain && live) put<T, V, ALIGNED>((T*)out + base + j, h[k], width - j);
    }
  }
  if (codes == kPlain) return;
  largest = over_group<Largest, THREADS>(largest, slots);
  const float most = codes == kInt8 ? 127.f : 448.f;
  const bool some = !(largest < kSmallestRow);   // a row with a NaN keeps it in its scale
  const float up = some ? most / largest : 0.f;
  if (live && t == 0) scales[row] = some ? largest * (1.f / most) : 0.f;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int j = (k * THREADS + t) * V;
    if (live && j < width) {
      Pack<unsigned char, V> c;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        // v * up can pass the largest code by an ulp (127.00001, 448.00003): both roundings take it back
        const float v = h[k][e] * up;
        if (codes == kInt8)
          c.v[e] = (unsigned char)(signed char)(int)rintf(v);
        else
          c.v[e] = (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(
                       fminf(fmaxf(v, -448.f), 448.f), 0.f, 0, false) & 0xff);
      }
      unsigned char* to = (unsigned char*)out + base + j;
      if (ALIGNED || j + V <= width) {
        __builtin_memcpy(ALIGNED ? (unsigned char*)__builtin_assume_aligned(to, V) : to, &c, V);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (j + e < width) to[e] = c.v[e];
      }
    }
  }
}

// Workgroup b takes rows b, b + gridDim.x, ... (times the rows that share a workgroup) and keeps its part of
// dw in registers; the parts are joined in their order by norm_weight_grad.
template <typename T, int V, int N, int THREADS, bool ALIGNED>
__global__ __launch_bounds__(kGroup<THREADS>) void norm_backward(
    const T* grad, const T* grad_sum, const T* h_in, const void* weight, int weight_float,
    const float* inverse, T* grad_x, float* parts, int64_t rows, int width) {
  constexpr int SHARE = kGroup<THREADS> / THREADS;
  __shared__ float slots[kGroup<THREADS> / 64];
  const int t = threadIdx.x % THREADS, sub = threadIdx.x / THREADS;
  float w[N][V], dw[N][V];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int j = (k * THREADS + t) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) w[k][e] = dw[k][e] = 0.f;
    if (j < width) load_weight<T, V, ALIGNED>(weight, weight_float, j, w[k], width - j);
  }
  for (int64_t first = (int64_t)blockIdx.x * SHARE; first < rows; first += (int64_t)gridDim.x * SHARE) {
    const int64_t row = first + sub, base = row * width;
    const bool live = row < rows;
    const float inv = live ? inverse[row] : 0.f;
    float h[N][V], g[N][V], dot = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int j = (k * THREADS + t) * V;
      if (live && j < width) {
        get<T, V, ALIGNED>(h_in + base + j, h[k], width - j);
        get<T, V, ALIGNED>(grad + base + j, g[k], width - j);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) h[k][e] = g[k][e] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        dw[k][e] += g[k][e] * (h[k][e] * inv);
        g[k][e] *= w[k][e];
        dot += g[k][e] * h[k][e];
      }
    dot = over_group<Add, THREADS>(dot, slots);
    if (grad_x) {
      const float along = inv * inv * (dot / (float)width);
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int j = (k * THREADS + t) * V;
        if (live && j < width) {
          float s[V];
#pragma unroll
          for (int e = 0; e < V; ++e) s[e] = 0.f;
          if (grad_sum) get<T, V, ALIGNED>(grad_sum + base + j, s, width - j);
#pragma unroll
          for (int e = 0; e < V; ++e) s[e] += inv * (g[k][e] - h[k][e] * along);
          put<T, V, ALIGNED>(grad_x + base + j, s, width - j);
        }
      }
    }
  }
  if (!parts) return;
  // the rows that share the workgroup are joined in LDS
  float* to = parts + (int64_t)blockIdx.x * width;
  if constexpr (SHARE > 1) {
    __shared__ float joined[SHARE][THREADS * N * V];
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) joined[sub][(k * V + e) * THREADS + t] = dw[k][e];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int j = (k * THREADS + t) * V + e;
        if ((k * V + e) % SHARE == sub && j < width) {
          float x = 0.f;
#pragma unroll
          for (int i = 0; i < SHARE; ++i) x += joined[i][(k * V + e) * THREADS + t];
          to[j] = x;
        }
      }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int j = (k * THREADS + t) * V;
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (j + e < width) to[j + e] = dw[k][e];
    }
  }
}

// dw[j] = sum over the parts: 64 columns a workgroup, a sixteenth of the parts a wave, eight at a time.
template <typename T>
__global__ __launch_bounds__(1024) void norm_weight_grad(const float* parts, int64_t count, int width,
                                                         void* grad_weight, int is_float) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int j = blockIdx.x * 64 + lane;
  const int64_t each = (count + 15) / 16, from = wave * each, to = from + each < count ? from + each : count;
  float s = 0.f;
  if (j < width) {
    int64_t i = from;
    for (; i + 8 <= to; i += 8) {
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = parts[(i + u) * width + j];
      s += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    }
    for (; i < to; ++i) s += parts[i * width + j];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && j < width) {
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += sums[w][lane];
    if (is_float)
      ((float*)grad_weight)[j] = s;
    else
      ((T*)grad_weight)[j] = (T)s;
  }
}

// out = codes * scale of the row, eight codes a thread; rows whose width is no multiple of eight end inside a thread's
// eight.
template <typename T>
__global__ __launch_bounds__(256) void dequantize(const unsigned char* codes, const float* scales, T* out, int64_t size,
                                                  int width, int fp8, int wide) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (at >= size) return;
  int64_t row = at / width;
  int left = (int)(width - (at - row * width));   // codes of this row from the thread's first on
  float s = scales[row];
  auto value = [&](unsigned char c) {
    return (fp8 ? __builtin_amdgcn_cvt_f32_fp8((int)c, 0) : (float)(signed char)c) * s;
  };
  if (wide && at + 8 <= size) {
    const Pack<unsigned char, 8> q = *reinterpret_cast<const Pack<unsigned char, 8>*>(codes + at);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (left == 0) s = scales[++row], left = width;
      f[e] = value(q.v[e]);
      --left;
    }
#pragma unroll
    for (int e = 0; e < 8; e += kWide<T>) store_pack<T, kWide<T>>(out + at + e, *reinterpret_cast<float(*)[kWide<T>]>(f + e));
  } else {
    for (int e = 0; e < 8 && at + e < size; ++e) {
      if (left == 0) s = scales[++row], left = width;
      out[at + e] = (T)value(codes[at + e]);
      --left;
    }
  }
}

// Threads of a row: at most 16 elements a thread.
int threads_of(int64_t width) { return width <= 1024 ? 64 : width <= 4096 ? 256 : 1024; }
constexpr int64_t kMostWidth = 16384;

// Runs `CALL` with V, N, THREADS and ALIGNED for rows of `width`; `wide`: 16-byte vectors fit rows and pointers.  (Rows
// that they do not fit are read by vectors all the same, at whatever address they begin: 41458 rows of 1235 float32
// values to int8 and back 194 us, value by value 298.)
#define NORM_SHAPE_N(NN, ...)                                             \
  do {                                                                    \
    constexpr int N = NN;                                                 \
    if (threads == 64) { constexpr int THREADS = 64; __VA_ARGS__; }       \
    else if (threads == 256) { constexpr int THREADS = 256; __VA_ARGS__; } \
    else { constexpr int THREADS = 1024; __VA_ARGS__; }                   \
  } while (0)
#define NORM_SHAPE_V(...)                                                 \
  do {                                                                    \
    constexpr int V = kWide<T>;                                           \
    const int64_t n = ceil_div(width, (int64_t)threads * V);              \
    if (n <= 1) NORM_SHAPE_N(1, __VA_ARGS__);                             \
    else if (n <= 2) NORM_SHAPE_N(2, __VA_ARGS__);                        \
    else if constexpr (V <= 4) NORM_SHAPE_N(4, __VA_ARGS__);              \
  } while (0)
#define NORM_SHAPE(...)                                                   \
  do {                                                                    \
    const int threads = threads_of(width);                                \
    if (wide) { constexpr bool ALIGNED = true; NORM_SHAPE_V(__VA_ARGS__); } \
    else { constexpr bool ALIGNED = false; NORM_SHAPE_V(__VA_ARGS__); }   \
  } while (0)

// The rows in launches of as many as one holds.
template <typename T, int V, int N, int THREADS, bool ALIGNED>
void run_forward(const T* x, const T* residual, const void* weight, int weight_float, void* out, float* scales, T* summed,
                 float* inverse, int64_t rows, int width, float eps, int codes, hipStream_t s) {
  constexpr int SHARE = kGroup<THREADS> / THREADS;
  constexpr int64_t EACH = most_groups(kGroup<THREADS>) * SHARE;
  for (int64_t row = 0; row < rows; row += EACH) {
    const int64_t count = std::min(EACH, rows - row), at = row * width;
    launch(norm_forward<T, V, N, THREADS, ALIGNED>, dim3((unsigned)ceil_div(count, SHARE)), dim3(kGroup<THREADS>), s, x + at,
           residual ? residual + at : nullptr, weight, weight_float,
           (void*)((char*)out + at * (codes == kPlain ? (int64_t)sizeof(T) : 1)), scales ? scales + row : nullptr,
           summed ? summed + at : nullptr, inverse ? inverse + row : nullptr, count, width, eps, codes);
  }
}

int64_t backward_groups(int64_t rows, int64_t width) {
  const int threads = threads_of(width), share = threads < 256 ? 256 / threads : 1;
  const int64_t groups = threads == 1024 ? 512 : 1024;
  return std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, share), groups));
}

int check(int64_t rows, int64_t width, int dtype, int weight_dtype) {
  SDK_REQUIRE(rows >= 0 && rows < (int64_t)1 << 31, "rows = %lld must be between 0 and 2^31", (long long)rows);
  SDK_REQUIRE(width >= 1 && width <= kMostWidth, "width = %lld must be between 1 and %lld",
              (long long)width, (long long)kMostWidth);
  SDK_REQUIRE(known(dtype), "unknown dtype %d (float32, bfloat16 and float16 only)", dtype);
  SDK_REQUIRE(weight_dtype == dtype || weight_dtype == SDK_F32,
              "weight's dtype %d must be the rows' or float32", weight_dtype);
  return SDK_OK;
}

}  // namespace
}  // namespace token
}  // namespace sdk

using namespace sdk;
using namespace sdk::token;

extern "C" {

int sdk_add_rms_norm(const void* x, const void* residual, const void* weight, void* out, float* scales,
                     void* summed, float* inverse, int64_t rows, int64_t width, double eps, int32_t codes,
                     int32_t dtype, int32_t weight_dtype, sdk_stream_t stream) {
  if (int rc = check(rows, width, dtype, weight_dtype)) return rc;
  SDK_REQUIRE(codes >= 0 && codes <= 2, "codes = %d must be 0 (none), 1 (int8) or 2 (float8 e4m3)", codes);
  SDK_REQUIRE(eps >= 0, "eps must not be negative");
  if (rows == 0) return SDK_OK;
  SDK_REQUIRE(x && weight && out, "x, weight and out must not be NULL");
  SDK_REQUIRE(codes == 0 || scales, "scales must not be NULL where the output is in 8 bits");
  hipStream_t s = (hipStream_t)stream;
  SDK_DISPATCH_TOKEN_DTYPE(dtype, {
    const bool wide = width % kWide<T> == 0 && aligned16(x) && aligned16(residual) && aligned16(weight) &&
                      aligned16(out) && aligned16(summed);
    NORM_SHAPE(run_forward<T, V, N, THREADS, ALIGNED>((const T*)x, (const T*)residual, weight, weight_dtype == SDK_F32, out,
                                                      scales, (T*)summed, inverse, rows, (int)width, (float)eps,
                                                      (int)codes, s));
  });
  SDK_LAUNCH_CHECK("add_rms_norm");
  return SDK_OK;
}

size_t sdk_add_rms_norm_backward_workspace_bytes(int64_t rows, int64_t width) {
  if (rows < 1 || width < 1 || width > kMostWidth) return 0;
  return (size_t)backward_groups(rows, width) * width * sizeof(float);
}

int sdk_add_rms_norm_backward(const void* grad, const void* grad_sum, const void* summed, const void* weight,
                              const float* inverse, void* grad_x, void* grad_weight, void* workspace,
                              size_t workspace_bytes, int64_t rows, int64_t width, int32_t dtype,
                              int32_t weight_dtype, sdk_stream_t stream) {
  if (int rc = check(rows, width, dtype, weight_dtype)) return rc;
  SDK_REQUIRE(weight && (grad_x || grad_weight), "weight and one gradient at least must not be NULL");
  SDK_REQUIRE(rows == 0 || (grad && summed && inverse), "grad, summed and inverse must not be NULL");
  const size_t need = grad_weight ? sdk_add_rms_norm_backward_workspace_bytes(rows, width) : 0;
  if (need && (!workspace || workspace_bytes < need))
    return fail(SDK_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  hipStream_t s = (hipStream_t)stream;
  const int64_t groups = rows ? backward_groups(rows, width) : 0;
  float* parts = grad_weight ? (float*)workspace : nullptr;
  SDK_DISPATCH_TOKEN_DTYPE(dtype, {
    const bool wide = width % kWide<T> == 0 && aligned16(grad) && aligned16(grad_sum) && aligned16(summed) &&
                      aligned16(weight) && aligned16(grad_x);
    if (rows)
      NORM_SHAPE(launch(norm_backward<T, V, N, THREADS, ALIGNED>, dim3((unsigned)groups), dim3(kGroup<THREADS>), s,
                        (const T*)grad, (const T*)grad_sum, (const T*)summed, weight,
                        (int)(weight_dtype == SDK_F32), inverse, (T*)grad_x, parts, rows, (int)width));
    if (grad_weight)
      launch(norm_weight_grad<T>, dim3((unsigned)ceil_div(width, 64)), dim3(1024), s, (const float*)parts,
             groups, (int)width, grad_weight, (int)(weight_dtype == SDK_F32));
  });
  SDK_LAUNCH_CHECK("add_rms_norm_backward");
  return SDK_OK;
}

int sdk_dequantize_rows(const void* codes, const float* scales, void* out, int64_t rows, int64_t width,
                        int32_t codes_kind, int32_t dtype, sdk_stream_t stream) {
  SDK_REQUIRE(rows >= 0 && rows < (int64_t)1 << 31 && width >= 1 && width < (int64_t)1 << 31,
              "rows %lld of width %lld", (long long)rows, (long long)width);
  SDK_REQUIRE(codes_kind == kInt8 || codes_kind == kFp8, "codes = %d must be 1 (int8) or 2 (float8 e4m3)",
              codes_kind);
  SDK_REQUIRE(known(dtype), "unknown dtype %d (float32, bfloat16 and float16 only)", dtype);
  if (rows == 0) return SDK_OK;
  SDK_REQUIRE(codes && scales && out, "codes, scales and out must not be NULL");
  hipStream_t s = (hipStream_t)stream;
  const int64_t each = most_groups(256) * 2048 / width;   // rows of a launch: 16 at least
  SDK_DISPATCH_TOKEN_DTYPE(dtype, for (int64_t row = 0; row < rows; row += each) {
    const unsigned char* from = (const unsigned char*)codes + row * width;
    T* to = (T*)out + row * width;
    const int64_t size = std::min(each, rows - row) * width;
    const int wide = ((uintptr_t)from & 7) == 0 && aligned16(to);
    launch(dequantize<T>, dim3((unsigned)ceil_div(size, 2048)), dim3(256), s, from, scales + row, to, size, (int)width,
           (int)(codes_kind == kFp8), wide);
  });
  SDK_LAUNCH_CHECK("dequantize_rows");
  return SDK_OK;
}

}  // extern "C"
