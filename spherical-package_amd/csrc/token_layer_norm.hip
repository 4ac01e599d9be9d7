// Addition of the residual and layer norm of rows, with the gradients of rows, weight and bias.
//
//   h = x + r     z_j = (h_j - mu) inv,  mu = mean_j h_j,  inv = 1 / sqrt(mean_j (h_j - mu)^2 + eps)
//   y_j = w_j z_j + b_j
//   dh_j = inv (q_j - mean_i q_i - z_j mean_i (q_i z_i)) + s_j,  q = w g     (g, s: the gradients of y and h)
//   dw_j = sum over rows of g_j z_j,  db_j = sum over rows of g_j
//
// Bound by memory: a row is read once and held in registers, where the mean is formed first and the squares of the
// distances from it after (their difference from sums of squares would lose a mean's square).  Sums are float32, and h is
// normalised before it is rounded to the tensors' type, in the backward too: there it is formed again from x and r.  h as
// the forward wrote it would be one read less (42 us for 46.7, 32768 rows of 768 bfloat16 values), but dw then carries h's
// rounding beside its own (2.5e-3 of its size for 1.8e-3).  In float32 that does not show, and h is read.
// 32768 rows of 768 bfloat16 values with residual: forward 32 us (201 MB, in part from the caches), backward 47 (252 MB, 5.4
// TB/s), joining the parts of dw and db 4.
#include <algorithm>

#include "token_types.hpp"

namespace sdk {
namespace token {
namespace {

// A row is dealt to THREADS threads (4 to 1024, the fewest that take it with 16 values each), in chunks of 16 bytes:
// chunk k of thread t begins at (k * THREADS + t) * V.  Workgroups of at least 256 threads: narrow rows share one.
template <int THREADS>
constexpr int kGroup = THREADS < 256 ? 256 : THREADS;
template <typename T>
constexpr int kChunks = 16 / kWide<T>;
constexpr int64_t kMostWidth = 16384;

// The sums of COUNT values over the row's threads.  slots: COUNT floats a wave, used again only after a barrier of another
// call.
template <int THREADS, int COUNT>
__device__ __forceinline__ void row_sums(float (&x)[COUNT], float (*slots)[COUNT]) {
#pragma unroll
  for (int c = 0; c < COUNT; ++c) x[c] = lane_sum<(THREADS < 64 ? THREADS : 64)>(x[c]);
  if constexpr (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int c = 0; c < COUNT; ++c) slots[threadIdx.x >> 6][c] = x[c];
    }
    __syncthreads();
    const int first = threadIdx.x / THREADS * (THREADS / 64);
#pragma unroll
    for (int c = 0; c < COUNT; ++c) {
      x[c] = slots[first][c];
#pragma unroll
      for (int w = 1; w < THREADS / 64; ++w) x[c] += slots[first + w][c];
    }
  }
}

// 16 bytes of a row as they lie in memory, `left` of their V values in the row.  A row that fits no vector ends inside one:
// what follows is the next row (`more`: there is one) and is read with it; the user leaves it out (in_row).  Words, not
// values: of values the compiler makes a request each.
typedef unsigned Words __attribute__((ext_vector_type(4)));
template <typename T, int V, bool ALIGNED>
__device__ __forceinline__ Words row_get(const T* p, int left, bool more) {
  typedef Words AnyWords __attribute__((aligned(2)));
  if (ALIGNED) return *reinterpret_cast<const Words*>(p);
  if (left >= V || more) return *reinterpret_cast<const AnyWords*>(p);
  Pack<T, V> x;
#pragma unroll
  for (int e = 0; e < V; ++e) x.v[e] = e < left ? p[e] : (T)0.f;
  return __builtin_bit_cast(Words, x);
}
template <typename T, int V, bool ALIGNED>
__device__ __forceinline__ void in_row(Words w, float (&f)[V], int left) {
  const Pack<T, V> x = __builtin_bit_cast(Pack<T, V>, w);
#pragma unroll
  for (int e = 0; e < V; ++e) f[e] = ALIGNED || e < left ? (float)x.v[e] : 0.f;
}

// The same into memory: what a vector does not hold goes in halves, quarters, ...
template <typename T, int V, bool ALIGNED>
__device__ __forceinline__ void row_put(T* p, const float (&f)[V], int left) {
  if (ALIGNED || left >= V) {
    put<T, V, ALIGNED>(p, f, left);
    return;
  }
  Pack<T, V> x;
#pragma unroll
  for (int e = 0; e < V; ++e) x.v[e] = (T)f[e];
  if constexpr (V == 8) {
    if (left & 4) {
      __builtin_memcpy(p, &x, 4 * sizeof(T));
      p += 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) x.v[e] = x.v[e + 4];
    }
  }
  if (left & 2) {
    __builtin_memcpy(p, &x, 2 * sizeof(T));
    p += 2;
    x.v[0] = x.v[2];
  }
  if (left & 1) *p = x.v[0];
}

// Rows of whole vectors: a workgroup a row (or the rows that share one).  Others: workgroup b takes rows b, b + gridDim.x,
// and so on, so that the weight's end, which has to be read in single values, is read once.
template <typename T, int THREADS, bool ALIGNED>
__global__ __launch_bounds__(kGroup<THREADS>) void layer_forward(const T* x, const T* residual, const void* weight,
                                                                 const void* bias, int weight_float, T* out, T* summed,
                                                                 float* mean, float* inverse, int64_t rows, int width,
                                                                 float eps) {
  constexpr int V = kWide<T>, N = kChunks<T>, SHARE = kGroup<THREADS> / THREADS;
  __shared__ float slots[2][kGroup<THREADS> / 64][1];
  const int t = threadIdx.x % THREADS;
  float w[N][V], b[N][V];
  auto weights = [&](int k) {
    const int j = (k * THREADS + t) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) w[k][e] = b[k][e] = 0.f;
    if (j < width) {
      load_weight<T, V, ALIGNED>(weight, weight_float, j, w[k], width - j);
      if (bias) load_weight<T, V, ALIGNED>(bias, weight_float, j, b[k], width - j);
    }
  };
  if (!ALIGNED) {
#pragma unroll
    for (int k = 0; k < N; ++k) weights(k);
  }
  for (int64_t first = (int64_t)blockIdx.x * SHARE; first < rows; first += (int64_t)gridDim.x * SHARE) {
    const int64_t row = first + threadIdx.x / THREADS, base = row * width;
    const bool live = row < rows, more = row + 1 < rows && width >= V;
    float h[N][V];
    float sum[1] = {0.f}, sq[1] = {0.f};
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int j = (k * THREADS + t) * V;
      Words a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
      if (live && j < width) {
        a = row_get<T, V, ALIGNED>(x + base + j, width - j, more);
        if (residual) b = row_get<T, V, ALIGNED>(residual + base + j, width - j, more);
      }
      float r[V];
      in_row<T, V, ALIGNED>(a, h[k], width - j);
      in_row<T, V, ALIGNED>(b, r, width - j);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        h[k][e] += r[e];
        sum[0] += h[k][e];
      }
    }
    if (summed) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int j = (k * THREADS + t) * V;
        if (live && j < width) row_put<T, V, ALIGNED>(summed + base + j, h[k], width - j);
      }
    }
    row_sums<THREADS>(sum, slots[0]);
    const float mu = sum[0] / (float)width;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int left = width - (k * THREADS + t) * V;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        h[k][e] -= mu;
        if (e < left) sq[0] += h[k][e] * h[k][e];
      }
    }
    row_sums<THREADS>(sq, slots[1]);
    const float inv = 1.f / sqrtf(sq[0] / (float)width + eps);
    if (live && t == 0) {
      if (mean) mean[row] = mu;
      if (inverse) inverse[row] = inv;
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int j = (k * THREADS + t) * V;
      if (live && j < width) {
        if (ALIGNED) weights(k);
#pragma unroll
        for (int e = 0; e < V; ++e) h[k][e] = h[k][e] * inv * w[k][e] + b[k][e];
        row_put<T, V, ALIGNED>(out + base + j, h[k], width - j);
      }
    }
  }
}

// Workgroup b takes rows b, b + gridDim.x, ... (times the rows that share a workgroup) and keeps its parts of dw and db
// in registers; the parts [group][dw, db][width] are joined in their order by join_parts.
template <typename T, int THREADS, bool ALIGNED>
__global__ __launch_bounds__(kGroup<THREADS>) void layer_backward(const T* grad, const T* grad_sum, const T* x,
                                                                  const T* residual, const void* weight, int weight_float,
                                                                  const float* mean, const float* inverse, T* grad_x,
                                                                  float* parts, int64_t rows, int width) {
  constexpr int V = kWide<T>, N = kChunks<T>, SHARE = kGroup<THREADS> / THREADS;
  __shared__ float slots[2][kGroup<THREADS> / 64][2];
  const int t = threadIdx.x % THREADS, sub = threadIdx.x / THREADS;
  float w[N][V], dw[N][V], db[N][V];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int j = (k * THREADS + t) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) w[k][e] = dw[k][e] = db[k][e] = 0.f;
    if (j < width) load_weight<T, V, ALIGNED>(weight, weight_float, j, w[k], width - j);
  }
  // a row as it lies in memory; the next one is requested while this one is worked on (32768 rows of 768 bfloat16 values,
  // of h alone: 75 us without that for 42), but for 1024 threads, whose registers do not hold two
  constexpr bool AHEAD = THREADS < 1024;
  struct Row {
    Words h[N], r[N], g[N], s[N];
    float mu, inv;
    bool live;
  };
  auto request = [&](Row& r, int64_t first) {
    const int64_t row = first + sub, base = row * width;
    const bool more = row + 1 < rows && width >= V;
    r.live = row < rows;
    r.inv = r.live ? inverse[row] : 0.f;
    r.mu = r.live ? mean[row] : 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int j = (k * THREADS + t) * V;
      r.h[k] = r.r[k] = r.g[k] = r.s[k] = Words{0, 0, 0, 0};
      if (r.live && j < width) {
        r.h[k] = row_get<T, V, ALIGNED>(x + base + j, width - j, more);
        if (residual) r.r[k] = row_get<T, V, ALIGNED>(residual + base + j, width - j, more);
        r.g[k] = row_get<T, V, ALIGNED>(grad + base + j, width - j, more);
        if (grad_sum) r.s[k] = row_get<T, V, ALIGNED>(grad_sum + base + j, width - j, more);
      }
    }
  };
  const int64_t begin = (int64_t)blockIdx.x * SHARE, step = (int64_t)gridDim.x * SHARE;
  Row now;
  if (AHEAD) request(now, begin);
  int turn = 0;
  for (int64_t first = begin; first < rows; first += step, turn ^= 1) {
    Row next;
    if (!AHEAD)
      request(now, first);
    else if (first + step < rows)
      request(next, first + step);
    float z[N][V], q[N][V], both[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < N; ++k) {
      // beyond the row's end q and w are zeros: z counts nowhere
      const int left = width - (k * THREADS + t) * V;
      float r[V];
      in_row<T, V, ALIGNED>(now.h[k], z[k], left);
      in_row<T, V, ALIGNED>(now.r[k], r, left);
      in_row<T, V, ALIGNED>(now.g[k], q[k], left);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        z[k][e] = ((z[k][e] + r[e]) - now.mu) * now.inv;
        dw[k][e] += q[k][e] * z[k][e];
        db[k][e] += q[k][e];
        q[k][e] *= w[k][e];
        both[0] += q[k][e];
        both[1] += q[k][e] * z[k][e];
      }
    }
    row_sums<THREADS>(both, slots[turn]);
    const float flat = both[0] / (float)width, along = both[1] / (float)width;
    if (grad_x) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int j = (k * THREADS + t) * V;
        if (now.live && j < width) {
          float s[V];
          in_row<T, V, true>(now.s[k], s, width - j);
#pragma unroll
          for (int e = 0; e < V; ++e) s[e] += now.inv * (q[k][e] - flat - z[k][e] * along);
          row_put<T, V, ALIGNED>(grad_x + (first + sub) * width + j, s, width - j);
        }
      }
    }
    if (AHEAD) now = next;
  }
  if (!parts) return;
  float* to = parts + (int64_t)blockIdx.x * 2 * width;
  if constexpr (SHARE > 1) {   // the rows that share the workgroup are joined in LDS
    __shared__ float joined[SHARE][THREADS * N * V];
#pragma unroll
    for (int which = 0; which < 2; ++which, to += width) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < N; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) joined[sub][(k * V + e) * THREADS + t] = which ? db[k][e] : dw[k][e];
      __syncthreads();
      for (int i = threadIdx.x; i < THREADS * N * V; i += kGroup<THREADS>) {
        const int ke = i / THREADS, j = (ke / V * THREADS + i % THREADS) * V + ke % V;
        float x = 0.f;
#pragma unroll
        for (int s = 0; s < SHARE; ++s) x += joined[s][i];
        if (j < width) to[j] = x;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int j = (k * THREADS + t) * V;
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (j + e < width) to[j + e] = dw[k][e], to[width + j + e] = db[k][e];
    }
  }
}

// The sums over the parts: 64 of the 2 width columns a workgroup, a sixteenth of the parts a wave, eight at a time.
template <typename T>
__global__ __launch_bounds__(1024) void join_parts(const float* parts, int64_t count, int width, void* grad_weight,
                                                   void* grad_bias, int is_float) {
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int j = blockIdx.x * 64 + lane;
  const int64_t each = (count + 15) / 16, from = wave * each, to = from + each < count ? from + each : count;
  float s = 0.f;
  if (j < 2 * width) {
    const int64_t step = 2 * (int64_t)width;
    int64_t i = from;
    for (; i + 8 <= to; i += 8) {
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = parts[(i + u) * step + j];
      s += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
    }
    for (; i < to; ++i) s += parts[i * step + j];
  }
  sums[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && j < 2 * width) {
    s = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) s += sums[w][lane];
    void* to_grad = j < width ? grad_weight : grad_bias;
    const int at = j < width ? j : j - width;
    if (!to_grad) return;
    if (is_float)
      ((float*)to_grad)[at] = s;
    else
      ((T*)to_grad)[at] = (T)s;
  }
}

// Threads of a row: a power of two from 4 on, at most 16 values each.
int threads_of(int64_t width) {
  int threads = 4;
  while (threads * 16 < width) threads *= 2;
  return threads;
}

#define LAYER_THREADS(THREADS_, ...) \
  case THREADS_: { constexpr int THREADS = THREADS_; __VA_ARGS__; break; }
#define LAYER_SHAPE_OF(...)               \
  switch (threads_of(width)) {            \
    LAYER_THREADS(4, __VA_ARGS__)         \
    LAYER_THREADS(8, __VA_ARGS__)         \
    LAYER_THREADS(16, __VA_ARGS__)        \
    LAYER_THREADS(32, __VA_ARGS__)        \
    LAYER_THREADS(64, __VA_ARGS__)        \
    LAYER_THREADS(128, __VA_ARGS__)       \
    LAYER_THREADS(256, __VA_ARGS__)       \
    LAYER_THREADS(512, __VA_ARGS__)       \
    default: { constexpr int THREADS = 1024; __VA_ARGS__; } \
  }
// Runs the statement with THREADS and ALIGNED for rows of `width`; `wide`: 16-byte vectors fit rows and pointers.
#define LAYER_SHAPE(...)                                                     \
  do {                                                                       \
    if (wide) { constexpr bool ALIGNED = true; LAYER_SHAPE_OF(__VA_ARGS__) }  \
    else { constexpr bool ALIGNED = false; LAYER_SHAPE_OF(__VA_ARGS__) }      \
  } while (0)

// The rows in launches of as many as one holds.
template <typename T, int THREADS, bool ALIGNED>
void run_forward(const T* x, const T* residual, const void* weight, const void* bias, int weight_float, T* out, T* summed,
                 float* mean, float* inverse, int64_t rows, int width, float eps, hipStream_t s) {
  constexpr int SHARE = kGroup<THREADS> / THREADS;
  constexpr int64_t EACH = most_groups(kGroup<THREADS>) * SHARE;
  for (int64_t row = 0; row < rows; row += EACH) {
    const int64_t count = std::min(EACH, rows - row), at = row * width;
    const int64_t groups = ceil_div(count, SHARE);
    launch(layer_forward<T, THREADS, ALIGNED>, dim3((unsigned)(ALIGNED ? groups : std::min<int64_t>(groups, 2048))),
           dim3(kGroup<THREADS>), s, x + at,
           residual ? residual + at : nullptr, weight, bias, weight_float, out + at, summed ? summed + at : nullptr,
           mean ? mean + row : nullptr, inverse ? inverse + row : nullptr, count, width, eps);
  }
}

// Workgroups of the backward, each of which keeps sums of dw and db for join_parts: few of them leave rows one after the
// other, many a longer join.  With residual in bfloat16 and float32, us by 256 / 512 / 1024 / 2048 of them: 32768 x 768
// 51 / 40 / 44 / 50 and 76 / 80 / 82 / 88, 262144 x 96 47 / 36 / 41 / 43 and 77 / 80 / 82 / 85, 8192 x 4096 (256 threads a row)
// 67 / 57 / 69 / 94 and 104 / 110 / 120 / 132, 4096 x 8192 (512 threads) 65 / 78 / 106 / 163 and 110 / 117 / 136 / 167,
// 2048 x 16384 (1024 threads) 97 / 127 / 190 / 326 and 148 / 174 / 215 / 313.  So half of these and less would do as well or
// better; more than them costs.
int64_t backward_groups(int64_t rows, int64_t width) {
  const int threads = threads_of(width), share = threads < 256 ? 256 / threads : 1;
  const int64_t groups = threads > 512 ? 256 : threads > 256 ? 512 : 1024;
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

int sdk_add_layer_norm(const void* x, const void* residual, const void* weight, const void* bias, void* out,
                       void* summed, float* mean, float* inverse, int64_t rows, int64_t width, double eps,
                       int32_t dtype, int32_t weight_dtype, sdk_stream_t stream) {
  if (int rc = check(rows, width, dtype, weight_dtype)) return rc;
  SDK_REQUIRE(eps >= 0, "eps must not be negative");
  if (rows == 0) return SDK_OK;
  SDK_REQUIRE(x && weight && out, "x, weight and out must not be NULL");
  hipStream_t s = (hipStream_t)stream;
  SDK_DISPATCH_TOKEN_DTYPE(dtype, {
    const bool wide = width % kWide<T> == 0 && aligned16(x) && aligned16(residual) && aligned16(weight) &&
                      aligned16(bias) && aligned16(out) && aligned16(summed);
    LAYER_SHAPE(run_forward<T, THREADS, ALIGNED>((const T*)x, (const T*)residual, weight, bias, weight_dtype == SDK_F32,
                                                 (T*)out, (T*)summed, mean, inverse, rows, (int)width, (float)eps, s));
  });
  SDK_LAUNCH_CHECK("add_layer_norm");
  return SDK_OK;
}

size_t sdk_add_layer_norm_backward_workspace_bytes(int64_t rows, int64_t width) {
  if (rows < 1 || width < 1 || width > kMostWidth) return 0;
  return (size_t)backward_groups(rows, width) * 2 * width * sizeof(float);
}

int sdk_add_layer_norm_backward(const void* grad, const void* grad_sum, const void* x, const void* residual,
                                const void* weight, const float* mean, const float* inverse, void* grad_x, void* grad_weight,
                                void* grad_bias, void* workspace, size_t workspace_bytes, int64_t rows, int64_t width,
                                int32_t dtype, int32_t weight_dtype, sdk_stream_t stream) {
  if (int rc = check(rows, width, dtype, weight_dtype)) return rc;
  SDK_REQUIRE(weight && (grad_x || grad_weight || grad_bias), "weight and one gradient at least must not be NULL");
  SDK_REQUIRE(rows == 0 || (grad && x && mean && inverse), "grad, x, mean and inverse must not be NULL");
  const bool sums = grad_weight || grad_bias;
  const size_t need = sums ? sdk_add_layer_norm_backward_workspace_bytes(rows, width) : 0;
  if (need && (!workspace || workspace_bytes < need))
    return fail(SDK_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  hipStream_t s = (hipStream_t)stream;
  const int64_t groups = rows ? backward_groups(rows, width) : 0;
  float* parts = sums ? (float*)workspace : nullptr;
  SDK_DISPATCH_TOKEN_DTYPE(dtype, {
    const bool wide = width % kWide<T> == 0 && aligned16(grad) && aligned16(grad_sum) && aligned16(x) &&
                      aligned16(residual) && aligned16(weight) && aligned16(grad_x);
    if (rows)
      LAYER_SHAPE(launch(layer_backward<T, THREADS, ALIGNED>, dim3((unsigned)groups), dim3(kGroup<THREADS>), s,
                         (const T*)grad, (const T*)grad_sum, (const T*)x, (const T*)residual, weight,
                         (int)(weight_dtype == SDK_F32), mean, inverse, (T*)grad_x, parts, rows, (int)width));
    if (sums)
      launch(join_parts<T>, dim3((unsigned)ceil_div(2 * width, 64)), dim3(1024), s, (const float*)parts, groups,
             (int)width, grad_weight, grad_bias, (int)(weight_dtype == SDK_F32));
  });
  SDK_LAUNCH_CHECK("add_layer_norm_backward");
  return SDK_OK;
}

}  // extern "C"
