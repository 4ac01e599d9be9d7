// One AdamW step over many tensors in few launches, moments in 32 bits or in 8.
//
//   m = m b1 + g (1 - b1)      v = v b2 + g g (1 - b2)
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8 bits: 256 consecutive values of a tensor share a scale s, the largest magnitude among them.
//   first moment   code c in -127 .. 127:  m = c |c| / 127^2 s      (steps of 2 / c of the value)
//   second moment  code c in 0 .. 255:     v = (c / 255)^4 s        (steps of 4 / c of the value)
// Squares and fourth powers give small values steps in proportion.  A second moment that is not zero keeps
// code 1 at least: a zero below a first moment would make that parameter jump.
//
// Bound by memory: 28 bytes a value with float32 parameters and moments, 16 with moments in 8 bits: 86 million values in
// 121 tensors take 447 us (5.4 TB/s) and 306 us (4.5 TB/s; the exact divisions and roots are the rest).  All
// arithmetic is float32, each operation rounded by itself in the order above (nothing is contracted), with
// exact division and square root.
#include <algorithm>
#include <cmath>

#include "token_types.hpp"

namespace sdk {
namespace token {
namespace {

constexpr int kTensors = 64;           // of a launch: their table is a kernel argument (4 KB at most)
constexpr int kBlock = 256;            // values that share a scale
constexpr float kSmallest = 0x1p-126f; // a block below it holds zeros: 1 / scale stays finite

struct Settings {
  float keep, b1, one_b1, b2, one_b2, root, eps, rate;
};

struct Tensors32 {
  void* p[kTensors];
  const void* g[kTensors];
  float* m[kTensors];
  float* v[kTensors];
  int64_t n[kTensors];
  unsigned start[kTensors];   // first workgroup of each tensor; beyond the last: more than the grid
};

struct Tensors8 {
  void* p[kTensors];
  const void* g[kTensors];
  signed char* mc[kTensors];
  float* ms[kTensors];
  unsigned char* vc[kTensors];
  float* vs[kTensors];
  int64_t n[kTensors];
  unsigned start[kTensors];
};
static_assert(sizeof(Tensors8) + sizeof(Settings) <= 4096, "kernel arguments are limited to 4 KB");

__device__ __forceinline__ void update(float& p, float g, float& m, float& v, const Settings& s) {
  m = m * s.b1 + g * s.one_b1;
  v = v * s.b2 + (g * g) * s.one_b2;
  const float below = sqrtf(v) * s.root + s.eps;
  p = p * s.keep - (m / below) * s.rate;
}

// The tensor that workgroup blockIdx.x works on: each lane looks at one start.
__device__ __forceinline__ int tensor_of(const unsigned* start) {
  const unsigned long long before = __ballot(start[threadIdx.x & 63] <= blockIdx.x);
  return __builtin_amdgcn_readfirstlane(__popcll(before) - 1);
}

constexpr int kRounds32 = 4;                        // vectors of four values a thread
constexpr int kPerGroup32 = 256 * 4 * kRounds32;

template <typename T>
__global__ __launch_bounds__(256) void adamw32(const Tensors32 t, const Settings s) {
  const int i = tensor_of(t.start);
  T* p = (T*)t.p[i];
  const T* g = (const T*)t.g[i];
  float *m = t.m[i], *v = t.v[i];
  const int64_t n = t.n[i], from = (int64_t)(blockIdx.x - t.start[i]) * kPerGroup32;
  const bool wide = (((uintptr_t)p | (uintptr_t)g) % (4 * sizeof(T)) | ((uintptr_t)m | (uintptr_t)v) % 16) == 0;
  if (wide && from + kPerGroup32 <= n) {
    float fp[kRounds32][4], fg[kRounds32][4], fm[kRounds32][4], fv[kRounds32][4];
#pragma unroll
    for (int r = 0; r < kRounds32; ++r) {
      const int64_t at = from + (r * 256 + threadIdx.x) * 4;
      load_pack<T, 4>(p + at, fp[r]);
      load_pack<T, 4>(g + at, fg[r]);
      load_pack<float, 4>(m + at, fm[r]);
      load_pack<float, 4>(v + at, fv[r]);
    }
#pragma unroll
    for (int r = 0; r < kRounds32; ++r) {
      const int64_t at = from + (r * 256 + threadIdx.x) * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) update(fp[r][e], fg[r][e], fm[r][e], fv[r][e], s);
      store_pack<T, 4>(p + at, fp[r]);
      store_pack<float, 4>(m + at, fm[r]);
      store_pack<float, 4>(v + at, fv[r]);
    }
    return;
  }
  const int64_t to = from + kPerGroup32 < n ? from + kPerGroup32 : n;
  for (int64_t at = from + threadIdx.x; at < to; at += 256) {
    float fp = (float)p[at], fm = m[at], fv = v[at];
    update(fp, (float)g[at], fm, fv, s);
    p[at] = (T)fp;
    m[at] = fm;
    v[at] = fv;
  }
}

__device__ __forceinline__ float avg_value(signed char c, float scale) {
  const float a = (float)c * (1.f / 127.f);
  return (a * fabsf(a)) * scale;
}
__device__ __forceinline__ float sq_value(unsigned char c, float scale) {
  const float a = (float)c * (1.f / 255.f), b = a * a;
  return (b * b) * scale;
}

// scale of a block, and what its values are multiplied with; NaN and infinity stay in the scale
__device__ __forceinline__ float scale_of(float largest, float& inverse) {
  if (largest < kSmallest) {
    inverse = 0.f;
    return 0.f;
  }
  inverse = 1.f / largest;
  return largest;
}

constexpr int kRounds8 = 4;                         // blocks of 256 values a wave
constexpr int kPerGroup8 = 4 * kRounds8 * kBlock;

// One block of 256 values, four consecutive ones a lane, on its way through a step.
template <typename T>
struct Block8 {
  float p[4], g[4], m_scale, v_scale;
  Pack<signed char, 4> cm;
  Pack<unsigned char, 4> cv;

  __device__ __forceinline__ void step(const Settings& s, int left) {   // left: values from this lane's first to the end
    float m[4], v[4], m_most = 0.f, v_most = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // beyond the tensor's end the values are zeros whatever the scale holds
      m[e] = e < left ? avg_value(cm.v[e], m_scale) : 0.f;
      v[e] = e < left ? sq_value(cv.v[e], v_scale) : 0.f;
      update(p[e], g[e], m[e], v[e], s);
      m_most = Largest::of(m_most, fabsf(m[e]));
      v_most = Largest::of(v_most, v[e]);
    }
    float m_inv, v_inv;
    m_scale = scale_of(over_wave<Largest>(m_most), m_inv);
    v_scale = scale_of(over_wave<Largest>(v_most), v_inv);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float c = rintf(sqrtf(fabsf(m[e]) * m_inv) * 127.f);
      cm.v[e] = (signed char)(int)(m[e] < 0.f ? -c : c);
      const float d = rintf(sqrtf(sqrtf(v[e] * v_inv)) * 255.f);
      cv.v[e] = (unsigned char)(int)(v[e] > 0.f && v_inv > 0.f && d < 1.f ? 1.f : d);
    }
  }
};

// A wave takes four blocks, all of them requested before the first is worked on.
template <typename T>
__global__ __launch_bounds__(256) void adamw8(const Tensors8 t, const Settings s) {
  const int i = tensor_of(t.start);
  T* p = (T*)t.p[i];
  const T* g = (const T*)t.g[i];
  signed char* mc = t.mc[i];
  unsigned char* vc = t.vc[i];
  float *ms = t.ms[i], *vs = t.vs[i];
  const int64_t n = t.n[i], from = (int64_t)(blockIdx.x - t.start[i]) * kPerGroup8;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool wide = (((uintptr_t)p | (uintptr_t)g) % (4 * sizeof(T)) | ((uintptr_t)mc | (uintptr_t)vc) % 4) == 0;
  if (wide && from + kPerGroup8 <= n) {
    Block8<T> x[kRounds8];
#pragma unroll
    for (int r = 0; r < kRounds8; ++r) {
      const int64_t first = from + (int64_t)(r * 4 + wave) * kBlock, at = first + lane * 4;
      load_pack<T, 4>(p + at, x[r].p);
      load_pack<T, 4>(g + at, x[r].g);
      x[r].cm = *reinterpret_cast<const Pack<signed char, 4>*>(mc + at);
      x[r].cv = *reinterpret_cast<const Pack<unsigned char, 4>*>(vc + at);
      x[r].m_scale = ms[first / kBlock];
      x[r].v_scale = vs[first / kBlock];
    }
#pragma unroll
    for (int r = 0; r < kRounds8; ++r) {
      const int64_t first = from + (int64_t)(r * 4 + wave) * kBlock, at = first + lane * 4;
      x[r].step(s, 4);
      store_pack<T, 4>(p + at, x[r].p);
      *reinterpret_cast<Pack<signed char, 4>*>(mc + at) = x[r].cm;
      *reinterpret_cast<Pack<unsigned char, 4>*>(vc + at) = x[r].cv;
      if (lane == 0) {
        ms[first / kBlock] = x[r].m_scale;
        vs[first / kBlock] = x[r].v_scale;
      }
    }
    return;
  }
  for (int r = 0; r < kRounds8; ++r) {
    const int64_t first = from + (int64_t)(r * 4 + wave) * kBlock, at = first + lane * 4;
    if (first >= n) break;
    const int left = (int)std::min<int64_t>(4, n - at);
    Block8<T> x;
    x.m_scale = ms[first / kBlock];
    x.v_scale = vs[first / kBlock];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x.p[e] = e < left ? (float)p[at + e] : 0.f;
      x.g[e] = e < left ? (float)g[at + e] : 0.f;
      x.cm.v[e] = e < left ? mc[at + e] : (signed char)0;
      x.cv.v[e] = e < left ? vc[at + e] : (unsigned char)0;
    }
    x.step(s, left);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) {
        p[at + e] = (T)x.p[e];
        mc[at + e] = x.cm.v[e];
        vc[at + e] = x.cv.v[e];
      }
    if (lane == 0) {
      ms[first / kBlock] = x.m_scale;
      vs[first / kBlock] = x.v_scale;
    }
  }
}

// The values that codes stand for, 16 a thread (one scale: kBlock is a multiple of 16).
template <typename T>
__global__ __launch_bounds__(256) void moment_values(const unsigned char* codes, const float* scales, T* out,
                                                     int64_t n, int second, int wide) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 16;
  if (at >= n) return;
  const float scale = scales[at / kBlock];
  if (wide && at + 16 <= n) {
    const Pack<unsigned char, 16> c = *reinterpret_cast<const Pack<unsigned char, 16>*>(codes + at);
#pragma unroll
    for (int k = 0; k < 16; k += kWide<T>) {
      float f[kWide<T>];
#pragma unroll
      for (int e = 0; e < kWide<T>; ++e)
        f[e] = second ? sq_value(c.v[k + e], scale) : avg_value((signed char)c.v[k + e], scale);
      store_pack<T, kWide<T>>(out + at + k, f);
    }
  } else {
    for (int e = 0; e < 16 && at + e < n; ++e) {
      const unsigned char c = codes[at + e];
      out[at + e] = (T)(second ? sq_value(c, scale) : avg_value((signed char)c, scale));
    }
  }
}

Settings settings_of(double lr, double b1, double b2, double eps, double weight_decay, int64_t step) {
  Settings s;
  s.keep = (float)(1 - lr * weight_decay);
  s.b1 = (float)b1;
  s.one_b1 = (float)(1 - b1);
  s.b2 = (float)b2;
  s.one_b2 = (float)(1 - b2);
  s.root = (float)(1 / std::sqrt(1 - std::pow(b2, (double)step)));
  s.eps = (float)eps;
  s.rate = (float)(lr / (1 - std::pow(b1, (double)step)));
  return s;
}

int check(int64_t count, double lr, double b1, double b2, double eps, double weight_decay, int64_t step, int dtype) {
  SDK_REQUIRE(count >= 0, "count = %lld must not be negative", (long long)count);
  SDK_REQUIRE(step >= 1, "step = %lld must be 1 or more", (long long)step);
  SDK_REQUIRE(lr >= 0 && eps >= 0 && weight_decay >= 0, "lr, eps and weight_decay must not be negative");
  SDK_REQUIRE(b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1, "betas must be in [0, 1)");
  SDK_REQUIRE(known(dtype), "unknown dtype %d (float32, bfloat16 and float16 only)", dtype);
  return SDK_OK;
}

// Deals the tensors to launches of at most kTensors tensors and as many workgroups as one holds.
template <typename Table, typename Put, typename Run>
int deal(int64_t count, const int64_t* sizes, int64_t per_group, Put put, Run run) {
  Table t;
  int used = 0;
  int64_t groups = 0;
  auto flush = [&] {
    for (int k = used; k < kTensors; ++k) t.start[k] = 0xffffffffu;
    const int rc = run(t, (unsigned)groups);
    used = 0;
    groups = 0;
    return rc;
  };
  for (int64_t i = 0; i < count; ++i) {
    if (sizes[i] == 0) continue;
    const int64_t mine = ceil_div(sizes[i], per_group);
    SDK_REQUIRE(mine <= most_groups(256), "tensor %lld of %lld values is too large", (long long)i,
                (long long)sizes[i]);
    if (used == kTensors || groups + mine > most_groups(256))
      if (int rc = flush()) return rc;
    put(t, used, i);
    t.n[used] = sizes[i];
    t.start[used++] = (unsigned)groups;
    groups += mine;
  }
  return used ? flush() : SDK_OK;
}

}  // namespace
}  // namespace token
}  // namespace sdk

using namespace sdk;
using namespace sdk::token;

extern "C" {

int sdk_adamw_step(void* const* params, const void* const* grads, float* const* avgs, float* const* sqs,
                   const int64_t* sizes, int64_t count, double lr, double beta1, double beta2, double eps,
                   double weight_decay, int64_t step, int32_t dtype, sdk_stream_t stream) {
  if (int rc = check(count, lr, beta1, beta2, eps, weight_decay, step, dtype)) return rc;
  SDK_REQUIRE(count == 0 || (params && grads && avgs && sqs && sizes), "a list of tensors is NULL");
  for (int64_t i = 0; i < count; ++i)
    SDK_REQUIRE(sizes[i] == 0 || (sizes[i] > 0 && params[i] && grads[i] && avgs[i] && sqs[i]),
                "tensor %lld: NULL pointer or negative size", (long long)i);
  const Settings s = settings_of(lr, beta1, beta2, eps, weight_decay, step);
  return deal<Tensors32>(
      count, sizes, kPerGroup32,
      [&](Tensors32& t, int k, int64_t i) {
        t.p[k] = params[i];
        t.g[k] = grads[i];
        t.m[k] = avgs[i];
        t.v[k] = sqs[i];
      },
      [&](const Tensors32& t, unsigned groups) -> int {
        SDK_DISPATCH_TOKEN_DTYPE(dtype, launch(adamw32<T>, dim3(groups), dim3(256), (hipStream_t)stream, t, s));
        SDK_LAUNCH_CHECK("adamw_step");
        return SDK_OK;
      });
}

int sdk_adamw_step_8bit(void* const* params, const void* const* grads, int8_t* const* avg_codes,
                        float* const* avg_scales, uint8_t* const* sq_codes, float* const* sq_scales,
                        const int64_t* sizes, int64_t count, double lr, double beta1, double beta2, double eps,
                        double weight_decay, int64_t step, int32_t dtype, sdk_stream_t stream) {
  if (int rc = check(count, lr, beta1, beta2, eps, weight_decay, step, dtype)) return rc;
  SDK_REQUIRE(count == 0 || (params && grads && avg_codes && avg_scales && sq_codes && sq_scales && sizes),
              "a list of tensors is NULL");
  for (int64_t i = 0; i < count; ++i)
    SDK_REQUIRE(sizes[i] == 0 || (sizes[i] > 0 && params[i] && grads[i] && avg_codes[i] && avg_scales[i] &&
                                  sq_codes[i] && sq_scales[i]),
                "tensor %lld: NULL pointer or negative size", (long long)i);
  const Settings s = settings_of(lr, beta1, beta2, eps, weight_decay, step);
  return deal<Tensors8>(
      count, sizes, kPerGroup8,
      [&](Tensors8& t, int k, int64_t i) {
        t.p[k] = params[i];
        t.g[k] = grads[i];
        t.mc[k] = (signed char*)avg_codes[i];
        t.ms[k] = avg_scales[i];
        t.vc[k] = sq_codes[i];
        t.vs[k] = sq_scales[i];
      },
      [&](const Tensors8& t, unsigned groups) -> int {
        SDK_DISPATCH_TOKEN_DTYPE(dtype, launch(adamw8<T>, dim3(groups), dim3(256), (hipStream_t)stream, t, s));
        SDK_LAUNCH_CHECK("adamw_step_8bit");
        return SDK_OK;
      });
}

int sdk_adamw_moment_values(const void* codes, const float* scales, void* out, int64_t size, int32_t second,
                            int32_t dtype, sdk_stream_t stream) {
  SDK_REQUIRE(size >= 0 && size < (int64_t)1 << 40, "size = %lld", (long long)size);
  SDK_REQUIRE(known(dtype), "unknown dtype %d (float32, bfloat16 and float16 only)", dtype);
  if (size == 0) return SDK_OK;
  SDK_REQUIRE(codes && scales && out, "codes, scales and out must not be NULL");
  const int wide = ((uintptr_t)codes & 15) == 0 && ((uintptr_t)out & 15) == 0;
  constexpr int64_t EACH = most_groups(256) * 4096;   // of a launch: whole blocks
  SDK_DISPATCH_TOKEN_DTYPE(dtype, for (int64_t from = 0; from < size; from += EACH) {
    const int64_t count = std::min(EACH, size - from);
    launch(moment_values<T>, dim3((unsigned)ceil_div(count, 4096)), dim3(256), (hipStream_t)stream,
           (const unsigned char*)codes + from, scales + from / kBlock, (T*)out + from, count, (int)(second != 0), wide);
  });
  SDK_LAUNCH_CHECK("adamw_moment_values");
  return SDK_OK;
}

}  // extern "C"
