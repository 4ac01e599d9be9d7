// Element types of the token operators (float32, bfloat16, float16): conversion to and from float,
// 16-byte vectors, sums and maxima over a workgroup.
#pragma once
#include <hip/hip_runtime.h>

#include "sdk_host.hpp"

namespace sdk {
namespace token {

using bf16 = __bf16;
using f16 = _Float16;

// A vector of E elements of T that is loaded and stored as one (E * sizeof(T) = 16, or one element).
template <typename T, int E>
struct alignas(sizeof(T) * E) Pack {
  T v[E];
};

template <typename T>
constexpr int kWide = 16 / (int)sizeof(T);   // elements of a 16-byte vector

template <typename T, int E>
__device__ __forceinline__ void load_pack(const T* p, float (&f)[E]) {
  const Pack<T, E> x = *reinterpret_cast<const Pack<T, E>*>(p);
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = (float)x.v[e];
}

template <typename T, int E>
__device__ __forceinline__ void store_pack(T* p, const float (&f)[E]) {
  Pack<T, E> x;
#pragma unroll
  for (int e = 0; e < E; ++e) x.v[e] = (T)f[e];
  *reinterpret_cast<Pack<T, E>*>(p) = x;
}

// E elements at any address of which `left` are there (the others read as zeros and are not written): rows whose width or
// address fits no vector.
template <typename T, int E>
__device__ __forceinline__ void load_part(const T* p, float (&f)[E], int left) {
  if (left >= E) {
    Pack<T, E> x;
    __builtin_memcpy(&x, p, sizeof(x));
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = (float)x.v[e];
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = e < left ? (float)p[e] : 0.f;
  }
}

template <typename T, int E>
__device__ __forceinline__ void store_part(T* p, const float (&f)[E], int left) {
  if (left >= E) {
    Pack<T, E> x;
#pragma unroll
    for (int e = 0; e < E; ++e) x.v[e] = (T)f[e];
    __builtin_memcpy(p, &x, sizeof(x));
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < left) p[e] = (T)f[e];
  }
}

struct Add {
  __device__ static float of(float a, float b) { return a + b; }
};
// NaN stays: a row or block that holds one has no largest value.
struct Largest {
  __device__ static float of(float a, float b) { return a != a ? a : (b > a || b != b ? b : a); }
};

template <typename Op>
__device__ __forceinline__ float over_wave(float x) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x = Op::of(x, __shfl_xor(x, d));
  return x;
}

// Over the THREADS consecutive threads of a group that starts at a multiple of THREADS; every thread
// gets the result.  `slots`: one float a wave of the workgroup; used again only after a barrier of
// this function's own, so that calls may follow each other.
template <typename Op, int THREADS>
__device__ __forceinline__ float over_group(float x, float* slots) {
  x = over_wave<Op>(x);
  if constexpr (THREADS > 64) {
    const int wave = threadIdx.x >> 6, first = (threadIdx.x / THREADS) * (THREADS / 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) slots[wave] = x;
    __syncthreads();
    x = slots[first];
#pragma unroll
    for (int i = 1; i < THREADS / 64; ++i) x = Op::of(x, slots[first + i]);
  }
  return x;
}

// Workgroups of `threads` that one launch holds along x: fewer than 2^32 threads.  A larger grid is cut without an error.
constexpr int64_t most_groups(int threads) { return (((int64_t)1 << 32) - 1) / threads; }

inline bool known(int dtype) { return dtype == SDK_F32 || dtype == SDK_BF16 || dtype == SDK_F16; }
inline size_t bytes_of(int dtype) { return dtype == SDK_F32 ? 4 : 2; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace token
}  // namespace sdk

// Runs `CALL` with `T` bound to the element type of `dtype`.
#define SDK_DISPATCH_TOKEN_DTYPE(dtype, ...)                              \
  do {                                                                     \
    if ((dtype) == SDK_F32) { using T = float; __VA_ARGS__; }                     \
    else if ((dtype) == SDK_BF16) { using T = sdk::token::bf16; __VA_ARGS__; }    \
    else { using T = sdk::token::f16; __VA_ARGS__; }                              \
  } while (0)
