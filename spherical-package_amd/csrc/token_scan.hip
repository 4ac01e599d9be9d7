// Gated linear recurrence along the tokens of sequences, with gradients, and its step for single tokens.
//
//   f_t = sigmoid(gate_t),  u_t = 1 - f_t        h_t = f_t h_{t-1} + u_t x_t = h_{t-1} + u_t (x_t - h_{t-1})
//   e_t = g_t + c_t,  c_{t-1} = f_t e_t          (g: the gradient of h_t; c behind the last token: that of the last state)
//   dx_t = u_t e_t    dgate_t = e_t (h_{t-1} - x_t) f_t u_t    gradient of the first state = c in front of the first token
//
// Each channel by itself.  A span of tokens acts on the state before it as h -> A h + H, and spans join: (A, H) then
// (A', H') is (A A', A' H + H').  So a workgroup takes 64 channels in 16 bits (32 in float32: 128 bytes of a token either
// way) and a tile of 128 tokens, of which each thread walks four in order; the threads' (A, H) are joined over the tile,
// and each walks its four again from the state in front of them.  The tile's values stay in registers meanwhile.
// Sequences with too few channels for the GPU are cut into segments: a first launch forms the (A, H) of each, the
// second begins each segment with the state that the ones before it leave.
//
// Bound by memory: three values read or written a token and channel forward, six backward (the gradients read h as
// it was rounded to the tensors' type); segments read two of them twice.  The state, its gradient, (A, H) and the gates
// are float32.  u is formed as sigmoid(-gate) and weighs the distance x - h: 1 - f of a rounded f near one would be
// off by a part of all that a long memory sums up.
#include <algorithm>

#include "token_types.hpp"

namespace sdk {
namespace token {
namespace {

constexpr int kThreads = 256;
constexpr int kRows = 4;                       // tokens of a tile that a thread walks

struct Scan {
  const void *x, *gate;
  const float* state;          // [batch][width] dense, or NULL
  const int32_t* lengths;      // [batch], or NULL
  void* out;                   // [batch][tokens][width] dense
  float* last;                 // [batch][width]
  const void* grad;            // backward: of out (may be NULL), strides below
  const float* grad_last;      // may be NULL
  void *grad_x, *grad_gate;    // [batch][tokens][width] dense, may be NULL
  float* grad_state;           // may be NULL
  float* sums;                 // [2][batch of the launch][segments][width]: A, H of the segments
  int64_t x_strides[2], gate_strides[2], grad_strides[2];   // batch, token
  int64_t tokens, segment;     // segment: tokens of one, a multiple of the tile unless there is one alone
  int width, segments, blocks; // blocks: of channels
  int batches;                 // of this launch
  int64_t first;               // its first batch element
  int reverse;
};

// f = sigmoid(g), u = 1 - f, both to a few units of their last place: e = exp(-|g|) by the power of two, whose argument
// is carried in two parts.
__device__ __forceinline__ void gates(float g, float& f, float& u) {
  constexpr float kLog2e = 1.44269502e+00f, kLog2eRest = 1.92596303e-08f, kLn2 = 6.93147182e-01f;
  const float m = fminf(fabsf(g), 128.f), t = m * kLog2e;
  const float rest = fmaf(m, kLog2eRest, fmaf(m, kLog2e, -t));
  float e = __builtin_amdgcn_exp2f(-t);
  e = fmaf(e * rest, -kLn2, e);
  const float d = 1.f + e;
  float r = __builtin_amdgcn_rcpf(d);
  r = fmaf(fmaf(-d, r, 1.f), r, r);
  f = g >= 0.f ? r : e * r;
  u = g >= 0.f ? e * r : r;
  if (g != g) f = u = g;
}

// h -> a h + b, for each of V channels
template <int V>
struct Span {
  float a[V], b[V];
};

template <int V>
__device__ __forceinline__ void unit(Span<V>& s) {
#pragma unroll
  for (int e = 0; e < V; ++e) s.a[e] = 1.f, s.b[e] = 0.f;
}

// Joins the spans of the workgroup's threads in the order of their time lanes (thread = time lane * LANES + channel lane):
// on return `in` is the state in front of this thread's span, and `carry`, the state in front of all of them, the one
// behind.  slots: [2][4 waves][LANES * V] floats, free to be written (the caller takes two in turn).
template <int V, int LANES>
__device__ __forceinline__ void over_tile(Span<V> s, float (&carry)[V], float (&in)[V], float* slots) {
  constexpr int C = LANES * V;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (threadIdx.x % LANES) * V;
#pragma unroll
  for (int d = LANES; d < 64; d *= 2) {
    const bool joins = lane >= d;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float a = __shfl_up(s.a[e], d), b = __shfl_up(s.b[e], d);
      if (joins) s.b[e] = fmaf(s.a[e], b, s.b[e]), s.a[e] *= a;
    }
  }
  if (lane >= 64 - LANES) {
#pragma unroll
    for (int e = 0; e < V; ++e) slots[wave * C + c + e] = s.a[e], slots[(4 + wave) * C + c + e] = s.b[e];
  }
  // the span of the threads before this one in the wave
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float a = __shfl_up(s.a[e], LANES), b = __shfl_up(s.b[e], LANES);
    s.a[e] = lane >= LANES ? a : 1.f;
    s.b[e] = lane >= LANES ? b : 0.f;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float h = carry[e];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w == wave) in[e] = fmaf(s.a[e], h, s.b[e]);
      h = fmaf(slots[w * C + c + e], h, slots[(4 + w) * C + c + e]);
    }
    carry[e] = h;
  }
}

// Where a workgroup works, and how tokens are counted: `at` counts them in the order of the recurrence.
template <typename T, int LANES>
struct Place {
  int64_t b, from, to, first_token, after_last;   // batch element, tokens of the segment, those that count (by `at`)
  int segment, channel, left, time;
  __device__ __forceinline__ Place(const Scan& p) {
    unsigned id = blockIdx.x;
    const int block = (int)(id % (unsigned)p.blocks);
    id /= (unsigned)p.blocks;
    segment = (int)(id % (unsigned)p.segments);
    b = id / (unsigned)p.segments;
    from = segment * p.segment;
    to = from + p.segment < p.tokens ? from + p.segment : p.tokens;
    channel = (block * LANES + (int)(threadIdx.x % LANES)) * kWide<T>;
    left = p.width - channel;
    time = threadIdx.x / LANES;
    int64_t n = p.tokens;
    if (p.lengths) n = p.lengths[p.first + b], n = n < 0 ? 0 : n > p.tokens ? p.tokens : n;
    first_token = p.reverse ? p.tokens - n : 0;
    after_last = p.reverse ? p.tokens : n;
  }
  __device__ __forceinline__ int64_t row(const Scan& p, int64_t at) const { return p.reverse ? p.tokens - 1 - at : at; }
  __device__ __forceinline__ bool counts(int64_t at) const { return left > 0 && at >= first_token && at < after_last; }
};

// The state in front of segment `at.segment` in the order that its sums go (backward: from the last segment down): the
// segments' spans are dealt to the time lanes.
template <typename T, int LANES, bool BACKWARD>
__device__ __forceinline__ void state_before(const Scan& p, const Place<T, LANES>& at, float (&carry)[kWide<T>], float* slots) {
  constexpr int V = kWide<T>, TIMES = kThreads / LANES;
  const int before = BACKWARD ? p.segments - 1 - at.segment : at.segment;
  if (before == 0) return;
  const int each = (before + TIMES - 1) / TIMES;
  Span<V> s;
  unit(s);
  const float* a = p.sums + ((int64_t)at.b * p.segments) * p.width + at.channel;
  const float* b = a + (int64_t)p.batches * p.segments * p.width;
  for (int i = at.time * each; i < (at.time + 1) * each && i < before; ++i) {
    const int64_t to = (int64_t)(BACKWARD ? p.segments - 1 - i : i) * p.width;
    float fa[V], fb[V];
    load_part<float, V>(a + to, fa, at.left);
    load_part<float, V>(b + to, fb, at.left);
#pragma unroll
    for (int e = 0; e < V; ++e) s.b[e] = fmaf(fa[e], s.b[e], fb[e]), s.a[e] *= fa[e];
  }
  float in[V];
  over_tile<V, LANES>(s, carry, in, slots);
  __syncthreads();
}

template <int V>
__device__ __forceinline__ void load_state(const float* p, int64_t at, float (&f)[V], int left) {
#pragma unroll
  for (int e = 0; e < V; ++e) f[e] = 0.f;
  if (p && left > 0) load_part<float, V>(p + at, f, left);
}

// The span of each segment: a time lane walks its part of the segment, without waiting for others until the end.
template <typename T, int LANES, bool ALIGNED, bool BACKWARD>
__global__ __launch_bounds__(kThreads) void scan_spans(const Scan p) {
  constexpr int V = kWide<T>, TIMES = kThreads / LANES;
  __shared__ float slots[8 * LANES * V];
  const Place<T, LANES> place(p);
  const void* source = BACKWARD ? p.grad : p.x;
  const int64_t(&strides)[2] = BACKWARD ? p.grad_strides : p.x_strides;
  const T* x = source ? (const T*)source + (p.first + place.b) * strides[0] + place.channel : nullptr;
  const T* gate = (const T*)p.gate + (p.first + place.b) * p.gate_strides[0] + place.channel;
  const int64_t each = p.segment / TIMES;   // a multiple of kRows
  Span<V> s;
  unit(s);
  for (int64_t i = 0; i < each; i += kRows) {
    const int64_t begin = place.time * each + i;
    float fx[kRows][V], fg[kRows][V];
    bool counts[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int64_t at = BACKWARD ? place.from + p.segment - 1 - begin - r : place.from + begin + r;
      counts[r] = at < place.to && place.counts(at);
#pragma unroll
      for (int e = 0; e < V; ++e) fx[r][e] = 0.f;
      if (counts[r]) {
        const int64_t row = place.row(p, at);
        if (x) get<T, V, ALIGNED>(x + row * strides[1], fx[r], place.left);
        get<T, V, ALIGNED>(gate + row * p.gate_strides[1], fg[r], place.left);
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (counts[r]) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float f, u;
          gates(fg[r][e], f, u);
          if constexpr (BACKWARD) {
            const float c = fx[r][e] + s.b[e];
            s.b[e] = fmaf(-u, c, c);
          } else {
            s.b[e] = fmaf(u, fx[r][e] - s.b[e], s.b[e]);
          }
          s.a[e] = fmaf(-u, s.a[e], s.a[e]);
        }
      }
  }
  float product[V], carry[V];
#pragma unroll
  for (int e = 0; e < V; ++e) carry[e] = 0.f;
  over_tile<V, LANES>(s, carry, product, slots);
#pragma unroll
  for (int e = 0; e < V; ++e) {   // the slots hold the waves' spans
    product[e] = 1.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) product[e] *= slots[w * LANES * V + (threadIdx.x % LANES) * V + e];
  }
  if (place.left <= 0 || place.time != 0) return;
  float* a = p.sums + ((int64_t)place.b * p.segments + place.segment) * p.width + place.channel;
  store_part<float, V>(a, product, place.left);
  store_part<float, V>(a + (int64_t)p.batches * p.segments * p.width, carry, place.left);
}

template <typename T, int LANES, bool ALIGNED>
__global__ __launch_bounds__(kThreads) void scan_forward(const Scan p) {
  constexpr int V = kWide<T>, TILE = kThreads / LANES * kRows;
  __shared__ float slots[2][8 * LANES * V];
  const Place<T, LANES> place(p);
  const int64_t b = p.first + place.b, lane_state = b * p.width + place.channel;
  const T* x = (const T*)p.x + b * p.x_strides[0] + place.channel;
  const T* gate = (const T*)p.gate + b * p.gate_strides[0] + place.channel;
  T* out = (T*)p.out + b * p.tokens * p.width + place.channel;
  float carry[V];
  load_state<V>(p.state, lane_state, carry, place.left);
  state_before<T, LANES, false>(p, place, carry, slots[1]);
  int turn = 0;
  for (int64_t tile = place.from; tile < place.to; tile += TILE, turn ^= 1) {
    const int64_t at = tile + place.time * kRows;
    float fx[kRows][V], fg[kRows][V], in[V];
    bool counts[kRows];
    Span<V> s;
    unit(s);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      counts[r] = at + r < place.to && place.counts(at + r);
      if (counts[r]) {
        const int64_t row = place.row(p, at + r);
        get<T, V, ALIGNED>(x + row * p.x_strides[1], fx[r], place.left);
        get<T, V, ALIGNED>(gate + row * p.gate_strides[1], fg[r], place.left);
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (counts[r]) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float f, u;
          gates(fg[r][e], f, u);
          fg[r][e] = u;
          s.b[e] = fmaf(u, fx[r][e] - s.b[e], s.b[e]);
          s.a[e] = fmaf(-u, s.a[e], s.a[e]);
        }
      }
    over_tile<V, LANES>(s, carry, in, slots[turn]);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (at + r >= place.to || place.left <= 0) continue;
      float h[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        h[e] = 0.f;
        if (counts[r]) h[e] = in[e] = fmaf(fg[r][e], fx[r][e] - in[e], in[e]);
      }
      put<T, V, ALIGNED>(out + place.row(p, at + r) * p.width, h, place.left);
    }
  }
  if (place.left > 0 && place.time == 0 && place.segment == p.segments - 1)
    store_part<float, V>(p.last + lane_state, carry, place.left);
}

// The same from the last token down.  Time lane 0 has the tile's last tokens.
template <typename T, int LANES, bool ALIGNED>
__global__ __launch_bounds__(kThreads) void scan_backward(const Scan p) {
  constexpr int V = kWide<T>, TILE = kThreads / LANES * kRows;
  __shared__ float slots[2][8 * LANES * V];
  const Place<T, LANES> place(p);
  const int64_t b = p.first + place.b, lane_state = b * p.width + place.channel;
  const T* x = (const T*)p.x + b * p.x_strides[0] + place.channel;
  const T* gate = (const T*)p.gate + b * p.gate_strides[0] + place.channel;
  const T* grad = p.grad ? (const T*)p.grad + b * p.grad_strides[0] + place.channel : nullptr;
  const T* h = (const T*)p.out + b * p.tokens * p.width + place.channel;
  T* grad_x = p.grad_x ? (T*)p.grad_x + b * p.tokens * p.width + place.channel : nullptr;
  T* grad_gate = p.grad_gate ? (T*)p.grad_gate + b * p.tokens * p.width + place.channel : nullptr;
  float carry[V];
  load_state<V>(p.grad_last, lane_state, carry, place.left);
  state_before<T, LANES, true>(p, place, carry, slots[1]);
  const int64_t tiles = (place.to - place.from + TILE - 1) / TILE;
  int turn = 0;
  for (int64_t tile = tiles - 1; tile >= 0; --tile, turn ^= 1) {
    // row r of the thread is token at - r
    const int64_t at = place.from + (tile + 1) * TILE - 1 - place.time * kRows;
    float fg[kRows][V], gg[kRows][V], fx[kRows][V], fh[kRows][V], in[V];
    bool counts[kRows];
    Span<V> s;
    unit(s);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      counts[r] = at - r < place.to && place.counts(at - r);
#pragma unroll
      for (int e = 0; e < V; ++e) gg[r][e] = 0.f;
      if (counts[r]) {
        const int64_t row = place.row(p, at - r);
        get<T, V, ALIGNED>(gate + row * p.gate_strides[1], fg[r], place.left);
        if (grad) get<T, V, ALIGNED>(grad + row * p.grad_strides[1], gg[r], place.left);
        get<T, V, ALIGNED>(x + row * p.x_strides[1], fx[r], place.left);
        if (at - r > place.first_token)
          get<T, V, ALIGNED>(h + place.row(p, at - r - 1) * p.width, fh[r], place.left);
        else
          load_state<V>(p.state, lane_state, fh[r], place.left);
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      if (counts[r]) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float f, u;
          gates(fg[r][e], f, u);
          const float c = gg[r][e] + s.b[e];
          s.b[e] = fmaf(-u, c, c);
          s.a[e] = fmaf(-u, s.a[e], s.a[e]);
        }
      }
    over_tile<V, LANES>(s, carry, in, slots[turn]);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (at - r >= place.to || place.left <= 0) continue;
      float dx[V], dg[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        dx[e] = dg[e] = 0.f;
        if (counts[r]) {
          float f, u;
          gates(fg[r][e], f, u);
          const float c = gg[r][e] + in[e];
          dx[e] = c * u;
          dg[e] = c * (fh[r][e] - fx[r][e]) * (f * u);
          in[e] = fmaf(-u, c, c);
        }
      }
      const int64_t row = place.row(p, at - r) * p.width;
      if (grad_x) put<T, V, ALIGNED>(grad_x + row, dx, place.left);
      if (grad_gate) put<T, V, ALIGNED>(grad_gate + row, dg, place.left);
    }
  }
  if (place.left > 0 && place.time == 0 && place.segment == 0 && p.grad_state)
    store_part<float, V>(p.grad_state + lane_state, carry, place.left);
}

// No tokens: the state, or its gradient, passes through.
__global__ __launch_bounds__(256) void pass_state(const float* from, float* to, int64_t size) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += (int64_t)gridDim.x * 256)
    to[i] = from ? from[i] : 0.f;
}

// One token of each sequence: 16 bytes of channels a thread, the state updated in place.
template <typename T, bool ALIGNED>
__global__ __launch_bounds__(256) void scan_step(const T* x, int64_t x_stride, const T* gate, int64_t gate_stride,
                                                 float* state, int64_t state_stride, T* out, int64_t batch, int width,
                                                 int blocks) {
  constexpr int V = kWide<T>;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x, b = id / blocks;
  if (b >= batch) return;
  const int c = (int)(id - b * blocks) * V, left = width - c;
  float fx[V], fg[V], h[V];
  get<T, V, ALIGNED>(x + b * x_stride + c, fx, left);
  get<T, V, ALIGNED>(gate + b * gate_stride + c, fg, left);
  load_part<float, V>(state + b * state_stride + c, h, left);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float f, u;
    gates(fg[e], f, u);
    h[e] = fmaf(u, fx[e] - h[e], h[e]);
  }
  store_part<float, V>(state + b * state_stride + c, h, left);
  put<T, V, ALIGNED>(out + b * width + c, h, left);
}

// Workgroups that fill the GPU: four a CU.
constexpr int64_t kFill = 1024;

// Channel lanes of a workgroup: the fewest of 2 and 8 that take the width.
int lanes_of(int64_t width, int wide) { return width <= 2 * wide ? 2 : 8; }

// Tokens of a segment: all, or as many tiles as leave four workgroups a CU.
int64_t segment_of(int64_t batch, int64_t tokens, int64_t width, int dtype) {
  const int wide = dtype == SDK_F32 ? 4 : 8, lanes = lanes_of(width, wide), tile = kThreads / lanes * kRows;
  const int64_t groups = batch * ceil_div(width, lanes * wide);
  if (groups >= kFill || tokens <= tile) return tokens;
  const int64_t segments = std::min(ceil_div(kFill, groups), ceil_div(tokens, tile));
  return std::min(tokens, ceil_div(ceil_div(tokens, segments), tile) * tile);
}

int check(const sdk_gated_scan* a) {
  SDK_REQUIRE(a, "the argument block must not be NULL");
  SDK_REQUIRE(known(a->dtype), "unknown dtype %d (float32, bfloat16 and float16 only)", a->dtype);
  SDK_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->width >= 0, "sizes must not be negative");
  SDK_REQUIRE(a->batch < (int64_t)1 << 31 && a->tokens < (int64_t)1 << 31 && a->width <= (int64_t)1 << 20,
              "batch %lld and tokens %lld must be below 2^31, width %lld at most 2^20", (long long)a->batch,
              (long long)a->tokens, (long long)a->width);
  return SDK_OK;
}

// The launch's arguments; batch elements go in launches of as many workgroups as one holds.
template <typename Run>
void in_launches(const sdk_gated_scan* a, Scan p, int lanes, int wide, Run run) {
  p.blocks = (int)ceil_div(p.width, lanes * wide);
  p.segments = (int)ceil_div(p.tokens, p.segment);
  const int64_t each = most_groups(kThreads) / ((int64_t)p.blocks * p.segments);
  for (p.first = 0; p.first < a->batch; p.first += each) {
    p.batches = (int)std::min(each, a->batch - p.first);
    run(p, dim3((unsigned)((int64_t)p.batches * p.blocks * p.segments)));
  }
}

Scan on_device(const sdk_gated_scan* a, void* workspace) {
  Scan p = {};
  p.x = a->x, p.gate = a->gate, p.state = a->state, p.lengths = a->lengths, p.out = a->output, p.last = a->last;
  p.grad = a->grad_output, p.grad_last = a->grad_last, p.grad_x = a->grad_x, p.grad_gate = a->grad_gate;
  p.grad_state = a->grad_state, p.sums = (float*)workspace;
  for (int i = 0; i < 2; ++i)
    p.x_strides[i] = a->x_strides[i], p.gate_strides[i] = a->gate_strides[i],
    p.grad_strides[i] = a->grad_output_strides[i];
  p.tokens = a->tokens, p.width = (int)a->width, p.reverse = a->reverse != 0;
  p.segment = segment_of(a->batch, a->tokens, a->width, a->dtype);
  return p;
}

template <typename T>
bool fits(const void* p, const int64_t (&strides)[2]) {
  return aligned16(p) && strides[0] % kWide<T> == 0 && strides[1] % kWide<T> == 0;
}

// Runs the statement with LANES and ALIGNED.
#define SCAN_SHAPE(...)                                                       \
  do {                                                                        \
    if (lanes == 2) {                                                         \
      constexpr int LANES = 2;                                                \
      if (wide) { constexpr bool ALIGNED = true; __VA_ARGS__; }               \
      else { constexpr bool ALIGNED = false; __VA_ARGS__; }                   \
    } else {                                                                  \
      constexpr int LANES = 8;                                                \
      if (wide) { constexpr bool ALIGNED = true; __VA_ARGS__; }               \
      else { constexpr bool ALIGNED = false; __VA_ARGS__; }                   \
    }                                                                         \
  } while (0)

int check_workspace(const sdk_gated_scan* a, const void* workspace, size_t bytes) {
  const size_t need = sdk_gated_scan_workspace_bytes(a);
  if (need && (!workspace || bytes < need))
    return fail(SDK_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", bytes, need);
  return SDK_OK;
}

}  // namespace
}  // namespace token
}  // namespace sdk

using namespace sdk;
using namespace sdk::token;

extern "C" {

size_t sdk_gated_scan_workspace_bytes(const sdk_gated_scan* a) {
  if (check(a) != SDK_OK || !a->batch || !a->tokens || !a->width) return 0;
  const int64_t segment = segment_of(a->batch, a->tokens, a->width, a->dtype);
  const int64_t segments = ceil_div(a->tokens, segment);
  return segments == 1 ? 0 : (size_t)(2 * a->batch * segments * a->width * (int64_t)sizeof(float));
}

int sdk_gated_scan_forward(const sdk_gated_scan* a, void* workspace, size_t workspace_bytes, sdk_stream_t stream) {
  if (int rc = check(a)) return rc;
  if (!a->batch || !a->width) return SDK_OK;
  if (!a->tokens) {
    SDK_REQUIRE(a->last, "last must not be NULL");
    launch(pass_state, dim3(64), dim3(256), (hipStream_t)stream, a->state, a->last, a->batch * a->width);
    SDK_LAUNCH_CHECK("gated_scan_forward");
    return SDK_OK;
  }
  SDK_REQUIRE(a->x && a->gate && a->output && a->last, "x, gate, output and last must not be NULL");
  if (int rc = check_workspace(a, workspace, workspace_bytes)) return rc;
  hipStream_t s = (hipStream_t)stream;
  SDK_DISPATCH_TOKEN_DTYPE(a->dtype, {
    const int lanes = lanes_of(a->width, kWide<T>);
    const bool wide = a->width % kWide<T> == 0 && fits<T>(a->x, a->x_strides) && fits<T>(a->gate, a->gate_strides) &&
                      aligned16(a->output);
    SCAN_SHAPE(in_launches(a, on_device(a, workspace), LANES, kWide<T>, [&](const Scan& p, dim3 grid) {
      if (p.segments > 1) launch(scan_spans<T, LANES, ALIGNED, false>, grid, dim3(kThreads), s, p);
      launch(scan_forward<T, LANES, ALIGNED>, grid, dim3(kThreads), s, p);
    }));
  });
  SDK_LAUNCH_CHECK("gated_scan_forward");
  return SDK_OK;
}

int sdk_gated_scan_backward(const sdk_gated_scan* a, void* workspace, size_t workspace_bytes, sdk_stream_t stream) {
  if (int rc = check(a)) return rc;
  if (!a->batch || !a->width) return SDK_OK;
  if (!a->tokens) {
    if (a->grad_state)
      launch(pass_state, dim3(64), dim3(256), (hipStream_t)stream, a->grad_last, a->grad_state, a->batch * a->width);
    SDK_LAUNCH_CHECK("gated_scan_backward");
    return SDK_OK;
  }
  SDK_REQUIRE(a->x && a->gate && a->output, "x, gate and output must not be NULL");
  SDK_REQUIRE(a->grad_x || a->grad_gate || a->grad_state, "one gradient at least must not be NULL");
  if (int rc = check_workspace(a, workspace, workspace_bytes)) return rc;
  hipStream_t s = (hipStream_t)stream;
  SDK_DISPATCH_TOKEN_DTYPE(a->dtype, {
    const int lanes = lanes_of(a->width, kWide<T>);
    const bool wide = a->width % kWide<T> == 0 && fits<T>(a->x, a->x_strides) && fits<T>(a->gate, a->gate_strides) &&
                      fits<T>(a->grad_output, a->grad_output_strides) && aligned16(a->output) && aligned16(a->grad_x) &&
                      aligned16(a->grad_gate);
    SCAN_SHAPE(in_launches(a, on_device(a, workspace), LANES, kWide<T>, [&](const Scan& p, dim3 grid) {
      if (p.segments > 1) launch(scan_spans<T, LANES, ALIGNED, true>, grid, dim3(kThreads), s, p);
      launch(scan_backward<T, LANES, ALIGNED>, grid, dim3(kThreads), s, p);
    }));
  });
  SDK_LAUNCH_CHECK("gated_scan_backward");
  return SDK_OK;
}

int sdk_gated_scan_step(const void* x, int64_t x_stride, const void* gate, int64_t gate_stride, float* state,
                        int64_t state_stride, void* output, int64_t batch, int64_t width, int32_t dtype,
                        sdk_stream_t stream) {
  SDK_REQUIRE(known(dtype), "unknown dtype %d (float32, bfloat16 and float16 only)", dtype);
  SDK_REQUIRE(batch >= 0 && batch < (int64_t)1 << 31 && width >= 0 && width <= (int64_t)1 << 20,
              "batch %lld must be below 2^31, width %lld at most 2^20", (long long)batch, (long long)width);
  if (!batch || !width) return SDK_OK;
  SDK_REQUIRE(x && gate && state && output, "x, gate, state and output must not be NULL");
  SDK_REQUIRE(batch == 1 || state_stride >= width, "states overlap: stride %lld of width %lld", (long long)state_stride,
              (long long)width);
  SDK_DISPATCH_TOKEN_DTYPE(dtype, {
    const int blocks = (int)ceil_div(width, kWide<T>);
    const bool wide = width % kWide<T> == 0 && aligned16(x) && aligned16(gate) && aligned16(output) &&
                      x_stride % kWide<T> == 0 && gate_stride % kWide<T> == 0;
    const int64_t each = most_groups(256) * 256 / blocks;
    for (int64_t b = 0; b < batch; b += each) {
      const int64_t count = std::min(each, batch - b);
      const dim3 grid((unsigned)ceil_div(count * blocks, 256));
      auto run = wide ? scan_step<T, true> : scan_step<T, false>;
      launch(run, grid, dim3(256), (hipStream_t)stream, (const T*)x + b * x_stride, x_stride, (const T*)gate + b * gate_stride,
             gate_stride, state + b * state_stride, state_stride, (T*)output + b * width, count, (int)width, blocks);
    }
  });
  SDK_LAUNCH_CHECK("gated_scan_step");
  return SDK_OK;
}

}  // extern "C"
