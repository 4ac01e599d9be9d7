// Gated linear recurrence along the tokens of sequences, with gradients, and its step for single tokens.
//
//   f_t = sigmoid(gate_t),  u_t = 1 - f_t        h_t = f_t h_{t-1} + u_t x_t
//   e_t = g_t + c_t,  c_{t-1} = f_t e_t          (g: the gradient of h_t; c behind the last token: that of the last state)
//   dx_t = u_t e_t    dgate_t = e_t (h_{t-1} - x_t) f_t u_t    gradient of the first state = c in front of the first token
//
// Each channel by itself.  A span of tokens acts on the state before it as h -> A h + H, and spans join: (A, H) then
// (A', H') is (A A', A' H + H').  So a workgroup takes 64 channels in 16 bits (32 in float32: 128 bytes of a token either
// way; a quarter of that where the width is no larger) and a tile of tokens, of which each thread walks 32 values
// (backward 16: two to eight tokens) in order; the threads' spans are joined over the tile, and each walks its tokens again
// from the state in front of them.  The tile's values stay in registers meanwhile.  Where batch and channels fill the GPU a
// workgroup goes through a whole sequence; otherwise it takes one tile, and tiles hand each other their spans while the
// kernel runs (scan_tiles).
//
// Bound by memory: three values read or written a token and channel forward, six backward (the gradients read h as
// it was rounded to the tensors' type).  2 x 8192 tokens of 1024 channels in bfloat16: forward 28 us (3.6 TB/s), backward 49
// (4.1 TB/s); all tiles of the forward are on the GPU at once, so that reading, waiting and writing follow each other.  A
// first launch for the spans of longer segments, which then were read again, took 49 and 74 us.  131072 tokens of 256
// channels in float16 forward: 53 us (3.8 TB/s; 95 with two launches).  Whole sequences, 64 of 512 tokens of 1024 channels in
// bfloat16: forward 45 us (4.5 TB/s), backward 101 (4.0 TB/s).
//
// The state, its gradient, the spans and the gates are float32.  Of f and u the lesser is formed, to its own relative
// precision, and weighs the distance of h and x:
//   open, f >= u:  h_t = h + u (x - h)        closed:  h_t = x + f (h - x)
// 1 - f of a rounded f near one would be off by a part of all that a long memory sums up, 1 - u of a rounded u near one by
// all that a closed gate leaves: at a gate of -14 by 3e-3 of f, from -18 on by f itself, in the gates' gradient and that of
// the states before, and a state of 1e4 would leave 2^-24 of itself where 1e-4 replaces it.
#include <algorithm>
#include <type_traits>

#include "token_types.hpp"

namespace sdk {
namespace token {
namespace {

constexpr int kThreads = 256;                  // of a workgroup that walks a whole sequence
constexpr int kWaiting = 512;                  // of one that takes a single tile of it

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
  unsigned long long* words;   // tickets and the tiles' spans
  int64_t x_strides[2], gate_strides[2], grad_strides[2];   // batch, token
  int64_t tokens, segment;     // segment: tokens of one, a multiple of the tile unless there is one alone
  int width, segments, blocks; // blocks: of channels
  int batches;                 // of this launch
  int64_t first;               // its first batch element
  int reverse;
};

// The lesser of f = sigmoid(g) and u = 1 - f, e / (1 + e) with e = e^-|g|, to its relative precision; its sign says which it
// is: f where it is +, a closed gate, u where it is -.
// FINE: to a few units of the last place (the power's argument in two parts, a correction of the reciprocal); 16-bit gates,
// whose results round to 16 bits, do without (5e-7 of it at gates of 8, 2e-6 at 30).
template <bool FINE>
__device__ __forceinline__ float gate_of(float g) {
  constexpr float kLog2e = 1.44269502e+00f, kLog2eRest = 1.92596303e-08f, kLn2 = 6.93147182e-01f;
  const float m = -fabsf(g), t = m * kLog2e;
  float e = __builtin_amdgcn_exp2f(t);
  if constexpr (FINE) {
    const float rest = fmaf(m, kLog2eRest, fmaf(m, kLog2e, -t));
    if (t > -126.f) e = fmaf(e * rest, kLn2, e);   // beyond it e is zero or nearly, and the rest may be no number
  }
  const float d = 1.f + e;
  float inverse = __builtin_amdgcn_rcpf(d);
  if constexpr (FINE) inverse = fmaf(fmaf(-d, inverse, 1.f), inverse, inverse);
  return copysignf(e * inverse, -g);
}
__device__ __forceinline__ bool closed(float s) { return __float_as_int(s) >= 0; }
// f h + u x
__device__ __forceinline__ float mixed(float s, float h, float x) { return fmaf(s, h - x, closed(s) ? x : h); }
// f c
__device__ __forceinline__ float kept(float s, float c) { return fmaf(s, c, closed(s) ? 0.f : c); }

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

// Joins the spans of the workgroup's threads in the order of their time lanes (thread = time lane * LANES + channel lane)
// up to the wave: on return `s` is the span of the threads before this one in its wave, and the waves' whole spans are in
// slots, [2][waves][LANES * V] floats that are free to be written.
template <int V, int LANES, int WAVES>
__device__ __forceinline__ void over_waves(Span<V>& s, float* slots) {
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
    for (int e = 0; e < V; ++e) slots[wave * C + c + e] = s.a[e], slots[(WAVES + wave) * C + c + e] = s.b[e];
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float a = __shfl_up(s.a[e], LANES), b = __shfl_up(s.b[e], LANES);
    s.a[e] = lane >= LANES ? a : 1.f;
    s.b[e] = lane >= LANES ? b : 0.f;
  }
}

// After a barrier: `in` is the state in front of this thread's span, and `carry`, the state in front of all of them, the
// one behind.
template <int V, int LANES, int WAVES>
__device__ __forceinline__ void from_waves(const Span<V>& s, float (&carry)[V], float (&in)[V], const float* slots) {
  constexpr int C = LANES * V;
  const int wave = threadIdx.x >> 6, c = (threadIdx.x % LANES) * V;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float h = carry[e];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w == wave) in[e] = fmaf(s.a[e], h, s.b[e]);
      h = fmaf(slots[w * C + c + e], h, slots[(WAVES + w) * C + c + e]);
    }
    carry[e] = h;
  }
}

// Where a workgroup works, and how tokens are counted: `at` counts them in the order of the recurrence.
template <typename T, int LANES>
struct Place {
  int64_t b, from, to, first_token, after_last;   // batch element, tokens of the segment, those that count (by `at`)
  int64_t lane_state;                             // of the thread's first channel in [batch][width]
  int segment, channel, left, time;
  // the thread of a workgroup that takes segment `segment_` of a block of channels
  __device__ __forceinline__ Place(const Scan& p, unsigned id, int segment_) {
    segment = segment_;
    channel = ((int)(id % (unsigned)p.blocks) * LANES + (int)(threadIdx.x % LANES)) * kWide<T>;
    time = threadIdx.x / LANES;
    begin(p, p.first + id / (unsigned)p.blocks);
  }
  // thread `id` of those that take a sequence's channels alone
  __device__ __forceinline__ Place(const Scan& p, int64_t id) {
    const int vectors = (p.width + kWide<T> - 1) / kWide<T>;
    segment = time = 0;
    channel = (int)(id % vectors) * kWide<T>;
    begin(p, p.first + id / vectors);
  }
  __device__ __forceinline__ void begin(const Scan& p, int64_t element) {
    b = element;
    from = segment * p.segment;
    to = from + p.segment < p.tokens ? from + p.segment : p.tokens;
    left = p.width - channel;
    lane_state = b * p.width + channel;
    int64_t n = p.tokens;
    if (p.lengths) n = p.lengths[b], n = n < 0 ? 0 : n > p.tokens ? p.tokens : n;
    first_token = p.reverse ? p.tokens - n : 0;
    after_last = p.reverse ? p.tokens : n;
  }
  __device__ __forceinline__ int64_t row(const Scan& p, int64_t at) const { return p.reverse ? p.tokens - 1 - at : at; }
  __device__ __forceinline__ bool counts(int64_t at) const { return left > 0 && at >= first_token && at < after_last; }
};

template <int V>
__device__ __forceinline__ void load_state(const float* p, int64_t at, float (&f)[V], int left) {
#pragma unroll
  for (int e = 0; e < V; ++e) f[e] = 0.f;
  if (p && left > 0) load_part<float, V>(p + at, f, left);
}

// 16 bytes of which the compiler no longer knows what has been made of them.
template <typename Raw>
__device__ __forceinline__ void anew(Raw& raw) {
  typedef unsigned Words __attribute__((ext_vector_type(4)));
  Words w = __builtin_bit_cast(Words, raw);
  asm("" : "+v"(w));
  raw = __builtin_bit_cast(Raw, w);
}

// ROWS tokens of a thread in the order of the walk, as they lie in memory, and what the walk does with them.  Forward they
// are at, at + 1, ..; backward at, at - 1, ..  FULL: all of the workgroup's tokens and channels count.
template <typename T, int LANES, bool ALIGNED, bool BACKWARD, int ROWS>
struct Walk {
  static constexpr int V = kWide<T>;
  static constexpr bool FINE = sizeof(T) == 4;
  static constexpr int STEP = BACKWARD ? -1 : 1;
  float s[ROWS][V];                       // the gate until open() or span(), which make it gate_of()
  Pack<T, V> x[ROWS], g[BACKWARD ? ROWS : 1], h[BACKWARD ? ROWS : 1];
  bool inside[ROWS], counts[ROWS];

  template <bool FULL>
  __device__ __forceinline__ void load(const Scan& p, const Place<T, LANES>& place, int64_t at) {
    // the thread's first token in memory, and the way from there to its others
    const int64_t row = place.row(p, at), way = (p.reverse != 0) != BACKWARD ? -1 : 1;
    const int64_t x_way = way * p.x_strides[1], gate_way = way * p.gate_strides[1], grad_way = way * p.grad_strides[1],
                  h_way = way * p.width;
    const T* px = (const T*)p.x + place.b * p.x_strides[0] + place.channel + row * p.x_strides[1];
    const T* pgate = (const T*)p.gate + place.b * p.gate_strides[0] + place.channel + row * p.gate_strides[1];
    const T* pgrad = (const T*)p.grad + place.b * p.grad_strides[0] + place.channel + row * p.grad_strides[1];
    const T* ph = (const T*)p.out + (place.b * p.tokens + row) * p.width + place.channel;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const int64_t t = at + STEP * r;
      inside[r] = FULL || (t >= place.from && t < place.to && place.left > 0);
      counts[r] = FULL || (inside[r] && place.counts(t));
      if constexpr (BACKWARD) {
#pragma unroll
        for (int e = 0; e < V; ++e) g[r].v[e] = (T)0.f;
      }
      if (counts[r]) {
        get<T, V, ALIGNED>(pgate + r * gate_way, s[r], place.left);
        get_raw<T, V, ALIGNED>(px + r * x_way, x[r], place.left);
        if constexpr (BACKWARD) {
          if (p.grad) get_raw<T, V, ALIGNED>(pgrad + r * grad_way, g[r], place.left);
          // the token before: backward that is the thread's next
          if (t > place.first_token) get_raw<T, V, ALIGNED>(ph + (r + 1) * h_way, h[r], place.left);
        }
      }
    }
  }

  // The gates of the tokens.
  __device__ __forceinline__ void open() {
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (counts[r]) s[r][e] = gate_of<FINE>(s[r][e]);
  }

  // The same, and what the tokens do to the state in front of them.
  template <bool FULL>
  __device__ __forceinline__ Span<V> span() {
    Span<V> all;
    unit(all);
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (FULL || counts[r]) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          s[r][e] = gate_of<FINE>(s[r][e]);
          if constexpr (BACKWARD)
            all.b[e] = kept(s[r][e], (float)g[r].v[e] + all.b[e]);
          else
            all.b[e] = mixed(s[r][e], all.b[e], (float)x[r].v[e]);
          all.a[e] = kept(s[r][e], all.a[e]);
        }
      }
    return all;
  }

  // The results of the tokens, given the state in front of them.
  template <bool FULL>
  __device__ __forceinline__ void finish(const Scan& p, const Place<T, LANES>& place, int64_t at, float (&in)[V]) {
    const int64_t way = ((p.reverse != 0) != BACKWARD ? -1 : 1) * p.width;
    const int64_t begin = (place.b * p.tokens + place.row(p, at)) * p.width + place.channel;
    if constexpr (BACKWARD) {
      // x and g are converted again here: kept from span() in 32 bits they leave no registers (scan_whole in 16 bits: 135 us
      // for 101; of the forward's one tensor they do not count)
#pragma unroll
      for (int r = 0; r < ROWS; ++r) anew(x[r]), anew(g[r]);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (!FULL && !inside[r]) continue;
      const int64_t row = begin + r * way;
      float y[V], z[V], before[V];
      if constexpr (BACKWARD) {
#pragma unroll
        for (int e = 0; e < V; ++e) before[e] = (float)h[r].v[e];
        if (at + STEP * r == place.first_token) {
#pragma unroll
          for (int e = 0; e < V; ++e) before[e] = p.state && e < place.left ? p.state[place.lane_state + e] : 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (!FULL) y[e] = z[e] = 0.f;
        if (FULL || counts[r]) {
          if constexpr (BACKWARD) {
            const float c = (float)g[r].v[e] + in[e], lesser = fabsf(s[r][e]);
            const float less = lesser * c, more = fmaf(-lesser, c, c);
            in[e] = closed(s[r][e]) ? less : more;
            y[e] = closed(s[r][e]) ? more : less;
            z[e] = more * lesser * (before[e] - (float)x[r].v[e]);
          } else {
            y[e] = in[e] = mixed(s[r][e], in[e], (float)x[r].v[e]);
          }
        }
      }
      if constexpr (BACKWARD) {
        if (p.grad_x) put<T, V, ALIGNED>((T*)p.grad_x + row, y, place.left);
        if (p.grad_gate) put<T, V, ALIGNED>((T*)p.grad_gate + row, z, place.left);
      } else {
        put<T, V, ALIGNED>((T*)p.out + row, y, place.left);
      }
    }
  }
};

// Whether all of `count` tokens from `first` on and all channels of the workgroup's block count.
template <typename T, int LANES, bool ALIGNED>
__device__ __forceinline__ bool is_full(const Scan& p, const Place<T, LANES>& place, int64_t first, int64_t count) {
  const int block_end = (place.channel / (LANES * kWide<T>) + 1) * LANES * kWide<T>;
  return ALIGNED && __builtin_amdgcn_readfirstlane(first >= place.from && first >= place.first_token &&
                                                   first + count <= place.to && first + count <= place.after_last &&
                                                   block_end <= p.width);
}

template <bool BACKWARD>
__device__ __forceinline__ const float* first_state(const Scan& p) { return BACKWARD ? p.grad_last : p.state; }

template <typename T, int LANES, bool BACKWARD>
__device__ __forceinline__ void store_last(const Scan& p, const Place<T, LANES>& place, const float (&carry)[kWide<T>]) {
  float* to = BACKWARD ? p.grad_state : p.last;
  if (to && place.left > 0 && place.time == 0) store_part<float, kWide<T>>(to + place.lane_state, carry, place.left);
}

// Tokens of a tile that a thread walks: a backward holds four tensors' values of each, a forward two.  (Half as many in
// float32: long scans 4 to 15 % slower.)
template <bool BACKWARD, int V>
constexpr int kRows = (BACKWARD ? 16 : 32) / V;

// Whole sequences, tile by tile: a workgroup a batch element and block of channels.
// (Backward two waves a SIMD, without which the compiler takes registers for one: 64 x 512 tokens of 1024 channels in
// bfloat16 188 us for 101.  Forward it arrives at two by itself, and is slower if told: 48 us for 45.)
template <typename T, int LANES, bool ALIGNED, bool BACKWARD>
__global__ __launch_bounds__(kThreads, BACKWARD ? 2 : 1) void scan_whole(const Scan p) {
  constexpr int V = kWide<T>, WAVES = kThreads / 64, ROWS = kRows<BACKWARD, V>, TILE = kThreads / LANES * ROWS;
  __shared__ float slots[2][2 * WAVES * LANES * V];
  const Place<T, LANES> place(p, blockIdx.x, 0);
  float carry[V];
  load_state<V>(first_state<BACKWARD>(p), place.lane_state, carry, place.left);
  const int64_t tiles = (p.tokens + TILE - 1) / TILE;
  for (int64_t i = 0; i < tiles; ++i) {
    const int64_t at = BACKWARD ? (tiles - i) * TILE - 1 - place.time * ROWS : i * TILE + place.time * ROWS;
    Walk<T, LANES, ALIGNED, BACKWARD, ROWS> walk;
    auto tile = [&](auto full) {
      constexpr bool FULL = decltype(full)::value;
      walk.template load<FULL>(p, place, at);
      Span<V> s = walk.template span<FULL>();
      float in[V];
      over_waves<V, LANES, WAVES>(s, slots[i & 1]);
      __syncthreads();
      from_waves<V, LANES, WAVES>(s, carry, in, slots[i & 1]);
      walk.template finish<FULL>(p, place, at, in);
    };
    if (is_full<T, LANES, ALIGNED>(p, place, (BACKWARD ? tiles - 1 - i : i) * TILE, TILE))
      tile(std::true_type());
    else
      tile(std::false_type());
  }
  store_last<T, LANES, BACKWARD>(p, place, carry);
}

// Short sequences: a thread takes 16 bytes of channels through all tokens.
template <typename T, bool ALIGNED, bool BACKWARD>
__global__ __launch_bounds__(kThreads) void scan_short(const Scan p) {
  constexpr int V = kWide<T>, ROWS = kRows<BACKWARD, V>;
  const int64_t id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (id >= (int64_t)p.batches * ((p.width + V - 1) / V)) return;
  const Place<T, 1> place(p, id);
  float carry[V];
  load_state<V>(first_state<BACKWARD>(p), place.lane_state, carry, place.left);
  for (int64_t i = 0; i < p.tokens; i += ROWS) {
    const int64_t at = BACKWARD ? p.tokens - 1 - i : i;
    Walk<T, 1, ALIGNED, BACKWARD, ROWS> walk;
    walk.template load<false>(p, place, at);
    walk.open();
    walk.template finish<false>(p, place, at, carry);
  }
  store_last<T, 1, BACKWARD>(p, place, carry);
}

// What other workgroups read of a tile: for each channel words {A, 1} and {H, 1} of its span, and of the last tile of a
// run the state behind it instead; zeros until they are written.  Value and tag arrive together, so nothing else has to be
// ordered.
typedef unsigned long long Word;
__device__ __forceinline__ Word word_of(float v, unsigned tag) { return (Word)tag << 32 | __float_as_uint(v); }
__device__ __forceinline__ void publish(Word* to, Word w) {
  __hip_atomic_store(to, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ Word seen(const Word* from) {
  return __hip_atomic_load(const_cast<Word*>(from), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
constexpr int kTicket = 16;       // words of a group's ticket: a line of its own
// About a second: a wait ends whatever happens, with NaN.  No wait gets there: it is for a workgroup that has begun (see
// scan_tiles) and waits for none behind it.
constexpr int kPolls = 1 << 20;

__global__ __launch_bounds__(256) void clear(Word* words, int64_t count) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) words[i] = 0;
}

// One tile of a sequence a workgroup, read once and held in registers while its span goes out and the state in front of it
// comes in.  Tiles form runs, of 32 where a workgroup has 64 channels: the state in front of a tile is the one behind the
// run before, carried over the spans of the tiles before it in its run, always in this order, so that results do not depend
// on who comes first.  Workgroups take the tiles of a group by its ticket, so those before a tile in its sequence have begun
// when it begins; each publishes its tile's span before it waits for others, and the last of a run waits for nothing that comes
// after it: every wait ends.
constexpr int kLook = 4;

template <typename T, int LANES, bool ALIGNED, bool BACKWARD>
__global__ __launch_bounds__(kWaiting, 4) void scan_tiles(const Scan p) {
  constexpr int V = kWide<T>, ROWS = kRows<BACKWARD, V>, WAVES = kWaiting / 64, C = LANES * V, SLOTS = kWaiting / C;
  __shared__ float slots[2 * WAVES * C], looked[2][SLOTS][C], entry[WAVES][C];
  __shared__ unsigned ticket;
  const unsigned groups = (unsigned)p.batches * p.blocks, id = blockIdx.x % groups;
  if (threadIdx.x == 0)
    ticket = __hip_atomic_fetch_add((unsigned*)(p.words + (int64_t)id * kTicket), 1u, __ATOMIC_RELAXED,
                                    __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  const int turn = (int)ticket;   // of the tile in the order of the walk
  const Place<T, LANES> place(p, id, BACKWARD ? p.segments - 1 - turn : turn);
  const int64_t at = BACKWARD ? place.from + p.segment - 1 - place.time * ROWS : place.from + place.time * ROWS;
  Walk<T, LANES, ALIGNED, BACKWARD, ROWS> walk;
  const bool full = is_full<T, LANES, ALIGNED>(p, place, place.from, p.segment);
  Span<V> s;
  if (full) {
    walk.template load<true>(p, place, at);
    s = walk.template span<true>();
  } else {
    walk.template load<false>(p, place, at);
    s = walk.template span<false>();
  }
  over_waves<V, LANES, WAVES>(s, slots);
  __syncthreads();

  // a channel a thread: words of tile `turn` are at [2][tiles][groups][C] behind the tickets
  const int c = threadIdx.x % C, slot = threadIdx.x / C;
  const int64_t step = (int64_t)groups * C;
  Word* products = p.words + groups * kTicket + (int64_t)id * C + c;
  Word* states = products + p.segments * step;
  constexpr int RUN = SLOTS * kLook;
  const bool closes = turn % RUN == RUN - 1;
  if (slot == 0 && !closes) {
    float a = 1.f, b = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      b = fmaf(slots[w * C + c], b, slots[(WAVES + w) * C + c]);
      a *= slots[w * C + c];
    }
    publish(products + turn * step, word_of(a, 1));
    publish(states + turn * step, word_of(b, 1));
  }
  // a channel a thread: four tiles of the run before this one, by slot
  const int start = turn / RUN * RUN, begin = start + slot * kLook;
  Word product[kLook], state[kLook];
#pragma unroll
  for (int i = 0; i < kLook; ++i) {
    const int other = begin + i < turn ? begin + i : 0;
    product[i] = seen(products + other * step);
    state[i] = seen(states + other * step);
  }
  float la = 1.f, lb = 0.f;
#pragma unroll
  for (int i = 0; i < kLook; ++i) {
    if (begin + i >= turn) continue;
    for (int polls = 0; !(state[i] >> 32 && product[i] >> 32) && polls < kPolls; ++polls) {
      __builtin_amdgcn_s_sleep(1);
      product[i] = seen(products + (begin + i) * step);
      state[i] = seen(states + (begin + i) * step);
    }
    const bool there = state[i] >> 32 && product[i] >> 32;
    const float oa = __uint_as_float((unsigned)product[i]);
    lb = fmaf(oa, lb, there ? __uint_as_float((unsigned)state[i]) : __builtin_nanf(""));
    la *= oa;
  }
  looked[0][slot][c] = la;
  looked[1][slot][c] = lb;
  __syncthreads();
  if (slot == 0) {
    const int channel = (int)(id % (unsigned)p.blocks) * C + c;
    const int64_t lane_state = place.b * p.width + channel;
    const float* first = first_state<BACKWARD>(p);
    float h = first && channel < p.width ? first[lane_state] : 0.f;
    if (start > 0) {
      Word w = seen(states + (start - 1) * step);
      for (int polls = 0; !(w >> 32) && polls < kPolls; ++polls) {
        __builtin_amdgcn_s_sleep(1);
        w = seen(states + (start - 1) * step);
      }
      h = w >> 32 ? __uint_as_float((unsigned)w) : __builtin_nanf("");
    }
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) h = fmaf(looked[0][i][c], h, looked[1][i][c]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      entry[w][c] = h;
      h = fmaf(slots[w * C + c], h, slots[(WAVES + w) * C + c]);
    }
    float* last = BACKWARD ? p.grad_state : p.last;
    if (closes) publish(states + turn * step, word_of(h, 1));
    if (turn + 1 == p.segments && last && channel < p.width) last[lane_state] = h;
  }
  __syncthreads();
  float in[V];
#pragma unroll
  for (int e = 0; e < V; ++e) in[e] = fmaf(s.a[e], entry[threadIdx.x >> 6][threadIdx.x % LANES * V + e], s.b[e]);
  if (full)
    walk.template finish<true>(p, place, at, in);
  else
    walk.template finish<false>(p, place, at, in);
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
    h[e] = mixed(gate_of<sizeof(T) == 4>(fg[e]), h[e], fx[e]);
  }
  store_part<float, V>(state + b * state_stride + c, h, left);
  put<T, V, ALIGNED>(out + b * width + c, h, left);
}

// Channel lanes of a workgroup: the fewest of 2 and 8 that take the width.
int lanes_of(int64_t width, int wide) { return width <= 2 * wide ? 2 : 8; }

// Tokens of a workgroup: all where batch and channels alone make four workgroups a CU, or a sequence is hardly longer than
// a tile; a tile otherwise.
constexpr int64_t kFill = 1024;
// Short sequences go to threads that walk them alone: up to 8 tokens, or 32 where such threads fill the GPU.  Forward in
// bfloat16, 1024 channels: 1024 sequences of 16 tokens 21 us (146 by tiles of 128 tokens), 512 of 32 28 (75), 256 of 64 48
// (42), 64 of 32 20 (10).
bool is_short(int64_t batch, int64_t tokens, int64_t vectors) {
  return tokens <= 8 || (tokens <= 32 && batch * vectors >= 32768);
}
int64_t segment_of(int64_t batch, int64_t tokens, int64_t width, int dtype, bool backward) {
  const int wide = dtype == SDK_F32 ? 4 : 8, lanes = lanes_of(width, wide);
  const int64_t groups = batch * ceil_div(width, lanes * wide), rows = (backward ? kRows<true, 1> : kRows<false, 1>) / wide;
  const int64_t tile = kWaiting / lanes * rows;
  return groups >= kFill || tokens <= tile || groups * ceil_div(tokens, tile) > most_groups(kWaiting) ? tokens : tile;
}

// Bytes for the tiles' words: a ticket's line a group, and two words a tile and channel (of whole blocks).
size_t words_of(const sdk_gated_scan* a, bool backward) {
  const int64_t segment = segment_of(a->batch, a->tokens, a->width, a->dtype, backward);
  if (segment == a->tokens) return 0;
  const int wide = a->dtype == SDK_F32 ? 4 : 8, c = lanes_of(a->width, wide) * wide;
  const int64_t groups = a->batch * ceil_div(a->width, c);
  return (size_t)(8 * groups * (kTicket + 2 * ceil_div(a->tokens, segment) * c));
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

Scan on_device(const sdk_gated_scan* a, void* workspace, int lanes, int wide, bool backward) {
  Scan p = {};
  p.x = a->x, p.gate = a->gate, p.state = a->state, p.lengths = a->lengths, p.out = a->output, p.last = a->last;
  p.grad = a->grad_output, p.grad_last = a->grad_last, p.grad_x = a->grad_x, p.grad_gate = a->grad_gate;
  p.grad_state = a->grad_state, p.words = (unsigned long long*)workspace;
  for (int i = 0; i < 2; ++i)
    p.x_strides[i] = a->x_strides[i], p.gate_strides[i] = a->gate_strides[i],
    p.grad_strides[i] = a->grad_output_strides[i];
  p.tokens = a->tokens, p.width = (int)a->width, p.reverse = a->reverse != 0;
  p.segment = segment_of(a->batch, a->tokens, a->width, a->dtype, backward);
  p.blocks = (int)ceil_div(p.width, lanes * wide);
  p.segments = (int)ceil_div(p.tokens, p.segment);
  return p;
}

template <typename T, int LANES, bool ALIGNED, bool BACKWARD>
void run(const sdk_gated_scan* a, void* workspace, hipStream_t s) {
  Scan p = on_device(a, workspace, LANES, kWide<T>, BACKWARD);
  const int64_t vectors = ceil_div(p.width, kWide<T>), most = most_groups(kThreads) * kThreads / vectors;
  if (is_short(a->batch, p.tokens, vectors)) {
    for (p.first = 0; p.first < a->batch; p.first += most) {
      p.batches = (int)std::min(most, a->batch - p.first);
      launch(scan_short<T, ALIGNED, BACKWARD>, dim3((unsigned)ceil_div(p.batches * vectors, kThreads)), dim3(kThreads), s, p);
    }
    return;
  }
  if (p.segments > 1) {   // fewer than kFill workgroups for a segment
    const int64_t words = (int64_t)(words_of(a, BACKWARD) / 8);
    launch(clear, dim3((unsigned)std::min<int64_t>(ceil_div(words, 256), 1024)), dim3(256), s, p.words, words);
    p.batches = (int)a->batch;
    launch(scan_tiles<T, LANES, ALIGNED, BACKWARD>,
           dim3((unsigned)((int64_t)p.batches * p.blocks * p.segments)), dim3(kWaiting), s, p);
    return;
  }
  const int64_t each = most_groups(kThreads) / p.blocks;   // batch elements of a launch
  for (p.first = 0; p.first < a->batch; p.first += each) {
    p.batches = (int)std::min(each, a->batch - p.first);
    launch(scan_whole<T, LANES, ALIGNED, BACKWARD>, dim3((unsigned)((int64_t)p.batches * p.blocks)), dim3(kThreads), s, p);
  }
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

int check_workspace(const sdk_gated_scan* a, const void* workspace, size_t bytes, bool backward) {
  const size_t need = words_of(a, backward);
  if (need && (!workspace || bytes < need || (uintptr_t)workspace % 8))
    return fail(SDK_ERR_WORKSPACE, "workspace of %zu bytes at a multiple of 8, %zu needed", bytes, need);
  return SDK_OK;
}

}  // namespace
}  // namespace token
}  // namespace sdk

using namespace sdk;
using namespace sdk::token;

extern "C" {

size_t sdk_gated_scan_workspace_bytes(const sdk_gated_scan* a, int32_t backward) {
  if (check(a) != SDK_OK || !a->batch || !a->tokens || !a->width) return 0;
  return words_of(a, backward != 0);
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
  if (int rc = check_workspace(a, workspace, workspace_bytes, false)) return rc;
  hipStream_t s = (hipStream_t)stream;
  SDK_DISPATCH_TOKEN_DTYPE(a->dtype, {
    const int lanes = lanes_of(a->width, kWide<T>);
    const bool wide = a->width % kWide<T> == 0 && fits<T>(a->x, a->x_strides) && fits<T>(a->gate, a->gate_strides) &&
                      aligned16(a->output);
    SCAN_SHAPE(run<T, LANES, ALIGNED, false>(a, workspace, s));
  });
  SDK_LAUNCH_CHECK("gated_scan_forward");
  return SDK_OK;
}

int sdk_gated_scan_backward(const sdk_gated_scan* a, void* workspace, size_t workspace_bytes, sdk_stream_t stream) {
  if (int rc = check(a)) return rc;
  if (!a->batch || !a->width) return SDK_OK;
  if (!a->tokens) {
    if (!a->grad_state) return SDK_OK;
    launch(pass_state, dim3(64), dim3(256), (hipStream_t)stream, a->grad_last, a->grad_state, a->batch * a->width);
    SDK_LAUNCH_CHECK("gated_scan_backward");
    return SDK_OK;
  }
  SDK_REQUIRE(a->x && a->gate && a->output, "x, gate and output must not be NULL");
  SDK_REQUIRE(a->grad_x || a->grad_gate || a->grad_state, "one gradient at least must not be NULL");
  if (int rc = check_workspace(a, workspace, workspace_bytes, true)) return rc;
  hipStream_t s = (hipStream_t)stream;
  SDK_DISPATCH_TOKEN_DTYPE(a->dtype, {
    const int lanes = lanes_of(a->width, kWide<T>);
    const bool wide = a->width % kWide<T> == 0 && fits<T>(a->x, a->x_strides) && fits<T>(a->gate, a->gate_strides) &&
                      fits<T>(a->grad_output, a->grad_output_strides) && aligned16(a->output) && aligned16(a->grad_x) &&
                      aligned16(a->grad_gate);
    SCAN_SHAPE(run<T, LANES, ALIGNED, true>(a, workspace, s));
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
