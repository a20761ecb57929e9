// recurrence.hip — gated linear recurrence over packed sequences, forward, backward and one step.
//
// Per channel, with r = sigmoid(gate_a), z = sigmoid(gate_x) and log a = -rate softplus(decay) r:
//   h_t = a_t h_{t-1} + m_t z_t x_t,   m_t = sqrt(1 - a_t^2),
// h before a sequence's first token from `state`, or 0.  In reverse, the scan runs from each
// sequence's last token to its first.
//
// A workgroup takes a chunk of kChunk tokens and 64 V channels, each of its waves kLen tokens in a
// row, a lane V channels.  A stretch of tokens is a map h -> A h + H of the state before it; maps are
// composed over the waves in LDS and over the chunks by scan_carry.  Pass 1 forms the chunks' maps,
// pass 2 the outputs from the states that the chunks begin with.  All in float32, whatever the inputs.
//
// The inputs are read twice in each direction, and still vector instructions bound the passes: 79 to 94%
// of a SIMD's cycles, for two sigmoids, a decay, a root and 1 - a^2 of every element.  131,072 tokens of
// 256 channels in bfloat16: pass 1 60 us, carry 9, pass 2 63; backward 34, 9 and 122, decay's sums 4.
#include "common.hpp"

namespace geo {
namespace rec {

// Longer stretches would hold more rows in registers than leave three workgroups a CU in the backward's
// second pass (which with two takes 145 us instead of 121 at 131,072 x 256 bfloat16).
constexpr int kLen = 8, kWaves = 8, kChunk = kLen * kWaves;
constexpr float kLog2e = 1.4426950408889634f;

template <typename T, int V> struct Pack;
template <> struct Pack<float, 1> { using Raw = float; };
template <> struct Pack<float, 2> { using Raw = float2; };
template <> struct Pack<__bf16, 1> { using Raw = uint16_t; };
template <> struct Pack<__bf16, 2> { using Raw = uint32_t; };
template <> struct Pack<_Float16, 1> { using Raw = uint16_t; };
template <> struct Pack<_Float16, 2> { using Raw = uint32_t; };

template <typename T, int V>
__device__ __forceinline__ void unpack(typename Pack<T, V>::Raw r, float (&f)[V]) {
  union { typename Pack<T, V>::Raw r; T t[V]; } u;
  u.r = r;
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = static_cast<float>(u.t[v]);
}
// Each value's float32 rounded.  (The product and sum that formed it would else be rounded to float16 at
// once in one instruction, here and there, and an output then not be its state's rounding.)
template <typename T, int V>
__device__ __forceinline__ typename Pack<T, V>::Raw pack(const float (&f)[V]) {
  union { typename Pack<T, V>::Raw r; T t[V]; } u;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float x = f[v];
    asm("" : "+v"(x));
    u.t[v] = static_cast<T>(x);
  }
  return u.r;
}

// Relatively exact far out too: exp2's argument loses |x| log2(e) units by its rounding, which the
// factor 1 + ln 2 err gives back.  (The median turns the NaN that err is for infinite x into a
// finite number; exp2 is then 0 or infinite, and NaN where x is.)
__device__ __forceinline__ float sigmoid(float x) {
  const float t = -x * kLog2e;
  const float err = __builtin_amdgcn_fmed3f(fmaf(-x, kLog2e, -t), -1.f, 1.f);
  return __builtin_amdgcn_rcpf(fmaf(__builtin_amdgcn_exp2f(t), fmaf(err, 0.6931471805599453f, 1.f), 1.f));
}
// 1 - exp(u) for u <= 0: near 0 the series of -expm1, since the difference would cancel (its first term left
// out is u^5 / 720 of it, 4e-8 at its end).  Just past it a unit of exp_u is 5e-7 of the difference; as
// the square of a rounded exponential exp_u is off by up to three, m, its root, by half of that.
__device__ __forceinline__ float one_minus_exp(float u, float exp_u) {
  float s = fmaf(u, 1.f / 120.f, 1.f / 24.f);
  s = fmaf(s, u, 1.f / 6.f);
  s = fmaf(s, u, 0.5f);
  s = fmaf(s, u, 1.f);
  return u > -0.125f ? -u * s : 1.f - exp_u;
}
// A channel's log a per unit of the gate, -rate softplus(decay); softplus(x) = x for large x, where
// exp(x) would overflow.
__device__ __forceinline__ float log_rate(float decay, float rate) {
  return -rate * (decay > 20.f ? decay : log1pf(expf(decay)));
}

struct Gates {
  float a, m, r, z;
};
__device__ __forceinline__ float decay_of(float r, float lr) { return __builtin_amdgcn_exp2f(lr * kLog2e * r); }
__device__ __forceinline__ Gates gates(float ga, float gx, float lr) {
  Gates g;
  g.r = sigmoid(ga);
  g.z = sigmoid(gx);
  g.a = decay_of(g.r, lr);
  g.m = __builtin_amdgcn_sqrtf(one_minus_exp(2.f * lr * g.r, g.a * g.a));
  return g;
}

struct Scan {
  const void *x, *ga, *gx;
  int64_t x_st, ga_st, gx_st;  // elements from token to token
  const float* decay;
  const int64_t* ptr;          // [B + 1], or null: one sequence
  const float* state;          // [B, C], or null
  int64_t T, C;
  int64_t B;
  float rate;
  int reverse;
};

// The tokens of a wave's stretch in scan order: lane l < kLen looks at token number l of it.
struct Stretch {
  int64_t n0;                    // the first token's number in scan order
  uint32_t begin, finish, live;  // bits: first of its sequence in scan order, last, of a sequence
  int seq;                       // this lane's token's sequence
  __device__ __forceinline__ bool plain() const { return live == (1u << kLen) - 1 && !(begin | finish); }
};
__device__ __forceinline__ int64_t token(const Scan& s, int64_t n) { return s.reverse ? s.T - 1 - n : n; }
__device__ __forceinline__ Stretch look(const Scan& s, int64_t n0) {
  constexpr uint32_t kAll = (1u << kLen) - 1;
  Stretch c;
  c.n0 = n0;
  c.seq = 0;
  if (!s.ptr) {  // one sequence: on the scalar unit
    const int64_t left = s.T - n0;
    c.live = left >= kLen ? kAll : left > 0 ? (1u << left) - 1 : 0u;
    c.begin = n0 == 0 ? 1u : 0u;
    c.finish = left > 0 && left <= kLen ? 1u << (left - 1) : 0u;
    return c;
  }
  const int T = static_cast<int>(s.T), n = static_cast<int>(n0) + (lane_id() & (kLen - 1));
  const int t = s.reverse ? T - 1 - min(n, T - 1) : min(n, T - 1);
  auto at = [&](int b) { return static_cast<int>(min(max(s.ptr[b], int64_t(-1)), int64_t(T))); };
  int lo = 0, hi = static_cast<int>(s.B) - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (at(mid) <= t) lo = mid; else hi = mid - 1;
  }
  const int first = at(lo), end = at(lo + 1), first_in = max(first, 0);
  const bool live = n < T && first <= t && t < end;
  c.live = static_cast<uint32_t>(__ballot(live)) & kAll;
  c.begin = static_cast<uint32_t>(__ballot(live && t == (s.reverse ? end - 1 : first_in))) & kAll;
  c.finish = static_cast<uint32_t>(__ballot(live && t == (s.reverse ? first_in : end - 1))) & kAll;
  c.seq = lo;
  return c;
}
__device__ __forceinline__ int64_t seq_at(const Stretch& c, int l) { return __builtin_amdgcn_readlane(c.seq, l); }

template <typename T, int V>
struct Rows {
  typename Pack<T, V>::Raw raw[kLen];
  __device__ __forceinline__ void load(const void* base, int64_t stride, const Scan& s, int64_t n0, int64_t at) {
#pragma unroll
    for (int l = 0; l < kLen; ++l) {
      const T* row = static_cast<const T*>(base) + token(s, min(n0 + l, s.T - 1)) * stride;
      raw[l] = *reinterpret_cast<const typename Pack<T, V>::Raw*>(row + at);
    }
  }
};

// Grid of the passes: (chunk, block of 64 V channels), channels fastest.
struct Place {
  int64_t chunk, n0, at;  // n0: the wave's first token's number; at: this lane's first channel, in range
  int64_t base;           // the workgroup's first channel
  int wave;
  bool mine;
};
template <int V>
__device__ __forceinline__ Place place(const Scan& s) {
  const int64_t blocks = (s.C + 64 * V - 1) / (64 * V), w = xcd_block();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t base = w % blocks * 64 * V, at = base + lane_id() * V, chunk = w / blocks;
  return {chunk, chunk * kChunk + wave * kLen, min(at, s.C - V), base, wave, at < s.C};
}

// log_rate of the lane's channels, formed once for the workgroup: its logarithm and exponential take
// as many instructions as two tokens.  The barrier leaves the rows' loads in flight.
template <int V>
__device__ __forceinline__ void share_rates(const Scan& s, const Place& p, float (&lr)[V]) {
  __shared__ float rates[64 * V];
  if (threadIdx.x < 64 * V) rates[threadIdx.x] = log_rate(s.decay[min(p.base + threadIdx.x, s.C - 1)], s.rate);
  lds_barrier();
#pragma unroll
  for (int v = 0; v < V; ++v) lr[v] = rates[lane_id() * V + v];
}

// The factor of a map across which nothing passes, as at the beginning of a sequence: a factor of 0
// would let the infinities and NaN of the sequence before through.  No decay is negative.
constexpr float kCut = -1.f;
__device__ __forceinline__ float after(float a, float add, float h) { return a == kCut ? add : fmaf(a, h, add); }
__device__ __forceinline__ float chain(float a1, float a2) { return a1 == kCut || a2 == kCut ? kCut : a1 * a2; }

// Where a chunk's map, state or sum of a channel lies: blocks of kCarryChannels channels, chunk after
// chunk, so that the workgroup that carries a block over the chunks reads and writes whole lines.  Narrow
// blocks spread the reading over CUs.
constexpr int kCarryChannels = 4;
__host__ __device__ inline int64_t padded(int64_t C) { return (C + kCarryChannels - 1) / kCarryChannels * kCarryChannels; }
__device__ __forceinline__ int64_t chunk_place(int64_t chunk, int64_t chunks, int64_t at) {
  return (at / kCarryChannels * chunks + chunk) * kCarryChannels + at % kCarryChannels;
}

// The waves' maps of a chunk, in LDS.
template <int V>
struct Maps {
  float a[kWaves][64 * V], h[kWaves][64 * V];
  __device__ __forceinline__ void put(int wave, const float (&A)[V], const float (&H)[V]) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      a[wave][lane_id() * V + v] = A[v];
      h[wave][lane_id() * V + v] = H[v];
    }
  }
  // state[v] through the maps of waves from .. to - 1 (or, to < from, from - 1 down to `to`)
  __device__ __forceinline__ void run(int from, int to, float (&state)[V]) const {
    const int step = to < from ? -1 : 1;
    for (int w = to < from ? from - 1 : from; w != (to < from ? to - 1 : to); w += step)
#pragma unroll
      for (int v = 0; v < V; ++v) state[v] = after(a[w][lane_id() * V + v], h[w][lane_id() * V + v], state[v]);
  }
};

// Factors and terms of a wave's tokens.
template <typename T, int V>
__device__ __forceinline__ void terms(const Rows<T, V>& x, const Rows<T, V>& ga, const Rows<T, V>& gx, const float (&lr)[V],
                                      Gates (&g)[kLen][V], float (&fb)[kLen][V]) {
#pragma unroll
  for (int l = 0; l < kLen; ++l) {
    float xf[V], af[V], gf[V];
    unpack<T, V>(x.raw[l], xf);
    unpack<T, V>(ga.raw[l], af);
    unpack<T, V>(gx.raw[l], gf);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      g[l][v] = gates(af[v], gf[v], lr[v]);
      fb[l][v] = g[l][v].m * g[l][v].z * xf[v];
    }
  }
}
// The map of a wave's stretch.  PLAIN: no border of a sequence lies in it.
template <bool PLAIN, int V>
__device__ __forceinline__ void steps(const Scan& s, const Stretch& c, const Place& p, const Gates (&g)[kLen][V],
                                      const float (&fb)[kLen][V], float (&A)[V], float (&H)[V]) {
#pragma unroll
  for (int l = 0; l < kLen; ++l) {
    const bool begin = !PLAIN && ((c.begin >> l) & 1), live = PLAIN || ((c.live >> l) & 1);
    const int64_t b = begin ? seq_at(c, l) : 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float a = g[l][v].a;
      if (begin) {
        A[v] = kCut;
        H[v] = s.state ? s.state[b * s.C + p.at + v] : 0.f;
      }
      if (PLAIN) {
        A[v] *= a;
        H[v] = fmaf(a, H[v], fb[l][v]);
      } else {
        A[v] = live ? chain(A[v], a) : kCut;
        H[v] = live ? fmaf(a, H[v], fb[l][v]) : 0.f;
      }
    }
  }
}

// The state that reaches a chunk from few others (at most kFew, so that each wave looks at kFew / kWaves
// of them): their maps composed by the workgroup itself, which saves the launch that carries them (2048
// tokens of 64 channels: 13.8 us of kernels instead of 17).  The backward has no registers for it.
constexpr int kFew = 32;
template <int V>
__device__ __forceinline__ void state_from_maps(Maps<V>& maps, const float2* __restrict__ map, const Place& p, int64_t chunks,
                                                float (&state)[V]) {
  constexpr int kEach = kFew / kWaves;
  float2 m[kEach][V];
  float A[V], H[V];
#pragma unroll
  for (int n = 0; n < kEach; ++n)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int64_t c = min(static_cast<int64_t>(p.wave * kEach + n), chunks - 1);
      m[n][v] = map[chunk_place(c, chunks, p.at + v)];
    }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = 1.f;
    H[v] = state[v] = 0.f;
#pragma unroll
    for (int n = 0; n < kEach; ++n)
      if (p.wave * kEach + n < p.chunk) {
        A[v] = chain(A[v], m[n][v].x);
        H[v] = after(m[n][v].x, m[n][v].y, H[v]);
      }
  }
  maps.put(p.wave, A, H);
  __syncthreads();
  maps.run(0, kWaves, state);
  __syncthreads();
}

// Pass 1: the chunk's map.
template <typename T, int V>
__global__ __launch_bounds__(64 * kWaves, 4) void scan_map(const Scan s, int64_t chunks, float2* __restrict__ map) {
  __shared__ Maps<V> maps;
  const Place p = place<V>(s);
  Rows<T, V> x, ga, gx;
  x.load(s.x, s.x_st, s, p.n0, p.at);
  ga.load(s.ga, s.ga_st, s, p.n0, p.at);
  gx.load(s.gx, s.gx_st, s, p.n0, p.at);
  const Stretch c = look(s, p.n0);
  float lr[V], A[V], H[V], fb[kLen][V];
  Gates g[kLen][V];
  share_rates(s, p, lr);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = 1.f;
    H[v] = 0.f;
  }
  terms(x, ga, gx, lr, g, fb);
  if (c.plain()) steps<true>(s, c, p, g, fb, A, H);
  else steps<false>(s, c, p, g, fb, A, H);
  maps.put(p.wave, A, H);
  __syncthreads();
  if (p.wave || !p.mine) return;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float Av = 1.f;
    for (int w = 0; w < kWaves; ++w) Av = chain(Av, maps.a[w][lane_id() * V + v]);
    A[v] = Av;
    H[v] = 0.f;
  }
  maps.run(0, kWaves, H);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    map[chunk_place(p.chunk, chunks, p.at + v)] = make_float2(A[v], H[v]);
  }
}

// Between the passes: maps composed over the chunks to the state before each chunk (or, `back`, after
// it, from the last chunk to the first).  A workgroup shares its channels among 64 runs of chunks, each
// held in registers by one thread per channel, so that a round of 2048 chunks costs one memory latency
// (the loads are at clamped places: under a condition each waited for the one before, 26 us instead of
// 9.4 us at 2048 chunks of 256 channels) and 64 steps over LDS.
constexpr int kRuns = 64, kHeld = 32;
__global__ __launch_bounds__(kCarryChannels * kRuns) void scan_carry(const float2* __restrict__ map, float* __restrict__ carry,
                                                                     int64_t chunks, int back) {
  __shared__ float2 runs[kRuns][kCarryChannels];
  const int ch = threadIdx.x % kCarryChannels, run = threadIdx.x / kCarryChannels;
  auto index = [&](int64_t c) { return (blockIdx.x * chunks + (back ? chunks - 1 - c : c)) * kCarryChannels + ch; };
  float ahead = 0.f;  // the state before the round
  for (int64_t r = 0; r < chunks; r += kRuns * kHeld) {
    // a run's length: the round's chunks shared evenly
    const int per = static_cast<int>(min((chunks - r + kRuns - 1) / kRuns, int64_t(kHeld)));
    const int64_t c0 = r + static_cast<int64_t>(run) * per, c1 = min(c0 + per, chunks);
    float2 m[kHeld];
    float A = 1.f, H = 0.f;
#pragma unroll
    for (int n = 0; n < kHeld; ++n) m[n] = map[index(min(c0 + min(n, per - 1), chunks - 1))];
#pragma unroll
    for (int n = 0; n < kHeld; ++n)
      if (c0 + n < c1) {
        A = chain(A, m[n].x);
        H = after(m[n].x, m[n].y, H);
      }
    __syncthreads();
    runs[run][ch] = make_float2(A, H);
    __syncthreads();
    if (threadIdx.x < kCarryChannels) {  // the state before each run, in the place of its map
      const int used = static_cast<int>(min((chunks - r + per - 1) / per, int64_t(kRuns)));
      for (int n0 = 0; n0 < used; n0 += 16) {
        float2 y[16];
#pragma unroll
        for (int n = 0; n < 16; ++n) y[n] = runs[n0 + n][ch];
#pragma unroll
        for (int n = 0; n < 16; ++n) {
          runs[n0 + n][ch].y = ahead;
          if (n0 + n < used) ahead = after(y[n].x, y[n].y, ahead);
        }
      }
    }
    __syncthreads();
    H = runs[run][ch].y;
#pragma unroll
    for (int n = 0; n < kHeld; ++n)
      if (c0 + n < c1) {
        carry[index(c0 + n)] = H;
        H = after(m[n].x, m[n].y, H);
      }
  }
}

// A sequence without tokens passes its state (or its state's gradient) on; a chunk's first wave sees
// to its share of them.
__device__ __forceinline__ void pass_empty(const Scan& s, const Place& p, int64_t chunks, int V, const float* from, float* to) {
  if (!s.ptr || !to || p.wave) return;
  const int64_t per = (s.B + chunks - 1) / chunks;
  for (int64_t b = p.chunk * per; b < min((p.chunk + 1) * per, s.B); ++b) {
    if (max(s.ptr[b], int64_t(0)) < min(s.ptr[b + 1], s.T) || !p.mine) continue;
    for (int v = 0; v < V; ++v) to[b * s.C + p.at + v] = from ? from[b * s.C + p.at + v] : 0.f;
  }
}

// Pass 2: the outputs.
template <typename T, int V>
__global__ __launch_bounds__(64 * kWaves, 4) void scan_out(const Scan s, int64_t chunks, const float2* __restrict__ map,
                                                           float* __restrict__ carry, T* __restrict__ h, float* __restrict__ last) {
  __shared__ Maps<V> maps;
  const Place p = place<V>(s);
  Rows<T, V> x, ga, gx;
  x.load(s.x, s.x_st, s, p.n0, p.at);
  ga.load(s.ga, s.ga_st, s, p.n0, p.at);
  gx.load(s.gx, s.gx_st, s, p.n0, p.at);
  const Stretch c = look(s, p.n0);
  float lr[V], A[V], H[V], state[V], fb[kLen][V];
  Gates g[kLen][V];
  share_rates(s, p, lr);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = 1.f;
    H[v] = 0.f;
    state[v] = chunks > kFew ? carry[chunk_place(p.chunk, chunks, p.at + v)] : 0.f;
  }
  if (chunks <= kFew) {
    if (chunks > 1) state_from_maps(maps, map, p, chunks, state);
    if (p.wave == 0 && p.mine)
#pragma unroll
      for (int v = 0; v < V; ++v) carry[chunk_place(p.chunk, chunks, p.at + v)] = state[v];
  }
  const bool plain = c.plain();
  terms(x, ga, gx, lr, g, fb);
  if (plain) steps<true>(s, c, p, g, fb, A, H);
  else steps<false>(s, c, p, g, fb, A, H);
  maps.put(p.wave, A, H);
  __syncthreads();
  maps.run(0, p.wave, state);
  if (plain) {
#pragma unroll
    for (int l = 0; l < kLen; ++l) {
#pragma unroll
      for (int v = 0; v < V; ++v) state[v] = fmaf(g[l][v].a, state[v], fb[l][v]);
      if (p.mine) *reinterpret_cast<typename Pack<T, V>::Raw*>(h + token(s, p.n0 + l) * s.C + p.at) = pack<T, V>(state);
    }
  } else {
#pragma unroll
    for (int l = 0; l < kLen; ++l) {
      const bool begin = (c.begin >> l) & 1, live = (c.live >> l) & 1;
      const int64_t b = seq_at(c, l), n = p.n0 + l;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (begin) state[v] = s.state ? s.state[b * s.C + p.at + v] : 0.f;
        state[v] = live ? fmaf(g[l][v].a, state[v], fb[l][v]) : 0.f;
      }
      if (p.mine && n < s.T)
        *reinterpret_cast<typename Pack<T, V>::Raw*>(h + token(s, n) * s.C + p.at) = pack<T, V>(state);
      if (((c.finish >> l) & 1) && p.mine)
#pragma unroll
        for (int v = 0; v < V; ++v) last[b * s.C + p.at + v] = state[v];
    }
  }
  pass_empty(s, p, chunks, V, s.state, last);
}

// Backward.  With e_t = a_t g_t, what token t's gradient hands to the token before:
//   g_t = dh_t + e_{t+1} (dlast beyond a sequence's last token),  e_t = a_t g_t,
// a scan against the order of the forward's, whose maps need gate_a and dh alone.
struct Grad {
  const void* dh;          // contiguous [T, C], or null
  const float* dlast;      // [B, C], or null
  void *dx, *dga, *dgx;    // contiguous [T, C]
  float *dstate;           // [B, C], or null
  float* ddecay;           // sums of the chunks, by chunk_place
};

// The map of a wave's stretch against the scan order, e before it from e behind it.
template <bool PLAIN, typename T, int V>
__device__ __forceinline__ void back_steps(const Scan& s, const Grad& d, const Stretch& c, const Place& p, const Rows<T, V>& dh,
                                           const Gates (&g)[kLen][V], float (&A)[V], float (&E)[V]) {
#pragma unroll
  for (int l = kLen - 1; l >= 0; --l) {
    float hf[V] = {};
    if (d.dh) unpack<T, V>(dh.raw[l], hf);
    const bool finish = !PLAIN && ((c.finish >> l) & 1), live = PLAIN || ((c.live >> l) & 1);
    const int64_t b = finish ? seq_at(c, l) : 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float a = g[l][v].a;
      if (finish) {
        A[v] = kCut;
        E[v] = d.dlast ? d.dlast[b * s.C + p.at + v] : 0.f;
      }
      if (PLAIN) {
        A[v] *= a;
        E[v] = a * (hf[v] + E[v]);
      } else {
        A[v] = live ? chain(A[v], a) : kCut;
        E[v] = live ? a * (hf[v] + E[v]) : 0.f;
      }
    }
  }
}

template <typename T, int V>
__global__ __launch_bounds__(64 * kWaves) void scan_bwd_map(const Scan s, const Grad d, int64_t chunks,
                                                            float2* __restrict__ map) {
  __shared__ Maps<V> maps;
  const Place p = place<V>(s);
  Rows<T, V> ga, dh;
  ga.load(s.ga, s.ga_st, s, p.n0, p.at);
  if (d.dh) dh.load(d.dh, s.C, s, p.n0, p.at);
  const Stretch c = look(s, p.n0);
  float lr[V], A[V], E[V];
  Gates g[kLen][V];
  share_rates(s, p, lr);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = 1.f;
    E[v] = 0.f;
  }
#pragma unroll
  for (int l = 0; l < kLen; ++l) {
    float af[V];
    unpack<T, V>(ga.raw[l], af);
#pragma unroll
    for (int v = 0; v < V; ++v) g[l][v].a = decay_of(sigmoid(af[v]), lr[v]);
  }
  if (c.plain()) back_steps<true>(s, d, c, p, dh, g, A, E);
  else back_steps<false>(s, d, c, p, dh, g, A, E);
  maps.put(p.wave, A, E);
  __syncthreads();
  if (p.wave || !p.mine) return;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float Av = 1.f;
    for (int w = 0; w < kWaves; ++w) Av = chain(Av, maps.a[w][lane_id() * V + v]);
    A[v] = Av;
    E[v] = 0.f;
  }
  maps.run(kWaves, 0, E);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    map[chunk_place(p.chunk, chunks, p.at + v)] = make_float2(A[v], E[v]);
  }
}

// Pass 2 of the backward: the states ahead of the wave's tokens again, then the gradients against the
// scan order.  The gates stay in registers between the two.
template <bool PLAIN, typename T, int V>
__device__ __forceinline__ void back_out(const Scan& s, const Grad& d, const Stretch& c, const Place& p, const Rows<T, V>& x,
                                         const Rows<T, V>& dh, const float (&lr)[V], const Gates (&g)[kLen][V],
                                         const float (&before)[kLen][V], float (&E)[V],
                                         float (&dlr)[V]) {
  using Raw = typename Pack<T, V>::Raw;
#pragma unroll
  for (int l = kLen - 1; l >= 0; --l) {
    float xf[V], hf[V] = {}, ox[V], oa[V], og[V];
    unpack<T, V>(x.raw[l], xf);
    if (d.dh) unpack<T, V>(dh.raw[l], hf);
    const bool finish = !PLAIN && ((c.finish >> l) & 1), live = PLAIN || ((c.live >> l) & 1);
    const int64_t b = PLAIN ? 0 : seq_at(c, l), n = p.n0 + l;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (finish) E[v] = d.dlast ? d.dlast[b * s.C + p.at + v] : 0.f;
      const float a = g[l][v].a, m = g[l][v].m, r = g[l][v].r, z = g[l][v].z, la = lr[v] * r;
      const float G = hf[v] + E[v], in = z * xf[v], gm = G * m;
      E[v] = a * G;
      ox[v] = gm * z;
      og[v] = gm * in * (1.f - z);
      // d log a of a h + m z x: a h - a^2 / m z x.  Times d log a / d gate = log a (1 - r), whose
      // log a / m has the limit 0 at m = 0 (no decay left in the type's range).
      const float lam = m > 0.f ? la * __builtin_amdgcn_rcpf(m) : 0.f;
      const float dla = G * a * (before[l][v] * la - a * in * lam);  // d log a times log a
      oa[v] = dla * (1.f - r);
      if (PLAIN || live) dlr[v] += dla;
      if (!PLAIN && !live) E[v] = ox[v] = oa[v] = og[v] = 0.f;
    }
    if (p.mine && (PLAIN || n < s.T)) {
      const int64_t at = token(s, n) * s.C + p.at;
      *reinterpret_cast<Raw*>(static_cast<T*>(d.dx) + at) = pack<T, V>(ox);
      *reinterpret_cast<Raw*>(static_cast<T*>(d.dga) + at) = pack<T, V>(oa);
      *reinterpret_cast<Raw*>(static_cast<T*>(d.dgx) + at) = pack<T, V>(og);
    }
    if (!PLAIN && ((c.begin >> l) & 1) && p.mine && d.dstate)
#pragma unroll
      for (int v = 0; v < V; ++v) d.dstate[b * s.C + p.at + v] = E[v];
  }
}

template <typename T>
__global__ __launch_bounds__(64 * kWaves, 6) void scan_bwd_out(const Scan s, const Grad d, int64_t chunks,
                                                               const float* __restrict__ carry,
                                                               const float* __restrict__ carry_e) {
  constexpr int V = 1;
  __shared__ Maps<V> maps, back;
  __shared__ float sum[kWaves][64 * V];
  const Place p = place<V>(s);
  Rows<T, V> x, ga, gx, dh;
  x.load(s.x, s.x_st, s, p.n0, p.at);
  ga.load(s.ga, s.ga_st, s, p.n0, p.at);
  gx.load(s.gx, s.gx_st, s, p.n0, p.at);
  if (d.dh) dh.load(d.dh, s.C, s, p.n0, p.at);
  const Stretch c = look(s, p.n0);
  float lr[V], A[V], H[V], B[V], E[V], state[V], dlr[V] = {}, fb[kLen][V];
  Gates g[kLen][V];
  share_rates(s, p, lr);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    A[v] = B[v] = 1.f;
    H[v] = E[v] = 0.f;
  }
  const bool plain = c.plain();
  terms(x, ga, gx, lr, g, fb);
  if (plain) {
    steps<true>(s, c, p, g, fb, A, H);
    back_steps<true>(s, d, c, p, dh, g, B, E);
  } else {
    steps<false>(s, c, p, g, fb, A, H);
    back_steps<false>(s, d, c, p, dh, g, B, E);
  }
  maps.put(p.wave, A, H);
  back.put(p.wave, B, E);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    state[v] = chunks > 1 ? carry[chunk_place(p.chunk, chunks, p.at + v)] : 0.f;
    E[v] = chunks > 1 ? carry_e[chunk_place(p.chunk, chunks, p.at + v)] : 0.f;
  }
  __syncthreads();
  maps.run(0, p.wave, state);
  back.run(kWaves, p.wave + 1, E);
#pragma unroll
  for (int l = 0; l < kLen; ++l) {  // fb becomes the state ahead of the token
    const bool begin = (c.begin >> l) & 1, live = (c.live >> l) & 1;
    const int64_t b = begin ? seq_at(c, l) : 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (begin) state[v] = s.state ? s.state[b * s.C + p.at + v] : 0.f;
      const float now = live ? fmaf(g[l][v].a, state[v], fb[l][v]) : 0.f;
      fb[l][v] = state[v];
      state[v] = now;
    }
  }
  if (plain) back_out<true>(s, d, c, p, x, dh, lr, g, fb, E, dlr);
  else back_out<false>(s, d, c, p, x, dh, lr, g, fb, E, dlr);
#pragma unroll
  for (int v = 0; v < V; ++v) sum[p.wave][lane_id() * V + v] = dlr[v];
  __syncthreads();
  if (p.wave == 0 && p.mine) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float y = dlr[v];
      for (int w = 1; w < kWaves; ++w) y += sum[w][lane_id() * V + v];
      d.ddecay[chunk_place(p.chunk, chunks, p.at + v)] = y;
    }
  }
  pass_empty(s, p, chunks, V, d.dlast, d.dstate);
}

// The chunks' sums of d log a times log a, added in their order; d log a / d decay = log a times
// sigmoid(decay) / softplus(decay).
__global__ __launch_bounds__(kCarryChannels * kRuns) void scan_bwd_decay(const float* __restrict__ part, int64_t chunks,
                                                                         int64_t C, const float* __restrict__ decay,
                                                                         float* __restrict__ out) {
  __shared__ float sum[kRuns][kCarryChannels];
  const int ch = threadIdx.x % kCarryChannels, run = threadIdx.x / kCarryChannels;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * kCarryChannels + ch;
  float x = 0.f;
  for (int64_t c = run; c < chunks; c += kRuns * 16) {
    float y[16];
#pragma unroll
    for (int n = 0; n < 16; ++n) y[n] = part[chunk_place(min(c + kRuns * n, chunks - 1), chunks, at)];
#pragma unroll
    for (int n = 0; n < 16; ++n) x += c + kRuns * n < chunks ? y[n] : 0.f;
  }
  sum[run][ch] = x;
  __syncthreads();
  if (run || at >= C) return;
  for (int n = 1; n < kRuns; ++n) x += sum[n][ch];
  const float y = decay[at];
  // sigmoid / softplus, near 1 where both are exp(y)
  const float ratio = y < -15.f ? 1.f - 0.5f * expf(y) : (y > 20.f ? 1.f / y : 1.f / (1.f + expf(-y)) / log1pf(expf(y)));
  out[at] = x * ratio;
}

// One token of each of B streams (s.ptr: their positions, or null), a thread for each lane's channels: 256 streams of 1024 channels in
// bfloat16 4.4 us, as long as a launch whose loads wait for one another once.
template <typename T, int V>
__global__ __launch_bounds__(256) void scan_step(const Scan s, float* __restrict__ state_out, T* __restrict__ h) {
  const int64_t per = s.C / V, n = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (n >= s.B * per) return;
  const int64_t b = n / per, at = n % per * V;
  using Raw = typename Pack<T, V>::Raw;
  float xf[V], af[V], gf[V], H[V];
  const int64_t position = s.ptr ? s.ptr[b] : 1;
  if (position < 0) {  // no token
#pragma unroll
    for (int v = 0; v < V; ++v) {
      H[v] = 0.f;
      state_out[b * s.C + at + v] = s.state[b * s.C + at + v];
    }
    *reinterpret_cast<Raw*>(h + b * s.C + at) = pack<T, V>(H);
    return;
  }
  unpack<T, V>(*reinterpret_cast<const Raw*>(static_cast<const T*>(s.x) + b * s.x_st + at), xf);
  unpack<T, V>(*reinterpret_cast<const Raw*>(static_cast<const T*>(s.ga) + b * s.ga_st + at), af);
  unpack<T, V>(*reinterpret_cast<const Raw*>(static_cast<const T*>(s.gx) + b * s.gx_st + at), gf);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const Gates g = gates(af[v], gf[v], log_rate(s.decay[at + v], s.rate));
    H[v] = fmaf(g.a, position ? s.state[b * s.C + at + v] : 0.f, g.m * g.z * xf[v]);
    state_out[b * s.C + at + v] = H[v];
  }
  *reinterpret_cast<Raw*>(h + b * s.C + at) = pack<T, V>(H);
}

// Packets of streams as sequences of a scan: each stream's tokens from position 0 on, and between the streams those at
// negative positions, whose states nobody takes.  The states ahead of the former are the streams', or 0 for
// those whose position 0 is in the packet.
__global__ __launch_bounds__(256) void scan_packets(const int64_t* __restrict__ ptr, const int64_t* __restrict__ start,
                                                    const float* __restrict__ state, int64_t state_st, int64_t B, int64_t C,
                                                    int64_t* __restrict__ parts, float* __restrict__ before) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < 2 * B) {
    const int64_t b = i / 2, begin = ptr[b], end = ptr[b + 1], at = start[b];
    parts[i] = i % 2 ? end : at >= 0 ? begin : at > begin - end ? begin - at : end;
  }
  if (i >= (2 * B - 1) * C) return;
  const int64_t row = i / C, b = row / 2, at = start[b];
  const bool goes_on = row % 2 == 0 && (at > 0 || at <= ptr[b] - ptr[b + 1]);
  before[i] = goes_on ? state[b * state_st + i % C] : 0.f;
}

// ---------------------------------------------------------------------- host ---

inline int64_t chunks_of(int64_t T) { return ceil_div(T, kChunk); }

inline int scan_args(const geo_recurrence_t* g, Scan* s) {
  GEO_REQUIRE(g, "gated recurrence: null arguments");
  GEO_REQUIRE(g->dtype == GEO_F32 || g->dtype == GEO_BF16 || g->dtype == GEO_F16, "gated recurrence: dtype code %d",
              static_cast<int>(g->dtype));
  GEO_REQUIRE(g->tokens >= 0 && g->tokens < (int64_t(1) << 31) - kChunk && g->channels >= 0 && g->sequences >= 1 &&
                  g->sequences < (int64_t(1) << 31) - 1, "gated recurrence: %lld tokens, %lld channels, %lld sequences",
              static_cast<long long>(g->tokens), static_cast<long long>(g->channels), static_cast<long long>(g->sequences));
  *s = Scan{g->x, g->gate_a, g->gate_x, g->x_token, g->gate_a_token, g->gate_x_token, g->decay, g->ptr, g->state,
            g->tokens, g->channels, g->sequences, g->rate, g->reverse};
  GEO_REQUIRE(g->tokens == 0 || g->channels == 0 || (g->x && g->gate_a && g->gate_x && g->decay), "gated recurrence: null tensor");
  GEO_REQUIRE(grid_fits(chunks_of(g->tokens) * ceil_div(g->channels, 64), 64 * kWaves), "gated recurrence: too many workgroups");
  return GEO_OK;
}

// Two 16-bit channels to a lane, half the loads, where every row begins on a multiple of 4 bytes and
// there are `least` elements.  Below that twice the waves are as good or better.  In bfloat16, us with
// two | one: forward of 2048 x 64 17.2 | 12.1, 8192 x 256 23.0 | 21.1, 65,536 x 256 66.6 | 71.7,
// 131,072 x 256 115.8 | 130.9, its backward's pass 1 34 | 46; step of 256 x 1024 4.8 | 4.2,
// 1024 x 4096 21.8 | 23.5.  Pass 2 of the backward holds too many values for two.
constexpr int64_t kPairsScan = int64_t(1) << 24, kPairsStep = int64_t(1) << 22;
inline bool in_pairs(const geo_recurrence_t& g, int64_t least) {
  auto even = [](const void* p, int64_t st) { return reinterpret_cast<uintptr_t>(p) % 4 == 0 && st % 2 == 0; };
  return g.dtype != GEO_F32 && g.tokens * g.channels >= least && g.channels % 2 == 0 && even(g.x, g.x_token) &&
         even(g.gate_a, g.gate_a_token) && even(g.gate_x, g.gate_x_token);
}

template <typename T, int V>
int forward(const Scan& s, void* h, float* last, float* carry, float2* map, hipStream_t stream) {
  const int64_t chunks = chunks_of(s.T), blocks = ceil_div(s.C, 64 * V);
  const dim3 grid(static_cast<uint32_t>(chunks * blocks));
  if (chunks > 1) {
    scan_map<T, V><<<grid, dim3(64 * kWaves), 0, stream>>>(s, chunks, map);
    GEO_LAUNCH_CHECK("scan_map");
  }
  if (chunks > kFew) {
    scan_carry<<<dim3(static_cast<uint32_t>(padded(s.C) / kCarryChannels)), dim3(kCarryChannels * kRuns), 0, stream>>>(map, carry, chunks, 0);
    GEO_LAUNCH_CHECK("scan_carry");
  }
  scan_out<T, V><<<grid, dim3(64 * kWaves), 0, stream>>>(s, chunks, map, carry, static_cast<T*>(h), last);
  GEO_LAUNCH_CHECK("scan_out");
  return GEO_OK;
}

template <typename T, int V>
int backward(const Scan& s, const Grad& d, const float* carry, float* carry_e, float2* map, float* ddecay, hipStream_t stream) {
  const int64_t chunks = chunks_of(s.T), blocks = ceil_div(s.C, 64);
  const dim3 across(static_cast<uint32_t>(padded(s.C) / kCarryChannels));
  if (chunks > 1) {
    scan_bwd_map<T, V><<<dim3(static_cast<uint32_t>(chunks * ceil_div(s.C, 64 * V))), dim3(64 * kWaves), 0, stream>>>(s, d, chunks, map);
    GEO_LAUNCH_CHECK("scan_bwd_map");
    scan_carry<<<across, dim3(kCarryChannels * kRuns), 0, stream>>>(map, carry_e, chunks, 1);
    GEO_LAUNCH_CHECK("scan_carry");
  }
  scan_bwd_out<T><<<dim3(static_cast<uint32_t>(chunks * blocks)), dim3(64 * kWaves), 0, stream>>>(s, d, chunks, carry, carry_e);
  GEO_LAUNCH_CHECK("scan_bwd_out");
  scan_bwd_decay<<<across, dim3(kCarryChannels * kRuns), 0, stream>>>(d.ddecay, chunks, s.C, s.decay, ddecay);
  GEO_LAUNCH_CHECK("scan_bwd_decay");
  return GEO_OK;
}

}  // namespace rec
}  // namespace geo

#define GEO_REC_CALL(F, pairs, ...)                                                              \
  (g->dtype == GEO_F32    ? geo::rec::F<float, 1>(__VA_ARGS__)                                   \
   : g->dtype == GEO_BF16 ? (pairs ? geo::rec::F<__bf16, 2>(__VA_ARGS__) : geo::rec::F<__bf16, 1>(__VA_ARGS__)) \
                          : (pairs ? geo::rec::F<_Float16, 2>(__VA_ARGS__) : geo::rec::F<_Float16, 1>(__VA_ARGS__)))

extern "C" int64_t geo_recurrence_carry_size(int64_t tokens, int64_t channels) {
  return tokens < 1 || channels < 1 ? 0 : geo::rec::chunks_of(tokens) * geo::rec::padded(channels);
}

extern "C" int geo_recurrence_fwd(const geo_recurrence_t* g, void* h, float* last, float* carry, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  geo::rec::Scan s;
  const int rc = geo::rec::scan_args(g, &s);
  if (rc != GEO_OK || s.T == 0 || s.C == 0) return rc;
  GEO_REQUIRE(h && last && carry, "gated recurrence: null output");
  const size_t need = static_cast<size_t>(geo_recurrence_carry_size(s.T, s.C)) * sizeof(float2);
  if (!workspace || workspace_bytes < need)
    return geo::set_error(GEO_ERR_WORKSPACE, "gated recurrence: workspace of %zu bytes, %zu needed",
                          workspace ? workspace_bytes : size_t(0), need);
  // half a block of channels would leave half the lanes idle
  const bool pairs = s.C % 128 == 0 && geo::rec::in_pairs(*g, geo::rec::kPairsScan) && reinterpret_cast<uintptr_t>(h) % 4 == 0;
  return GEO_REC_CALL(forward, pairs, s, h, last, carry, static_cast<float2*>(workspace), geo::as_stream(stream));
}

extern "C" size_t geo_recurrence_bwd_workspace_bytes(int64_t tokens, int64_t channels) {
  return static_cast<size_t>(geo_recurrence_carry_size(tokens, channels)) * 4 * sizeof(float);
}

extern "C" int geo_recurrence_bwd(const geo_recurrence_t* g, const float* carry, const void* dh, const float* dlast, void* dx,
                                  void* dgate_a, void* dgate_x, float* ddecay, float* dstate, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  geo::rec::Scan s;
  const int rc = geo::rec::scan_args(g, &s);
  if (rc != GEO_OK || s.T == 0 || s.C == 0) return rc;
  GEO_REQUIRE(carry && dx && dgate_a && dgate_x && ddecay, "gated recurrence backward: null tensor");
  const size_t need = geo_recurrence_bwd_workspace_bytes(s.T, s.C);
  if (!workspace || workspace_bytes < need)
    return geo::set_error(GEO_ERR_WORKSPACE, "gated recurrence backward: workspace of %zu bytes, %zu needed",
                          workspace ? workspace_bytes : size_t(0), need);
  const int64_t n = geo_recurrence_carry_size(s.T, s.C);
  float* w = static_cast<float*>(workspace);  // maps, states, sums
  const geo::rec::Grad d{dh, dlast, dx, dgate_a, dgate_x, dstate, w + 3 * n};
  const bool pairs = s.C % 128 == 0 && geo::rec::in_pairs(*g, geo::rec::kPairsScan) && reinterpret_cast<uintptr_t>(dh) % 4 == 0;
  return GEO_REC_CALL(backward, pairs, s, d, carry, w + 2 * n, reinterpret_cast<float2*>(w), ddecay, geo::as_stream(stream));
}

namespace geo {
namespace rec {
template <typename T, int V>
int step(const Scan& s, float* state_out, void* h, hipStream_t stream) {
  const int64_t blocks = ceil_div(s.B * (s.C / V), 256);
  GEO_REQUIRE(grid_fits(blocks, 256), "gated recurrence step: too many workgroups");
  scan_step<T, V><<<dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, stream>>>(s, state_out, static_cast<T*>(h));
  GEO_LAUNCH_CHECK("scan_step");
  return GEO_OK;
}
}  // namespace rec
}  // namespace geo

extern "C" int geo_recurrence_packets(const int64_t* ptr, const int64_t* start, const float* state, int64_t state_stream, int64_t streams,
                                      int64_t channels, int64_t* parts, float* before, void* stream) {
  using namespace geo;
  GEO_REQUIRE(streams >= 1 && streams < (int64_t(1) << 30) && channels >= 0 && channels < (int64_t(1) << 31),
              "gated recurrence packets: %lld streams of %lld channels", static_cast<long long>(streams), static_cast<long long>(channels));
  GEO_REQUIRE(ptr && start && parts && (channels == 0 || (state && before)), "gated recurrence packets: null tensor");
  const int64_t rows = 2 * streams - 1, blocks = ceil_div(rows * channels > 2 * streams ? rows * channels : 2 * streams, int64_t(256));
  GEO_REQUIRE(grid_fits(blocks, 256), "gated recurrence packets: too many workgroups");
  rec::scan_packets<<<dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, as_stream(stream)>>>(ptr, start, state, state_stream, streams, channels,
                                                                                             parts, before);
  GEO_LAUNCH_CHECK("scan_packets");
  return GEO_OK;
}

extern "C" int geo_recurrence_step(const geo_recurrence_t* g, float* state_out, void* h, void* stream) {
  geo::rec::Scan s;
  const int rc = geo::rec::scan_args(g, &s);
  if (rc != GEO_OK || s.T == 0 || s.C == 0) return rc;
  GEO_REQUIRE(g->sequences == g->tokens, "gated recurrence step: one token for each of %lld streams, got %lld",
              static_cast<long long>(g->sequences), static_cast<long long>(g->tokens));
  GEO_REQUIRE(s.state && state_out && h, "gated recurrence step: null tensor");
  const bool pairs = geo::rec::in_pairs(*g, geo::rec::kPairsStep) && reinterpret_cast<uintptr_t>(h) % 4 == 0;
  return GEO_REC_CALL(step, pairs, s, state_out, h, geo::as_stream(stream));
}
