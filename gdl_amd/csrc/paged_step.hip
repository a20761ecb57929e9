// paged_step.hip — attention of one new token per stream over its pages, split over the stream's
// length and joined.
//
// Sᵀ = K Qᵀ and Oᵀ = Vᵀ Pᵀ on 16x16 matrix instructions, 16 query heads of a key head as the columns.  A
// lane holds column lane % 16 and, of every product's inner dimension, the part of its group lane / 16.
// A block is the blk tokens that 64 bytes hold; a group owns a quarter of them, 16 bytes of each row of Vᵀ.
// The rows of Sᵀ are dealt out so that a group's results are just its own tokens: weights become the second
// product's operand without leaving their lane, and both operands from memory are read 16 bytes a lane,
// straight into the registers that the instructions take.  Nothing goes through LDS but the join.
//
// The work is the reading of the histories.  16 heads of 128 behind a key head of 16-bit values are 16 operations a byte,
// far under what the matrix units do, and tiles of 16 columns cost the same for one head.  Shares are equal numbers of
// 64-token tiles for as many workgroups as run at a time (two to four times as many were slower).  Of 6.3 TB/s that a kernel can read here: 64 streams to 16,384 tokens, 16 (4) heads of 128, bfloat16,
// 252 us and 5 for the join, 5.6 TB/s; 128 in int8 with a bias 277 + 5 us, 5.2 TB/s (vector instructions in 50% of the cycles,
// for codes to bfloat16, scales and weights); one of 131,072 tokens 16 + 7 us.  The least call takes 7-8 us.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

#include "paged.hpp"

namespace geo {
namespace paged {

using f32x4 = float __attribute__((ext_vector_type(4)));

struct Step {
  Pool pool;
  const void *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  const int64_t* pos;
  attn::Bias bias;
  int B, Hq;
  float scale;
};

constexpr int kCols = 16;

// Workgroups of the kernel on a CU, by the registers that it takes.
constexpr int kMostWaves = 4;
template <typename T, typename C, int DP>
constexpr int step_waves() {
  if (DP == 128) return 2;
  return !Code<C>::kNarrow ? kMostWaves : sizeof(T) == 4 ? 2 : 3;
}

// --- operands ---

__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// The queries of a column in operand order: LOADS pieces of the 64 bytes of a pool row each.
template <typename T, typename C, int LOADS>
struct Query {  // pools in the queries' type: the pieces themselves
  Bytes16 x[LOADS];
  __device__ __forceinline__ void load(const T* q, int g, int D) {
#pragma unroll
    for (int c = 0; c < LOADS; ++c) {
      const int d = (c * 64 + g * 16) / static_cast<int>(sizeof(T));
      x[c].u = d < D ? *reinterpret_cast<const uint4*>(q + d) : uint4{};
    }
  }
  __device__ __forceinline__ void ready() {}
  __device__ __forceinline__ f32x4 times(int c, const Bytes16& k, f32x4 s) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s = mma(k.f[e], x[c].f[e], s);
    } else if constexpr (__is_same(T, __bf16)) {
      s = mma(k.b, x[c].b, s);
    } else {
      s = mma(k.h, x[c].h, s);
    }
    return s;
  }
};
template <typename T, typename C, int LOADS>
struct NarrowQuery {  // 8-bit pools
  static constexpr int kParts = parts_of<T>();
  union Raw {
    uint4 u[sizeof(T) / 2];
    T t[8];
  } raw[LOADS][2];
  bf16x8 x[LOADS][2][kParts];
  __device__ __forceinline__ void load(const T* q, int g, int D) {
#pragma unroll
    for (int c = 0; c < LOADS; ++c)
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int n = 0; n < static_cast<int>(sizeof(T) / 2); ++n) {
          const int d = c * 64 + g * 16 + 8 * half;
          raw[c][half].u[n] = d < D ? reinterpret_cast<const uint4*>(q + d)[n] : uint4{};
        }
  }
  __device__ __forceinline__ void ready() {
#pragma unroll
    for (int c = 0; c < LOADS; ++c)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = static_cast<float>(raw[c][half].t[e]);
        split8<kParts>(y, x[c][half]);
      }
  }
  __device__ __forceinline__ f32x4 times(int c, const Bytes16& k, f32x4 s) const {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const bf16x8 a = decode8<C>(k.w[2 * half], k.w[2 * half + 1]);
#pragma unroll
      for (int n = 0; n < kParts; ++n) s = mma(a, x[c][half][n], s);
    }
    return s;
  }
};

// The weights of a group's tokens as the second product's operand, 16-bit ones in two parts: rounded once they would add
// an error as large as the output's own rounding, and the reading of the values leaves the time for it.
template <typename T, typename C>
struct Weights {
  static constexpr int kParts = sizeof(T) == 4 ? 1 : 2;
  using F = typename std::conditional<__is_same(T, __bf16), bf16x8, f16x8>::type;
  float f[4];
  F x[kParts];
  __device__ __forceinline__ void from(const float (&p)[16 / sizeof(T)]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = p[e];
    } else {
      split8<kParts>(p, x);
    }
  }
  __device__ __forceinline__ f32x4 times(const Bytes16& v, f32x4 o) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 4; ++e) o = mma(v.f[e], f[e], o);
    } else {
#pragma unroll
      for (int n = 0; n < kParts; ++n) {
        if constexpr (__is_same(T, __bf16)) o = mma(v.b, x[n], o);
        else o = mma(v.h, x[n], o);
      }
    }
    return o;
  }
  // what the parts leave of float16 weights (Faint)
  static __device__ __forceinline__ bool some_faint(const float (&p)[16 / sizeof(T)]) {
    bool some = false;
#pragma unroll
    for (int e = 0; e < static_cast<int>(16 / sizeof(T)); ++e) some |= p[e] < Faint<T>::below(kParts) && p[e] > 0.f;
    return some;
  }
  static __device__ __forceinline__ f32x4 faint(const Bytes16& v, const f16x8& rest, f32x4 o) {
    return mma(v.h, rest, o * Faint<T>::kUp) * Faint<T>::kDown;
  }
};
template <typename T, typename C>
struct NarrowWeights {
  static constexpr int kParts = sizeof(T) == 4 ? 3 : 2;
  bf16x8 x[2][kParts];
  __device__ __forceinline__ void from(const float* p) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = p[8 * half + e];
      split8<kParts>(y, x[half]);
    }
  }
  __device__ __forceinline__ f32x4 times(const Bytes16& v, f32x4 o) const {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const bf16x8 a = decode8<C>(v.w[2 * half], v.w[2 * half + 1]);
#pragma unroll
      for (int n = 0; n < kParts; ++n) o = mma(a, x[half][n], o);
    }
    return o;
  }
};

// x times log2 e for a key `back` tokens behind, of head h.
__device__ __forceinline__ float bias_at(const attn::Bias& b, int Hq, int h, int64_t back) {
  const int n = static_cast<int>(min(back, static_cast<int64_t>(b.maxd)));
  return attn::bias_value(b, static_cast<int64_t>(b.lut[b.maxd - n]) * Hq + h);
}

// Over 16 lanes, in all of them.
__device__ __forceinline__ float group_sum(float x) {
  x += __uint_as_float(dpp_u32<kDppXor1>(__float_as_uint(x)));
  x += __uint_as_float(dpp_u32<kDppXor2>(__float_as_uint(x)));
  x += __uint_as_float(dpp_u32<kDppHalfMirror>(__float_as_uint(x)));
  return x + __uint_as_float(dpp_u32<kDppMirror>(__float_as_uint(x)));
}

// A row of DP values, 16 lanes to a row, DP / 16 adjoining ones each: as it comes, and as the pool keeps it.
template <typename T, int DP>
struct Raw {
  T x[DP / 16];
  __device__ __forceinline__ void load(const T* row, int e, int D) {
    struct alignas(DP / 16 * sizeof(T) < 16 ? DP / 16 * sizeof(T) : 16) Piece { T x[DP / 16]; };
    if (DP / 16 * e < D) {
      const Piece p = reinterpret_cast<const Piece*>(row)[e];
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) x[n] = p.x[n];
    } else {
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) x[n] = static_cast<T>(0.f);
    }
  }
};
template <typename T, typename C, int DP>
struct NewRow {
  struct alignas(DP / 16 * sizeof(C) < 16 ? DP / 16 * sizeof(C) : 16) Piece { C c[DP / 16]; } kept;
  float value[DP / 16], scale;
  __device__ __forceinline__ void from(const Raw<T, DP>& raw) {
    uint32_t most = 0;
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) {
      value[n] = static_cast<float>(raw.x[n]);
      most = max(most, __float_as_uint(value[n]) & 0x7fffffffu);
    }
    scale = 1.f;
    if constexpr (Code<C>::kNarrow) {
      const RowScale s = row_scale<C>(group_most<16>(most));
      scale = s.scale;
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
        kept.c[n].bits = Code<C>::bits(encode<C>(value[n], s.rate));
        value[n] = Code<C>::value(kept.c[n].bits) * s.scale;
      }
    } else {
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) kept.c[n] = raw.x[n];
    }
  }
};

// How the work is dealt out.  A row is a stream, a key head and up to 16 of its query heads; its work is the
// 64-token tiles that the stream holds, at least one.  The tiles of all rows, in a row, are cut into equal
// shares, one for each of `groups` workgroups, which are as many as the card runs at a time: lengths are
// read on the device, so streams of any ages fill it evenly.  A share of `least` tiles is worth a workgroup.
// Without `parts` a workgroup takes a whole row.
struct Deal {
  int groups, least;
  int by_row;    // desc has a place for each row, else for each workgroup (whichever are fewer)
  // the row, or the last one that begins in the workgroup: how many shares have a part of it (0: it is whole) and,
  // 16 bits up, its heads; the first of these; its output row
  int4* desc;
  float* parts;  // by workgroup: what it adds to the row that it begins with, and to the one that it ends with
};
constexpr int kTile = 64;

__device__ __forceinline__ int tiles_at(int64_t p, int room) {
  return max(1, static_cast<int>((min(max(p, int64_t(0)), static_cast<int64_t>(room)) + kTile - 1) / kTile));
}
__device__ __forceinline__ int64_t scalar(int64_t x) { return static_cast<int64_t>(attn::uniform(static_cast<uint64_t>(x))); }
// Quotients of whole numbers below 2^52, in a tenth of a 64-bit division's instructions.
__device__ __forceinline__ int64_t quotient(int64_t x, int64_t by) {
  int64_t q = static_cast<int64_t>(static_cast<double>(x) / static_cast<double>(by));
  const int64_t rest = x - q * by;
  q += rest < 0 ? -1 : rest >= by ? 1 : 0;
  return scalar(q);
}
__device__ __forceinline__ int64_t wave_sum64(int64_t x) {
#pragma unroll
  for (int n = 1; n < 64; n *= 2) x += __shfl_xor(x, n, 64);
  return x;
}

// One workgroup: a share.  The part of a row goes to its four or eight waves in equal pieces.  The new token is no part of
// that: who has the row's beginning forms its row as the pool keeps it, writes it, and adds it to the join, so
// that no read waits for the write.
template <typename T, typename C, int DP, int WAVES>
__global__ __launch_bounds__(64 * WAVES, (WAVES == 4 ? step_waves<T, C, DP>() : 2)) void paged_step(const Step a, const Deal deal, const int32_t* __restrict__ table,
                                                                        const int64_t* __restrict__ positions, T* __restrict__ out) {
  constexpr bool kNarrow = Code<C>::kNarrow, kHalf = Faint<C>::kHalf;
  constexpr float kLift = Faint<C>::kLift, kLazy = Faint<C>::kLazy;
  constexpr int kWaves = WAVES, kThreads = 64 * WAVES, kCells = kCols * 4 / WAVES;  // heads that there is room to join
  constexpr int kSize = sizeof(C), kBlk = block_tokens<C>(), kOwn = kBlk / 4, kTiles = kBlk / 16;
  constexpr int kLoads = DP * kSize / 64, kRows = DP / 16, kLds = DP + 4;
  using Q = typename std::conditional<kNarrow, NarrowQuery<T, C, kLoads>, Query<T, C, kLoads>>::type;
  using W = typename std::conditional<kNarrow, NarrowWeights<T, C>, Weights<T, C>>::type;
  __shared__ float sm[kWaves + 1][kCells], sl[kWaves + 1][kCells], fresh[DP];
  __shared__ __attribute__((aligned(16))) float so[kWaves][kCells][kLds];
  extern __shared__ float sbias[];  // with a bias: [buckets][kCols], the row's heads; then the bucket of each distance back, a byte each
  const Pool& pool = a.pool;
  const int D = pool.D, group = a.Hq / pool.Hk, chunks = (group + kCols - 1) / kCols, room = pool.columns * pool.page;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int per_stream = pool.Hk * chunks;  // rows

  uint8_t* const bucket = reinterpret_cast<uint8_t*>(sbias + a.bias.buckets * kCols);
  if (a.bias.table)
    for (int x = threadIdx.x; x <= a.bias.maxd; x += kThreads) bucket[x] = static_cast<uint8_t>(a.bias.lut[a.bias.maxd - x]);

  // the share u .. end of all tiles, and where it begins: stream, row of the stream, tile
  int b, r, t0;
  int64_t u = 0, end, share = 0, before = 0;  // before: tiles ahead of the stream's
  int64_t p;
  if (deal.parts) {
    const int lane = threadIdx.x & 63;
    int64_t total = 0;
    for (int i = lane; i < a.B; i += 64) total += tiles_at(positions[i], room);
    total = scalar(wave_sum64(total)) * per_stream;
    share = max(quotient(total + deal.groups - 1, deal.groups), static_cast<int64_t>(deal.least));
    u = blockIdx.x * share;
    end = min(u + share, total);
    if (threadIdx.x == 0 && !deal.by_row) deal.desc[blockIdx.x] = int4{0, 0, 0, 0};
    if (u >= end) return;
    const int64_t at = quotient(u, per_stream);  // the stream is the one with this tile of all streams'
    for (b = 0;; b += 64) {
      const int i = b + lane, n = i < a.B ? tiles_at(positions[i], room) : 0;
      int64_t upto = n;
#pragma unroll
      for (int k = 1; k < 64; k *= 2) {
        const int64_t x = __shfl_up(upto, k, 64);
        if (lane >= k) upto += x;
      }
      const uint64_t past = __ballot(before + upto > at);
      if (past) {
        const int k = __builtin_ctzll(past);
        b += k;
        before += scalar(__shfl(upto - n, k, 64));
        break;
      }
      before += scalar(__shfl(upto, 63, 64));
    }
    b = __builtin_amdgcn_readfirstlane(b);
    p = positions[b];
    const int64_t in = u - before * per_stream, n = tiles_at(p, room);
    r = static_cast<int>(quotient(in, n));
    t0 = static_cast<int>(in - r * n);
  } else {
    b = static_cast<int>(blockIdx.x / per_stream);
    r = static_cast<int>(blockIdx.x % per_stream);
    t0 = 0;
    p = positions[b];
    end = int64_t(1) << 40;
  }
  for (bool again = false;; again = true) {
  uint32_t thread = threadIdx.x;
  asm volatile("" : "+v"(thread));  // keeps what is formed from it in the row's part: ahead of them all it takes the registers
  const int lane = thread & 63, g = lane >> 4, col = lane & 15;
  // what does not depend on the stream's length is asked for first: the queries as an operand, and for the end
  // the new token's rows and the queries again, 16 lanes to a head
  const int gc = r % chunks, hk = r / chunks;
  const int heads = min(kCols, group - gc * kCols), h0 = hk * group + gc * kCols;
  const int head = h0 + min(col, heads - 1), cell = thread >> 4;
  const bool begins = t0 == 0;
  Q q;
  q.load(static_cast<const T*>(a.q) + b * a.q_st + head * a.q_sh, g, D);
  Raw<T, DP> kraw, vraw, qraw;
  if (begins) {
    kraw.load(static_cast<const T*>(a.k) + b * a.k_st + hk * a.k_sh, col, D);
    vraw.load(static_cast<const T*>(a.v) + b * a.v_st + hk * a.v_sh, col, D);
    qraw.load(static_cast<const T*>(a.q) + b * a.q_st + (h0 + min(cell, heads - 1)) * a.q_sh, col, D);
  }
  if (again) __syncthreads();  // the waves are done with the LDS of the row before
  const int tiles = tiles_at(p, room);
  const int t1 = static_cast<int>(min(static_cast<int64_t>(tiles), t0 + (end - u)));
  const bool ends = t1 == tiles;
  const int held = static_cast<int>(min(max(p, int64_t(0)), static_cast<int64_t>(room)));  // tokens before the new one
  const int s0 = t0 * kTile, s1 = min(held, t1 * kTile);
  const int piece = ((s1 - s0 + kWaves - 1) / kWaves + kBlk - 1) / kBlk * kBlk;
  const int w0 = s0 + wave * piece, w1 = min(s1, w0 + piece);

  // where the wave reads: a column of the table and a place in its page
  const int32_t* const row = table + b * pool.table_st;
  int column = w0 / pool.page, off = w0 - column * pool.page;
  bool bad = false;
  int at = 0, next = 0;
  auto entry = [&](int n) { return __builtin_amdgcn_readfirstlane(row[min(n, pool.columns - 1)]); };
  auto page_here = [&]() {  // the entry behind it is on its way while this page is read
    at = next;
    next = entry(column + 1);
    if (static_cast<uint32_t>(at) >= static_cast<uint32_t>(pool.pages)) {
      bad = true;
      at = 0;
    }
  };
  if (w0 < w1) {
    next = entry(column);
    page_here();
  }
  // the new token's place; `room`: beyond the table
  const int pi = static_cast<int>(min(p, static_cast<int64_t>(room))), new_column = pi / pool.page, place = pi - new_column * pool.page;
  int page = begins && p >= 0 && new_column < pool.columns ? entry(new_column) : -1;

  // this lane's places in a block: row 4 g' + i of tile n is token g' kOwn + 4 n + i
  uint32_t kat[kLoads];
  bool idle[kLoads];
#pragma unroll
  for (int c = 0; c < kLoads; ++c) {
    idle[c] = (c * 64 + g * 16) / kSize >= D;  // past the head: read the row's first values instead and count them as zeros
    kat[c] = ((col >> 2) * kOwn + (col & 3)) * D * kSize + (idle[c] ? 0 : c * 64 + g * 16);
  }
  const bool some_idle = D < DP;
  // dimension 16 m + col of the values; past the head, rows that are not kept, any does
  const uint32_t vat = col * 64 + g * 16, vat_edge = (col & 7) * 64 + g * 16;
  Bytes16 kx[kTiles][kLoads], vx[kRows];
  float ksx = 0.f, vsx = 0.f;  // the scales of the group's token `col`
  auto load_k = [&](int page, int place) {
    const int64_t slot0 = (static_cast<int64_t>(page) * pool.Hk + hk) * pool.page + place;
    const char* const base = pool.k + slot0 * D * kSize;
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int c = 0; c < kLoads; ++c) kx[n][c].u = *reinterpret_cast<const uint4*>(base + n * 4 * D * kSize + kat[c]);
    if constexpr (kNarrow) ksx = pool.ks[slot0 + lane];
  };
  auto load_v = [&](int page, int place) {
    const int64_t slot0 = (static_cast<int64_t>(page) * pool.Hk + hk) * pool.page + place;
    const char* const base = pool.v + slot0 * D * kSize;
#pragma unroll
    for (int m = 0; m < kRows; ++m)
      vx[m].u = *reinterpret_cast<const uint4*>(base + (16 * m < D ? m * 1024 : 0) + (16 * m + 16 <= D ? vat : vat_edge));
    if constexpr (kNarrow) vsx = pool.vs[slot0 + lane];
  };
  if (w0 < w1) {
    load_k(at, off);
    load_v(at, off);
  }

  q.ready();
  const bool near = a.bias.table && (t1 * kTile > p - a.bias.maxd || begins);  // distances with a bias of their own, the new token's
  if (near) {
    for (int x = thread; x < a.bias.buckets * kCols; x += kThreads)
      sbias[x] = attn::bias_value(a.bias, static_cast<int64_t>(x / kCols) * a.Hq + h0 + min(x % kCols, heads - 1));
    __syncthreads();
  }
  f32x4 o[kRows];
#pragma unroll
  for (int m = 0; m < kRows; ++m) o[m] = f32x4{};
  float top = -kInf, sum = 0.f;  // what scores are taken less by (Faint)
  const float scale2 = a.scale * kLog2e;
  const float far = a.bias.table ? bias_at(a.bias, a.Hq, head, a.bias.maxd) : 0.f;

  for (int t = w0; t < w1; t += kBlk) {
    if (some_idle) {
#pragma unroll
      for (int c = 0; c < kLoads; ++c)
        if (idle[c]) {
#pragma unroll
          for (int n = 0; n < kTiles; ++n) kx[n][c].u = uint4{};
        }
    }
    float x[kOwn];
#pragma unroll
    for (int n = 0; n < kTiles; ++n) {
      f32x4 s = {};
#pragma unroll
      for (int c = 0; c < kLoads; ++c) s = q.times(c, kx[n][c], s);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * n + i] = s[i] * scale2;
      if constexpr (kNarrow) __builtin_amdgcn_sched_barrier(0);  // decode a tile at a time: all at once take the registers
    }
    if constexpr (kNarrow) by_group(x, ksx);
    // the next block's keys are on their way while this one's weights are formed
    const bool more = t + kBlk < w1;
    if (more) {
      off += kBlk;
      if (off == pool.page) {
        off = 0;
        ++column;
        page_here();
      }
      load_k(at, off);
    }
    if (a.bias.table) {
      if (p - (t + kBlk - 1) < a.bias.maxd) {
#pragma unroll
        for (int n = 0; n < kOwn; ++n) {
          const int back = static_cast<int>(min(max(p - (t + g * kOwn + n), int64_t(0)), static_cast<int64_t>(a.bias.maxd)));
          x[n] += sbias[bucket[back] * kCols + col];
        }
      } else {
#pragma unroll
        for (int n = 0; n < kOwn; ++n) x[n] += far;
      }
    }
    if (t + kBlk > s1) {  // the block behind the last token: what it holds may be anything
      const int in = s1 - (t + g * kOwn);
#pragma unroll
      for (int n = 0; n < kOwn; ++n)
        if (n >= in) x[n] = -kInf;
      uint32_t keep[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int bits = 8 * kSize * in - 32 * n;
        keep[n] = bits >= 32 ? ~0u : bits <= 0 ? 0u : (1u << bits) - 1;
      }
#pragma unroll
      for (int m = 0; m < kRows; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n) vx[m].w[n] &= keep[n];
      if constexpr (kNarrow) vsx = col < in ? vsx : 0.f;
    }
    float most = x[0];
#pragma unroll
    for (int n = 1; n < kOwn; ++n) most = fmaxf(most, x[n]);
    if (__any(most - top > kLazy + kLift)) {
      most = fmaxf(most, __shfl_xor(most, 16, 64));
      most = fmaxf(Faint<C>::lifted(fmaxf(most, __shfl_xor(most, 32, 64))), top);
      const float keep = top == -kInf ? 0.f : exp2_hw(top - most);
      if (top != -kInf) {
#pragma unroll
        for (int m = 0; m < kRows; ++m) o[m] *= keep;
        sum *= keep;
      }
      top = most;
    }
    const float shift = top == -kInf ? 0.f : top;
#pragma unroll
    for (int n = 0; n < kOwn; ++n) {
      x[n] = exp2_hw(x[n] - shift);
      sum += x[n];
    }
    if constexpr (kNarrow) by_group(x, vsx);
    W weights;
    weights.from(x);
#pragma unroll
    for (int m = 0; m < kRows; ++m) {
      o[m] = weights.times(vx[m], o[m]);
      if constexpr (kNarrow) __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kHalf) {
      if (__any(W::some_faint(x))) {
        const f16x8 rest = faint8<W::kParts>(x);
#pragma unroll
        for (int m = 0; m < kRows; ++m) o[m] = W::faint(vx[m], rest, o[m]);
      }
    }
    if (more) load_v(at, off);
  }

  sum += __shfl_xor(sum, 16, 64);
  sum += __shfl_xor(sum, 32, 64);
  if (g == 0 && col < kCells) {
    sm[wave][col] = top;
    sl[wave][col] = bad ? __builtin_nanf("") : sum;
  }
  if (col < kCells) {
#pragma unroll
    for (int m = 0; m < kRows; ++m) *reinterpret_cast<f32x4*>(&so[wave][col][16 * m + 4 * g]) = o[m];
  }

  if (begins && p >= 0) {
    NewRow<T, C, DP> nk, nv;
    nk.from(kraw);
    nv.from(vraw);
    float s = 0.f;
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) s = fmaf(static_cast<float>(qraw.x[n]), nk.value[n], s);
    s = group_sum(s) * scale2;
    if (a.bias.table) s += sbias[bucket[0] * kCols + min(cell, kCols - 1)];
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(pool.pages)) page = -1;
    if (col == 0 && cell < kCells) {
      sm[kWaves][cell] = s;
      sl[kWaves][cell] = page < 0 ? __builtin_nanf("") : 1.f;
    }
    if (cell == 0) {
      const int64_t slot0 = (static_cast<int64_t>(max(page, 0)) * pool.Hk + hk) * pool.page;
      const int d0 = DP / 16 * col;
      const bool kept = gc == 0 && page >= 0 && d0 < D;
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) fresh[d0 + n] = nv.value[n];
      if (kept) {
        C* const vp = reinterpret_cast<C*>(pool.v) + slot0 * D + place / kBlk * (kBlk * D) + place % kBlk;
        *reinterpret_cast<typename NewRow<T, C, DP>::Piece*>(reinterpret_cast<C*>(pool.k) + (slot0 + place) * D + d0) = nk.kept;
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) vp[(d0 + n) * kBlk] = nv.kept.c[n];
      }
      if constexpr (kNarrow) {
        if (kept && col == 0) {
          pool.ks[slot0 + place] = nk.scale;
          pool.vs[slot0 + place] = nv.scale;
        }
      }
    }
  }
  __syncthreads();
  const bool whole = begins && ends, token = begins && p >= 0;
  float* const part = whole ? nullptr : deal.parts + (2 * static_cast<int64_t>(blockIdx.x) + (begins ? 1 : 0)) * min(group, kCols) * (DP + 4);
  for (int x = thread; x < heads * DP; x += kThreads) {
    const int c = x / DP, d = x % DP;
    float ms[kWaves + 1], ls[kWaves + 1], ys[kWaves + 1];
#pragma unroll
    for (int n = 0; n <= kWaves; ++n) {
      const bool is = n < kWaves || token;
      ms[n] = is ? sm[n][c] : -kInf;
      ls[n] = is ? sl[n][c] : 0.f;
      ys[n] = n < kWaves ? so[n % kWaves][c][d] : is ? fresh[d] : 0.f;
    }
    float m = ms[kWaves];
#pragma unroll
    for (int n = 0; n < kWaves; ++n) m = fmaxf(m, ms[n]);
    float l = 0.f, y = 0.f;
#pragma unroll
    for (int n = 0; n <= kWaves; ++n) {
      const float keep = ms[n] == -kInf ? 0.f : exp2_hw(ms[n] - m);
      // no page: its sum is NaN whatever the maximum; weights of nothing but -inf: 0 / 0 at the end
      l += ls[n] == ls[n] ? ls[n] * keep : ls[n];
      y += ys[n] * keep;
    }
    if (whole) {
      if (d < D) out[(static_cast<int64_t>(b) * a.Hq + h0 + c) * D + d] = static_cast<T>(p < 0 ? 0.f : y / l);
    } else {
      float* const to = part + c * (DP + 4);
      to[4 + d] = y;
      if (d == 0) {
        to[0] = m;
        to[1] = l;
      }
    }
  }
  if (deal.parts && begins && (!ends || deal.by_row) && thread == 0) {  // whoever has a part of this row comes behind this workgroup
    const int64_t last = quotient(before * per_stream + static_cast<int64_t>(r + 1) * tiles - 1, share);
    const int64_t to = static_cast<int64_t>(b) * a.Hq + h0;
    deal.desc[deal.by_row ? b * per_stream + r : blockIdx.x] =
        int4{ends ? 0 : static_cast<int>(last - blockIdx.x + 1) | heads << 16, static_cast<int>(blockIdx.x), static_cast<int>(to),
             static_cast<int>(to >> 32)};
  }
  u += t1 - t0;
  if (u >= end || !deal.parts) return;
  t0 = 0;
  if (++r == per_stream) {
    r = 0;
    before += tiles;
    p = positions[++b];
  }
  }
}

// The pieces of one head of a row that several shares have parts of, four dimensions to a lane.
constexpr int kMostGroups = 256 * kMostWaves;
struct Pieces {
  const float* parts;
  int first, cells, cell;
  // the first piece is the last one of its workgroup, the others are the first ones of theirs
  template <int ROW>
  __device__ __forceinline__ const float* at(int n) const {
    return parts + ((2 * static_cast<int64_t>(first + n) + (n == 0 ? 1 : 0)) * cells + cell) * ROW;
  }
};
__device__ __forceinline__ int64_t row_of(const int4& what) { return static_cast<int64_t>(what.w) << 32 | static_cast<uint32_t>(what.z); }

// A few pieces: a wave for 256 / DP heads, one pass.
template <typename T, int DP>
__global__ __launch_bounds__(64) void paged_join_few(int D, int cells, const int4* __restrict__ desc, const float* __restrict__ parts,
                                                     T* __restrict__ out) {
  constexpr int kRow = DP + 4, kLanes = DP / 4;
  const int4 what = desc[blockIdx.x];
  const int used = what.x & 0xffff, lane = threadIdx.x % kLanes, cell = blockIdx.y * (64 / kLanes) + threadIdx.x / kLanes;
  if (cell >= what.x >> 16 || 4 * lane >= D) return;
  const Pieces p{parts, what.y, cells, cell};
  float top = -kInf, sum = 0.f;
  f32x4 y = {};
#pragma unroll 4
  for (int n = 0; n < used; ++n) {
    const float* const row = p.at<kRow>(n);
    const float m = row[0], l = row[1], most = fmaxf(top, m);
    const f32x4 v = *reinterpret_cast<const f32x4*>(row + 4 + 4 * lane);
    const float before = top == -kInf ? 0.f : exp2_hw(top - most), keep = m == -kInf ? 0.f : exp2_hw(m - most);
    sum = (sum == sum ? sum * before : sum) + (l == l ? l * keep : l);
    y = y * before + v * keep;
    top = most;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) out[(row_of(what) + cell) * D + 4 * lane + e] = static_cast<T>(y[e] / sum);
}

// Many pieces: a workgroup for a head.
template <typename T, int DP>
__global__ __launch_bounds__(1024) void paged_join_many(int D, int cells, const int4* __restrict__ desc, const float* __restrict__ parts,
                                                        T* __restrict__ out) {
  constexpr int kRow = DP + 4, kLanes = DP / 4, kSets = 1024 / kLanes, kW = 16;
  __shared__ float weight[kMostGroups], wave_top[kW], wave_sum[kW];
  __shared__ f32x4 acc[kSets][kLanes];
  const int4 what = desc[blockIdx.x];
  const int used = what.x & 0xffff;
  if (static_cast<int>(blockIdx.y) >= what.x >> 16) return;
  const Pieces p{parts, what.y, cells, static_cast<int>(blockIdx.y)};
  static_assert(kMostGroups <= 1024, "a thread for each piece");
  const int n = threadIdx.x;
  const float m = n < used ? p.at<kRow>(n)[0] : -kInf, l = n < used ? p.at<kRow>(n)[1] : 0.f;
  float top = m;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) top = fmaxf(top, __shfl_xor(top, k, 64));
  if ((threadIdx.x & 63) == 0) wave_top[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kW; ++k) top = fmaxf(top, wave_top[k]);
  const float keep = m == -kInf ? 0.f : exp2_hw(m - top);
  float sum = l == l ? l * keep : l;
  weight[n] = keep;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) sum += __shfl_xor(sum, k, 64);
  if ((threadIdx.x & 63) == 0) wave_sum[threadIdx.x >> 6] = sum;
  __syncthreads();
  const int lane = threadIdx.x % kLanes, set = threadIdx.x / kLanes;
  f32x4 y = {};
#pragma unroll 8
  for (int k = set; k < used; k += kSets) y += *reinterpret_cast<const f32x4*>(p.at<kRow>(k) + 4 + 4 * lane) * weight[k];
  acc[set][lane] = y;
  __syncthreads();
  if (set == 0 && 4 * lane < D) {
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < kW; ++k) sum += wave_sum[k];
#pragma unroll
    for (int k = 1; k < kSets; ++k) y += acc[k][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) out[(row_of(what) + p.cell) * D + 4 * lane + e] = static_cast<T>(y[e] / sum);
  }
}

inline int padded(int D, bool narrow) { return D <= 32 && !narrow ? 32 : D <= 64 ? 64 : 128; }

// Workgroups, the least share (in tiles) and the workspace of a call: whole rows where no stream can hold many
// tiles, more where there are more rows to fill the card; else as many shares as run at a time.  In us, shares | whole
// rows: 4 rows of 1000 tokens (float32, heads of 32) 11.9 | 12.8, but 16.5 | 12.0 a call with the host's time, of which the join's
// launch and the workspace take 4; 16 of up to 1000 (int8, of 64) 15.7 | 11.2, 1024 (bfloat16, of 128) 87 | 81; of up to 2000
// tokens 4 (float32) 12.4 | 19.8, 32 (bfloat16) 18 | 26, 128 (int8) 21.2 | 16.2, 256 (bfloat16) 40 | 36, 256 (float32) 27 | 24.
struct StepPlan {
  int groups, least, waves;
  size_t bytes;
};
constexpr int kLeast = 4;
inline StepPlan plan_step(const geo_paged_step_t* g, int waves) {
  const int group = g->heads / g->cache.kv_heads, cells = group < kCols ? group : kCols;
  const int64_t most = ceil_div(g->cache.columns * g->cache.page, static_cast<int64_t>(kTile));
  const int64_t rows = g->batch * g->cache.kv_heads * ceil_div(static_cast<int64_t>(group), static_cast<int64_t>(kCols));
  // whole rows by eight waves where CUs have no more than one and joining heads takes no more LDS (four | eight: 1 stream of 1000
  // tokens, 4 float32 heads of 32, 15.2 | 13.4 us, 64 of 2000 32 | 24; 16 of 2 int8 heads of 64, 1000 tokens 16.2 | 15.2)
  const bool eight = group <= 8 && rows <= 256 && most > 4;
  if (most <= 24 || (most <= 64 && most <= 12 + 2 * std::sqrt(static_cast<double>(rows)))) return {0, 0, eight ? 8 : 4, 0};
  int64_t groups = 256 * waves;
  if (most < (int64_t(1) << 30) / rows) groups = std::min(groups, ceil_div(most * rows, static_cast<int64_t>(kLeast)));
  const bool narrow = g->cache.stored == GEO_I8 || g->cache.stored == GEO_E4M3;
  const size_t row = padded(g->cache.head_dim, narrow) + 4;
  return {static_cast<int>(groups), kLeast, 4, static_cast<size_t>(std::min(groups, rows)) * sizeof(int4) + static_cast<size_t>(groups) * 2 * cells * row * sizeof(float)};
}

template <typename T, typename C, int DP>
int launch_step(const Step& a, const geo_paged_step_t* g, void* out, void* workspace, size_t bytes, hipStream_t stream) {
  const int group = a.Hq / a.pool.Hk;
  const StepPlan s = plan_step(g, step_waves<T, C, DP>());
  if (s.bytes > bytes || (s.bytes && !workspace))
    return set_error(GEO_ERR_WORKSPACE, "paged attention step: workspace of %zu bytes, %zu needed", workspace ? bytes : size_t(0), s.bytes);
  const int64_t rows = static_cast<int64_t>(a.B) * a.pool.Hk * ceil_div(static_cast<int64_t>(group), static_cast<int64_t>(kCols));
  const int64_t blocks = s.groups ? s.groups : rows;
  GEO_REQUIRE(grid_fits(blocks, 64 * s.waves), "paged attention step: too many workgroups");
  Deal deal{s.groups, s.least, rows <= s.groups, nullptr, nullptr};
  const uint32_t places = static_cast<uint32_t>(std::min(rows, static_cast<int64_t>(s.groups)));
  if (s.groups) {
    deal.desc = static_cast<int4*>(workspace);
    deal.parts = reinterpret_cast<float*>(deal.desc + places);
  }
  const size_t lds = a.bias.table ? sizeof(float) * kCols * a.bias.buckets + align_up(a.bias.maxd + 1, 16) : 0;
  auto* const kernel = s.waves == 8 ? &paged_step<T, C, DP, 8> : &paged_step<T, C, DP, 4>;
  kernel<<<dim3(static_cast<uint32_t>(blocks)), dim3(64 * s.waves), lds, stream>>>(a, deal, a.pool.table, a.pos, static_cast<T*>(out));
  GEO_LAUNCH_CHECK("paged_step");
  if (s.groups) {
    const int cells = std::min(group, kCols);
    // one stream of 2500 tokens (10 pieces a row) 10.7 us in all with the wave, 12.2 with the workgroup; of 8000 (31) 16.1, 14.3
    if (s.groups > 16 * rows) {
      paged_join_many<T, DP><<<dim3(places, static_cast<uint32_t>(cells)), dim3(1024), 0, stream>>>(a.pool.D, cells, deal.desc, deal.parts,
                                                                                                 static_cast<T*>(out));
    } else {
      paged_join_few<T, DP><<<dim3(places, static_cast<uint32_t>(ceil_div(cells, 256 / DP))), dim3(64), 0, stream>>>(
          a.pool.D, cells, deal.desc, deal.parts, static_cast<T*>(out));
    }
    GEO_LAUNCH_CHECK("paged_join");
  }
  return GEO_OK;
}
template <typename T, typename C>
int choose_head(const Step& a, const geo_paged_step_t* g, void* out, void* ws, size_t bytes, hipStream_t stream) {
  switch (padded(a.pool.D, Code<C>::kNarrow)) {
    case 32:
      if constexpr (!Code<C>::kNarrow) return launch_step<T, C, 32>(a, g, out, ws, bytes, stream);
      [[fallthrough]];
    case 64: return launch_step<T, C, 64>(a, g, out, ws, bytes, stream);
    default: return launch_step<T, C, 128>(a, g, out, ws, bytes, stream);
  }
}
template <typename T>
int choose_stored(int stored, const Step& a, const geo_paged_step_t* g, void* out, void* ws, size_t bytes, hipStream_t stream) {
  if (stored == GEO_I8) return choose_head<T, I8>(a, g, out, ws, bytes, stream);
  return stored == GEO_E4M3 ? choose_head<T, E4>(a, g, out, ws, bytes, stream) : choose_head<T, T>(a, g, out, ws, bytes, stream);
}

}  // namespace paged
}  // namespace geo

extern "C" size_t geo_paged_attention_step_workspace_bytes(const geo_paged_step_t* g) {
  using namespace geo::paged;
  if (!g || !sizes_ok(g->cache, g->batch, g->heads)) return 0;
  return plan_step(g, kMostWaves).bytes;
}

extern "C" int geo_paged_attention_step(const geo_paged_step_t* g, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace geo;
  const char* const name = "paged attention step";
  GEO_REQUIRE(g, "%s: null arguments", name);
  paged::Step a;
  if (const int rc = paged::pool_args(name, &g->cache, &a.pool, g->batch != 0)) return rc;
  GEO_REQUIRE(paged::type_ok(g->dtype, g->cache.stored), "%s: tokens of type code %d, a pool of %d", name,
              static_cast<int>(g->dtype), static_cast<int>(g->cache.stored));
  GEO_REQUIRE(g->batch >= 0 && g->batch < (int64_t(1) << 31) && g->heads >= 1 && g->heads < (1 << 20) &&
                  g->heads % g->cache.kv_heads == 0,
              "%s: %d heads are no multiple of %d key heads (below 2^20)", name, g->heads, g->cache.kv_heads);
  if (g->bias) {
    GEO_REQUIRE(g->bias_dtype == GEO_F32 || g->bias_dtype == GEO_BF16 || g->bias_dtype == GEO_F16, "%s: bias dtype code %d", name,
                static_cast<int>(g->bias_dtype));
    GEO_REQUIRE(g->bias_lut && g->buckets >= 1 && g->buckets <= 256 && g->max_distance >= 1 && g->max_distance <= 1024,
                "%s: bias of %d buckets up to distance %d (at most 256 and 1024)", name, g->buckets, g->max_distance);
  }
  if (g->batch == 0) return GEO_OK;
  const int size = g->dtype == GEO_F32 ? 4 : 2;
  auto in_pieces = [size](const void* p, int64_t st, int64_t sh) {
    return p && reinterpret_cast<uintptr_t>(p) % 16 == 0 && st * size % 16 == 0 && sh * size % 16 == 0;
  };
  GEO_REQUIRE(in_pieces(g->q, g->q_stream, g->q_head) && in_pieces(g->k, g->k_stream, g->k_head) &&
                  in_pieces(g->v, g->v_stream, g->v_head),
              "%s: null q, k or v, or rows not on multiples of 16 bytes", name);
  GEO_REQUIRE(out && g->positions, "%s: null output or positions", name);
  a.q = g->q, a.k = g->k, a.v = g->v;
  a.q_st = g->q_stream, a.q_sh = g->q_head, a.k_st = g->k_stream, a.k_sh = g->k_head, a.v_st = g->v_stream, a.v_sh = g->v_head;
  a.pos = g->positions;
  a.bias = {g->bias, g->bias_lut, g->bias_dtype, g->buckets, g->max_distance};
  a.B = static_cast<int>(g->batch), a.Hq = g->heads, a.scale = g->scale;
  const hipStream_t on = as_stream(stream);
  if (g->dtype == GEO_F32) return paged::choose_stored<float>(g->cache.stored, a, g, out, workspace, workspace_bytes, on);
  if (g->dtype == GEO_BF16) return paged::choose_stored<__bf16>(g->cache.stored, a, g, out, workspace, workspace_bytes, on);
  return paged::choose_stored<_Float16>(g->cache.stored, a, g, out, workspace, workspace_bytes, on);
}
