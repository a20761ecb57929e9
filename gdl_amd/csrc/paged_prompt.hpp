// paged_prompt.hpp — attention of several new tokens per stream, which its pages hold already, over all
// the stream's tokens up to each: a prompt, or a piece of one behind a history.
//
// o = sum over tiles of keys of exp2(s - top) V in one pass, s = scale log2 e q.K + bias, with the largest score so far as
// `top`, moved only when a tile exceeds it by 8.
//
// Sᵀ = K Qᵀ and Oᵀ = Vᵀ Pᵀ on 32x32x16 products, a query to a lane (and its twin in the other half), as in the
// window's attention.  Four waves of 32 queries share tiles of keys and values in LDS, which are filled
// through registers one tile ahead: 8-bit codes are decoded once there, for four waves.  A workgroup's queries are
// `heads` heads of one key head by up to 128 / heads tokens, token by token, so that the keys' way through memory and LDS is
// shared and calls of few tokens fill their rows.  Values come in columns (one dimension's tokens
// adjoin), as the second product takes them; the rows of Sᵀ are read in the order that leaves each lane the
// weights of eight adjoining tokens.
//
// A wave's scores, exponentials and product with V follow one another, and two (to head size 64 three) waves a SIMD cover for
// each other: 8 pieces of up to 2048 tokens behind 8192, 16 (4) heads of 128, bfloat16, 966 us, 823 TFLOP/s, matrix instructions
// in 39% of the cycles, vector instructions in 40%; int8 1.08 ms, float32 100 TFLOP/s (matrix instructions 77%).
// Codes cost a conversion each and their scales two products a score: 32 packets of up to 384 behind 4000 e4m3
// tokens, 8 (2) heads of 64, 151 us with the join, vector instructions in 63% of the cycles.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

#include "paged.hpp"

namespace geo {
namespace paged {

using attn::f32x16;
using attn::halves_max;
using attn::halves_sum;
using attn::Type;

struct Prompt {
  Pool pool;
  const void* q;
  int64_t q_st, q_sh;
  const int64_t *ptr, *start;
  attn::Bias bias;
  int64_t T;
  int B, Hq, heads, U;  // heads of a key head that a workgroup takes together, and how many tokens of each
  int bias_row;          // floats of a head's biases in LDS
  int fine;              // sequences whose middle query sees at most so many keys have their weights in two parts
  float scale;
};

constexpr int kPromptThreads = 256;
using Words = uint32_t __attribute__((ext_vector_type(4)));

// How a pool of C meets queries of T: key tiles of type K, value tiles of type V.  Codes stay codes where a
// 16-bit type holds them (float16 weights times a scale could leave its range, so those meet bf16 values in two
// parts) and are multiplied out for float32.  FINE: sequences that plan_prompt says so of have weights in two parts.
template <typename T, typename C, bool FINE = false>
struct Meet {
  static constexpr bool kNarrow = Code<C>::kNarrow, kFloat = sizeof(T) == 4;
  static constexpr bool kScaled = kNarrow && !kFloat;  // scales meet scores and weights, not the tiles
  using K = T;
  using V = typename std::conditional<kScaled, __bf16, T>::type;
  static constexpr int kParts = kFloat ? 1 : kScaled ? parts_of<T>() : 1;
  static constexpr bool kFine = FINE && !kFloat && kParts == 1;
  static constexpr int kKeys = kFloat ? 32 : 64;
};

// A word of values (two of 16 bits) of the tokens `key` on: zeros in the place of those from `limit` on and of
// infinities and NaN, whose tokens are noted.  In words: as an array of elements they would go through memory.
template <typename V>
__device__ __forceinline__ uint32_t seen_and_finite(uint32_t w, int key, int limit, uint32_t* note) {
  constexpr uint32_t kPower = sizeof(V) == 4 ? 0x7f800000u : __is_same(V, __bf16) ? 0x7f80u : 0x7c00u;
#pragma unroll
  for (int e = 0; e < 4 / static_cast<int>(sizeof(V)); ++e) {
    const uint32_t power = kPower << (16 * e), all = sizeof(V) == 4 ? ~0u : 0xffffu << (16 * e);
    const bool in = key + e < limit, wild = (w & power) == power;
    if (in && wild) atomicOr(&note[(key + e) >> 5], 1u << ((key + e) & 31));
    if (!in || wild) w &= ~all;
  }
  return w;
}

template <typename T, typename C, int DP>
struct PromptLds {
  using M = Meet<T, C>;
  static constexpr int kKRow = DP * sizeof(T) + 16, kVRow = M::kKeys * sizeof(typename M::V) + 16;  // bytes: rows in other banks
  static constexpr int kK = M::kKeys * kKRow, kV = DP * kVRow, kS = M::kScaled ? 2 * M::kKeys * 4 : 0;
  static constexpr int kBuffer = kK + kV + kS;
};

// Workgroups of the kernel on a CU, by the registers that it takes.
constexpr int prompt_waves(int DP) { return DP == 128 ? 2 : 3; }

template <typename T, typename C, int DP, bool FINE>
__global__ __launch_bounds__(kPromptThreads, (prompt_waves(DP))) void paged_prompt(const Prompt a, int64_t tiles, int pieces,
                                                                  const int32_t* __restrict__ table, float* __restrict__ part,
                                                                  T* __restrict__ out) {
  using M = Meet<T, C, FINE>;
  using L = PromptLds<T, C, DP>;
  using TK = typename M::K;
  using TV = typename M::V;
  using KFrag = typename Type<TK>::Frag;
  using VFrag = typename Type<TV>::Frag;
  typedef KFrag KLds __attribute__((aligned(16)));  // as LDS holds them
  typedef VFrag VLds __attribute__((aligned(16)));
  constexpr int kSize = sizeof(C), kKeys = M::kKeys, kBlk = block_tokens<C>(), kPer = 16 / kSize;
  constexpr int kSub = kKeys / 32, kKc = DP / 16, kMt = DP / 32;
  constexpr bool kHalf = Faint<TV>::kHalf;
  constexpr float kLift = Faint<TV>::kLift, kLazy = Faint<TV>::kLazy;
  constexpr int kLoads = (kKeys * DP * kSize + 16 * kPromptThreads - 1) / (16 * kPromptThreads);
  constexpr int kSpan = kKeys < kBlk ? kKeys : kBlk, kCpb = kSpan * kSize / 16;  // tokens and pieces of a dimension in a block
  extern __shared__ __attribute__((aligned(16))) char lds[];
  // rows of a tile's values that hold infinities or NaN, which are taken out: tile n's in wild[n % 3], cleared while tile
  // n - 2 is worked on, filled during n - 1, read during n
  __shared__ uint32_t wild[3][2];
  float* const sbias = reinterpret_cast<float*>(lds + 2 * L::kBuffer);
  const Pool& pool = a.pool;
  const int D = pool.D, group = a.Hq / pool.Hk, sets = group / a.heads;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // One XCD works through one key head's sequences, so that their pages stay in its L2; where the heads and pieces
  // are not as many as to go round, in short runs (a prompt of 16,000 in 2 | 4 pieces of 2 heads: 496, 476 us in
  // runs, 624, 451 us otherwise).
  int64_t w = pieces == 1 || pieces * (a.Hq / a.heads) % 8 == 0 ? xcd_block() : xcd_block_runs(8);
  const int64_t tile = tiles - 1 - w % tiles;  // the longest first
  w /= tiles;
  const int piece = static_cast<int>(w % pieces);
  w /= pieces;
  const int set = static_cast<int>(w % sets), hk = static_cast<int>(w / sets), head0 = hk * group + set * a.heads;
  const int64_t rows = a.T * a.Hq;  // of a piece's partial results

  // tokens that see nothing: outside all sequences, or at negative positions
  auto nothing = [&](int64_t t) {
    const int64_t first = t * a.Hq + head0;
    if (pieces == 1) {
      for (int x = threadIdx.x; x < a.heads * D; x += kPromptThreads) out[first * D + x] = static_cast<T>(0.f);
    } else if (static_cast<int>(threadIdx.x) < a.heads) {
      float* const row = part + (piece * rows + first + threadIdx.x) * (DP + 4);
      row[0] = -kInf;
      row[1] = -1.f;
    }
  };
  if (a.ptr) {
    const int64_t first = a.ptr[0], end = a.ptr[a.B], from = tile * a.U, to = min(from + a.U, a.T);
    for (int64_t t = from; t < min(first, to); ++t) nothing(t);
    for (int64_t t = max(from, max(first, end)); t < to; ++t) nothing(t);
  }
  const Span s = span_of<kFromFirst>(a.ptr, a.start, a.B, a.T, tile, a.U);
  for (int64_t t = 0; t < s.before; ++t) nothing(s.first + t);
  if (s.lo >= s.hi) return;

  const int room = pool.columns * pool.page;  // tokens that the table has a place for
  auto held = [&](int64_t p) { return static_cast<int>(min(p, static_cast<int64_t>(room))); };
  const int row = 32 * wave + (lane & 31), place = row / a.heads;  // the lane's query in the workgroup, its token in the tile
  const int head = head0 + row - place * a.heads;
  const int p = held(s.tile0 + place);                    // its position; `room`: beyond the table
  // the first and last positions of the wave's; of a wave without any, none
  const int first_place = 32 * wave / a.heads, last_place = min((32 * wave + 31) / a.heads, s.hi - 1);
  const int wave_first = held(s.tile0 + first_place), wave_last = first_place < s.hi ? held(s.tile0 + last_place) : -1;
  const int first_query = held(s.tile0 + s.lo), end = held(s.tile0 + s.hi);  // keys that someone here sees end there
  const int per = ((end + pieces - 1) / pieces + 63) & ~63, k0 = piece * per, k1 = min(end, k0 + per);
  const int64_t token = s.first + s.tile0 - s.start + place;
  const bool real = place >= s.lo && place < s.hi;
  const bool fine = M::kFine && __builtin_amdgcn_readfirstlane(s.middle <= a.fine);

  KFrag q[kKc];
  {
    const int64_t t = s.first + s.tile0 - s.start + min(max(place, s.lo), s.hi - 1);
    const T* const from = static_cast<const T*>(a.q) + t * a.q_st + head * a.q_sh;
#pragma unroll
    for (int c = 0; c < kKc; ++c) {
      const int d = 16 * c + 8 * half;
      union { Words u[sizeof(T) / 2]; KFrag f; } x = {};
      if (d < D && a.scale != 0.f) {
        const uint32_t flip = a.scale < 0.f ? (sizeof(T) == 4 ? 0x80000000u : 0x80008000u) : 0u;
#pragma unroll
        for (int n = 0; n < static_cast<int>(sizeof(T) / 2); ++n) {
          x.u[n] = reinterpret_cast<const Words*>(from + d)[n];
          x.u[n] ^= flip;
        }
      }
      q[c] = x.f;
    }
  }
  // positive, so that the products' largest is the scores': the queries carry its sign, or are zeros
  const float scale2 = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
  float far = 0.f;
  const float* const near = sbias + (head - head0) * a.bias_row;
  if (a.bias.table) {
    for (int x = threadIdx.x; x < a.heads * (a.bias.maxd + 1); x += kPromptThreads) {
      const int h = x / (a.bias.maxd + 1), back = x % (a.bias.maxd + 1);
      sbias[h * a.bias_row + back] = attn::bias_value(a.bias, static_cast<int64_t>(a.bias.lut[a.bias.maxd - back]) * a.Hq + head0 + h);
    }
  }
  if (threadIdx.x < 6) wild[threadIdx.x >> 1][threadIdx.x & 1] = 0;
  if (D < DP)  // keys' values past the head count as zeros
    for (int x = threadIdx.x; x < 2 * kKeys * (DP - D); x += kPromptThreads) {
      const int r = x / (DP - D);
      reinterpret_cast<TK*>(lds + (r / kKeys) * L::kBuffer + (r % kKeys) * L::kKRow)[D + x % (DP - D)] = static_cast<TK>(0.f);
    }

  // this thread's pieces of a tile: 16 bytes each, from where and to where
  const int pieces_of_tile = kKeys * D / kPer;
  uint32_t kto[kLoads], vfrom[kLoads], vto[kLoads];
#pragma unroll
  for (int n = 0; n < kLoads; ++n) {
    const int x = threadIdx.x + n * kPromptThreads, per_row = D / kPer;
    kto[n] = x / per_row * L::kKRow + x % per_row * kPer * static_cast<int>(sizeof(TK));
    const int blk = x / (kCpb * D), d = x / kCpb % D, at = x % kCpb;
    vfrom[n] = blk * 64 * D + d * 64 + at * 16;
    vto[n] = d * L::kVRow + (blk * kSpan + at * kPer) * static_cast<int>(sizeof(TV));
  }
  Words kx[kLoads], vx[kLoads];
  float ksx = 0.f, vsx = 0.f;
  // where the next fetch reads: a column of the table and a place in its page; the entry behind it is on its way
  const int32_t* const entries = table + s.b * pool.table_st;
  auto entry = [&](int n) { return __builtin_amdgcn_readfirstlane(entries[min(n, pool.columns - 1)]); };
  int column = k0 / pool.page, place_in = k0 - column * pool.page, entry_now = 0, entry_next = 0;
  if (k0 < k1) entry_now = entry(column), entry_next = entry(column + 1);
  int at = -1, off = 0;  // the fetched tile's page, and its place there
  auto fetch = [&]() {
    at = static_cast<uint32_t>(entry_now) < static_cast<uint32_t>(pool.pages) ? entry_now : -1;
    off = place_in;
    place_in += kKeys;
    if (place_in == pool.page) {
      place_in = 0;
      entry_now = entry_next;
      entry_next = entry(++column + 1);
    }
    const int64_t slot0 = (static_cast<int64_t>(max(at, 0)) * pool.Hk + hk) * pool.page + off;
    const char* const kb = pool.k + slot0 * D * kSize;
    const char* const vb = pool.v + (slot0 / kBlk * kBlk) * D * kSize + slot0 % kBlk * kSize;
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int x = threadIdx.x + n * kPromptThreads;
      if (x < pieces_of_tile) {
        kx[n] = *reinterpret_cast<const Words*>(kb + static_cast<uint32_t>(x) * 16);
        vx[n] = *reinterpret_cast<const Words*>(vb + vfrom[n]);
      }
    }
    if constexpr (M::kScaled) {
      if (threadIdx.x < kKeys) {
        uint32_t key = threadIdx.x;
        asm volatile("" : "+v"(key));  // a scalar base and a lane's 32 bits: 64-bit sums of pool and lane would be kept, and spilled
        ksx = (pool.ks + slot0)[key];
        vsx = (pool.vs + slot0)[key];
      }
    }
  };
  // `edge`: a tile whose later keys some query does not see.  Values there must not reach it through a
  // weight of 0: what lies behind the last token becomes 0, and infinities and NaN are taken out, noted, and
  // given back to those that do see them.
  auto store = [&](int t, char* to, uint32_t* note) {
    const bool edge = t + kKeys - 1 > first_query;
    const int64_t slot0 = (static_cast<int64_t>(max(at, 0)) * pool.Hk + hk) * pool.page + off;
    char *const kt = to, *const vt = to + L::kK;
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      int x = threadIdx.x + n * kPromptThreads;
      if (x >= pieces_of_tile) continue;
      if (edge) asm volatile("" : "+v"(x));  // as below: not ahead of the loop
      const int key0 = x / (kCpb * D) * kSpan + x % kCpb * kPer;  // first of the values' tokens
      if constexpr (!M::kNarrow) {
        *reinterpret_cast<Words*>(kt + kto[n]) = kx[n];
        Words v = vx[n];
        if (edge) {
          constexpr int kWord = 4 / kSize;  // tokens of a word
          v.x = seen_and_finite<TV>(v.x, key0, end - t, note);
          v.y = seen_and_finite<TV>(v.y, key0 + kWord, end - t, note);
          v.z = seen_and_finite<TV>(v.z, key0 + 2 * kWord, end - t, note);
          v.w = seen_and_finite<TV>(v.w, key0 + 3 * kWord, end - t, note);
        }
        *reinterpret_cast<Words*>(vt + vto[n]) = v;
      } else if constexpr (M::kFloat) {
        const float ks = pool.ks[slot0 + x / (D / kPer)];
        union { Words u; uint8_t c[16]; } y, z;
        y.u = kx[n];
        z.u = vx[n];
        float* const kr = reinterpret_cast<float*>(kt + kto[n]);
        float* const vr = reinterpret_cast<float*>(vt + vto[n]);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          kr[e] = Code<C>::value(y.c[e]) * ks;
          float v = Code<C>::value(z.c[e]) * pool.vs[slot0 + key0 + e];
          if (edge) {
            const bool in = t + key0 + e < end, fine = fabsf(v) < kInf;
            if (in && !fine) atomicOr(&note[(key0 + e) >> 5], 1u << ((key0 + e) & 31));
            if (!in || !fine) v = 0.f;
          }
          vr[e] = v;
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t klo = h ? kx[n].z : kx[n].x, khi = h ? kx[n].w : kx[n].y;
          if constexpr (__is_same(T, _Float16)) reinterpret_cast<f16x8*>(kt + kto[n])[h] = decode8_f16<C>(klo, khi);
          else reinterpret_cast<bf16x8*>(kt + kto[n])[h] = decode8<C>(klo, khi);
          Bytes16 v;
          v.b = decode8<C>(h ? vx[n].z : vx[n].x, h ? vx[n].w : vx[n].y);
          if (edge) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v.w[e] = seen_and_finite<__bf16>(v.w[e], key0 + 8 * h + 2 * e, end - t, note);
          }
          reinterpret_cast<bf16x8*>(vt + vto[n])[h] = v.b;
        }
      }
    }
    if constexpr (M::kScaled) {
      if (threadIdx.x < kKeys) {
        float* const scales = reinterpret_cast<float*>(to + L::kK + L::kV);
        scales[threadIdx.x] = ksx * scale2;
        scales[kKeys + threadIdx.x] = vsx;
      }
    }
  };

  f32x16 o[kMt];
#pragma unroll
  for (int m = 0; m < kMt; ++m) o[m] = f32x16{};
  float top = -kInf, sum = 0.f;  // what scores are taken less by (Faint)
  bool lost = p >= room;

  __syncthreads();  // zeros past the head, biases, notes
  if (a.bias.table) far = near[a.bias.maxd];
  int page_now = -1;
  if (k0 < k1) {
    fetch();
    page_now = at;
    store(k0, lds, wild[0]);
  }
  int buf = 0, turn = 0;
  for (int t = k0; t < k1; t += kKeys, buf ^= 1, turn = turn == 2 ? 0 : turn + 1) {
    __syncthreads();
    if (threadIdx.x < 2) wild[turn == 0 ? 2 : turn - 1][threadIdx.x] = 0;
    const char *const kt = lds + buf * L::kBuffer, *const vt = kt + L::kK;
    const bool more = t + kKeys < k1;
    const int off_now = off;
    if (more) fetch();
    const int page_next = at;
    if (t <= wave_last) {
      const bool whole = t + kKeys - 1 <= wave_first;
      // In float32 the products are what takes the time, and those past the head's size are left out (heads of 8: 193 | 163 us,
      // of 80 646 | 496, of 128 664 | 674); in 16 bits the branches cost more (of 80 175 | 190 us, of 128 192 | 218).
      f32x16 product[kSub];
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        product[u] = f32x16{};
        // row 16 c + 8 a + 4 h + i of the product is token 16 c + 8 h + 4 a + i
        const int r = lane & 31, key = 32 * u + ((r & 19) | (r >> 2 & 1) << 3 | (r >> 3 & 1) << 2);
        const char* const row = kt + key * L::kKRow + half * 8 * static_cast<int>(sizeof(TK));
#pragma unroll
        for (int c = 0; c < kKc; ++c)
          if (!M::kFloat || 32 * c < DP || 16 * c < D) product[u] = Type<TK>::mma(*reinterpret_cast<const KLds*>(row + c * 16 * sizeof(TK)), q[c], product[u]);
      }
      if constexpr (!M::kFloat) attn::reads_ahead<kSub * kKc, 4, 1>();
      // number 8 c + j of x[u] is token t + 32 u + 16 c + 8 half + j; single registers, which branches may change
      // without a copy of all sixteen
      float x[kSub][16];
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[u][r] = product[u][r];
      float vs[kSub];
      if constexpr (M::kScaled) {  // lane r of 16 holds the scale of the half's register r, and hands it round
        const float* const scales = reinterpret_cast<const float*>(kt + L::kK + L::kV) + 16 * (lane >> 3 & 1) + 8 * half + (lane & 7);
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          by_group(x[u], scales[32 * u]);
          vs[u] = scales[kKeys + 32 * u];
        }
      }
      if (a.bias.table) {
        const float by = M::kScaled ? 1.f : scale2;
        if (wave_first - (t + kKeys - 1) < a.bias.maxd) {
#pragma unroll
          for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              x[u][r] = fmaf(x[u][r], by, near[min(max(p - (t + 32 * u + 16 * (r >> 3) + 8 * half + (r & 7)), 0), a.bias.maxd)]);
        } else {
#pragma unroll
          for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) x[u][r] = fmaf(x[u][r], by, far);
        }
      }
      float by = M::kScaled || a.bias.table ? 1.f : scale2;  // what the scores still lack
      const int seen = p - t - 8 * half;  // a lane's tokens 32 u + 16 c + j up to this one
      if (!whole) {
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (32 * u + 16 * (r >> 3) + (r & 7) > seen) x[u][r] = -kInf;
      }
      float most = x[0][0];
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, x[u][r]);
      most = halves_max(most) * by;
      const bool up = most - top > kLazy + kLift;
      if (__any(up)) {
        most = Faint<TV>::lifted(most);
        const float keep = up ? exp2_hw(top - most) : 1.f;
        top = up ? most : top;
        sum *= keep;
#pragma unroll
        for (int m = 0; m < kMt; ++m) o[m] *= keep;
      }
      const float shift = top == -kInf ? 0.f : top;
      if constexpr (!M::kScaled) {
        // `top` is a product rounded once; taken from exact ones, far out, it would leave their step's half, and weights of
        // more than the type holds
        const bool far_out = fabsf(shift) > 0x1p20f;
        if (__any(far_out)) {
          const float rounded = far_out ? by : 1.f;
#pragma unroll
          for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) x[u][r] *= rounded;
          by = far_out ? 1.f : by;
        }
      }
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          x[u][r] = exp2_hw(fmaf(x[u][r], by, -shift));
          sum += x[u][r];
        }
      if constexpr (M::kScaled) {
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          by_group(x[u], vs[u]);
          if (!whole) {  // an unseen scale may be NaN
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (32 * u + 16 * (r >> 3) + (r & 7) > seen) x[u][r] = 0.f;
          }
        }
      }
      auto add = [&](auto part) {  // the product with a further part of the weights
#pragma unroll
        for (int u = 0; u < kSub; ++u)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = x[u][8 * c + e];
            const VFrag w = part(y);
            const char* const col = vt + (lane & 31) * L::kVRow + (32 * u + 16 * c + 8 * half) * static_cast<int>(sizeof(TV));
#pragma unroll
            for (int m = 0; m < kMt; ++m) o[m] = Type<TV>::mma(*reinterpret_cast<const VLds*>(col + 32 * m * L::kVRow), w, o[m]);
          }
      };
      // ahead of the first part's product where scales and their mask end a block anyway: 2% less than behind it
      if constexpr (M::kFine && M::kScaled) {
        if (fine) add([](const float(&y)[8]) { return second8<VFrag>(y); });
      }
      using Half2 = _Float16 __attribute__((ext_vector_type(2)));
      Half2 least = {static_cast<_Float16>(1.f), static_cast<_Float16>(1.f)};
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          VFrag w[M::kParts];
          if constexpr (!M::kFloat) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = x[u][8 * c + e];
            split8<M::kParts>(y, w);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[0][e] = static_cast<TV>(x[u][8 * c + e]);
          }
          if constexpr (kHalf) {
#pragma unroll
            for (int e = 0; e < 4; ++e) least = __builtin_elementwise_minimum(least, Half2{w[0][2 * e], w[0][2 * e + 1]});
          }
          const char* const col = vt + (lane & 31) * L::kVRow + (32 * u + 16 * c + 8 * half) * static_cast<int>(sizeof(TV));
#pragma unroll
          for (int m = 0; m < kMt; ++m) {
            if (M::kFloat && 64 * m >= DP && 32 * m >= D) continue;
            const VFrag v = *reinterpret_cast<const VLds*>(col + 32 * m * L::kVRow);
#pragma unroll
            for (int n = 0; n < M::kParts; ++n) o[m] = Type<TV>::mma(v, w[n], o[m]);
          }
        }
      if constexpr (!M::kFloat && M::kParts == 1) attn::reads_ahead<kSub * 2 * kMt, 4, 1>();
      if constexpr (M::kFine && !M::kScaled) {
        if (fine) add([](const float(&y)[8]) { return second8<VFrag>(y); });
      }
      if constexpr (kHalf) {
        const float below = Faint<TV>::below(fine ? 2 : 1);
        bool some = static_cast<float>(least.x) < below || static_cast<float>(least.y) < below;
        if (!whole) {  // weights that the mask made 0 are none
          some = false;
#pragma unroll
          for (int u = 0; u < kSub; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) some |= x[u][r] > 0.f && x[u][r] < below;
        }
        if (__any(some)) {
#pragma unroll
          for (int m = 0; m < kMt; ++m) o[m] *= Faint<TV>::kUp;
          add([&](const float(&y)[8]) { return fine ? faint8<2>(y) : faint8<1>(y); });
#pragma unroll
          for (int m = 0; m < kMt; ++m) o[m] *= Faint<TV>::kDown;
        }
      }
      for (int u = 0; u < kSub; ++u) {
        uint32_t rest = wild[turn][u];
        while (rest) {  // rare: the queries that see an infinity or NaN have one in its dimension
          const int key = 32 * u + __builtin_ctz(rest);
          rest &= rest - 1;
          const int slot = off_now + key;
          const int64_t slot0 = (static_cast<int64_t>(max(page_now, 0)) * pool.Hk + hk) * pool.page;
          const C* col = reinterpret_cast<const C*>(pool.v) + slot0 * D + static_cast<int64_t>(slot / kBlk) * kBlk * D + slot % kBlk;
          int d0 = 4 * half;
          asm volatile("" : "+v"(d0));  // nothing of this ahead of the loop: it would take the products' registers
          float scale = 1.f;
          if constexpr (M::kNarrow) scale = pool.vs[slot0 + slot];
#pragma unroll
          for (int m = 0; m < kMt; ++m)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int d = d0 + 32 * m + 8 * (r >> 2) + (r & 3);
              if (d < D && p >= t + key) {
                float v;
                if constexpr (M::kNarrow) v = Code<C>::value(col[d * kBlk].bits) * scale;
                else v = static_cast<float>(col[d * kBlk]);
                if (!(fabsf(v) < kInf)) o[m][r] = __builtin_nanf("");
              }
              if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);
            }
        }
      }
      if (page_now < 0 && p >= t) lost = true;
    }
    if (more) store(t + kKeys, lds + (buf ^ 1) * L::kBuffer, wild[turn == 2 ? 0 : turn + 1]);
    page_now = page_next;
  }
  sum = halves_sum(sum);
  if (lost) sum = __builtin_nanf("");
  if (!real) return;
  if (pieces == 1) {
    attn::store_row<T>(out + (token * a.Hq + head) * D, o, 1.f / sum, D);  // weights of nothing but -inf: 0 times infinity
  } else {
    float* const to = part + (piece * rows + token * a.Hq + head) * (DP + 4);
    if (half == 0) {
      to[0] = top;
      to[1] = sum;
    }
    if (k0 < k1) attn::store_row<float>(to + 4, o, 1.f, DP);
  }
}

// The pieces of a row joined: DP / 4 lanes to a row, four dimensions each, SETS of them with a share of the pieces.
template <typename T, int DP, int SETS>
__global__ __launch_bounds__(kPromptThreads) void paged_prompt_join(int D, int64_t rows, int pieces, const float* __restrict__ part,
                                                                    T* __restrict__ out) {
  constexpr int kLanes = DP / 4, kAtOnce = kPromptThreads / (kLanes * SETS), kRow = DP + 4;
  using f32x4 = float __attribute__((ext_vector_type(4)));
  struct Part { float top, sum; f32x4 y; };
  __shared__ float tops[SETS][kAtOnce], sums[SETS][kAtOnce];
  __shared__ f32x4 acc[SETS][kAtOnce][kLanes];
  const int lane = threadIdx.x % kLanes, set = threadIdx.x / kLanes % SETS, place = threadIdx.x / (kLanes * SETS);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kAtOnce + place;
  if (SETS == 1 && row >= rows) return;
  const float* const first = part + min(row, rows - 1) * kRow;
  Part a{-kInf, 0.f, {}};
  auto add = [&](float m, float l, const f32x4& v) {
    const float most = fmaxf(a.top, m), before = a.top == -kInf ? 0.f : exp2_hw(a.top - most), keep = m == -kInf ? 0.f : exp2_hw(m - most);
    a.sum = (a.sum == a.sum ? a.sum * before : a.sum) + (l == l ? l * keep : l);
    a.y = a.y * before + (m == -kInf && l == 0.f ? f32x4{} : v) * keep;  // a piece without tokens holds no values
    a.top = most;
  };
#pragma unroll 4
  for (int n = set; n < pieces; n += SETS) {
    const float* const from = first + n * rows * kRow;
    add(from[0], from[1], *reinterpret_cast<const f32x4*>(from + 4 + 4 * lane));
  }
  if constexpr (SETS > 1) {
    acc[set][place][lane] = a.y;
    if (lane == 0) {
      tops[set][place] = a.top;
      sums[set][place] = a.sum;
    }
    __syncthreads();
    if (set > 0 || row >= rows) return;
    for (int n = 1; n < SETS; ++n) add(tops[n][place], sums[n][place], acc[n][place][lane]);
  }
  const int d = 4 * lane;
  if (d >= D) return;
  union { T t[4]; uint2 u2; uint4 u4; } w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w.t[e] = static_cast<T>(first[1] == -1.f ? 0.f : a.y[e] / a.sum);
  if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(out + row * D + d) = w.u2;
  else *reinterpret_cast<uint4*>(out + row * D + d) = w.u4;
}

inline int prompt_padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

// A key head's query heads that one workgroup takes together, and the pieces into which it cuts a tile's keys.
struct PromptPlan {
  int heads, U, bias_row, pieces, fine;
  int64_t tiles, blocks;
};
// The pieces are those of the least time by this estimate, in microseconds: a workgroup takes `tile` for 64 keys on a CU
// that has all it can hold, two thirds of it on others (in float32, where two fill a CU's matrix units, when alone), and
// 1.3 tiles to begin; full CUs end 0.38 of the longest workgroup apart; a join costs 6.3, 0.06 a piece and the
// parts' way through memory at 6.6 TB/s.  Over 40 kinds of
// calls, from prompts of 300 tokens to packets behind 60,000, the choice is within 2% of the best at the median, 11% at
// most.  In us, whole | 2, 4, 8, 16 pieces: 8 (2) heads of 64 over e4m3, 16 packets of 100 behind 1000 41 | 31, 27, 31, 41,
// 32 of up to 384 behind 4000 192 | 182, 178, 204, a prompt of 16,000 815 | 496, 451, 507, 667; 16 (4) heads of
// 128, bfloat16, 2 of up to 2048 behind 8192 334 | 314, 294, 338.
inline PromptPlan plan_prompt(const geo_paged_prompt_t* g) {
  PromptPlan p;
  const int Hq = g->heads, group = Hq / g->cache.kv_heads, DP = prompt_padded(g->cache.head_dim), waves = prompt_waves(DP);
  const int64_t most = g->cache.columns * g->cache.page;
  const double T = static_cast<double>(g->tokens), B = static_cast<double>(g->batch);
  // All heads of the key head, or the most that divide them and leave at most 13 of 128 rows empty, with biases that let two
  // workgroups of the largest head size share a CU's LDS
  const int places = std::min(std::max(g->max_distance, 0), 1024) + 1;
  p.heads = p.bias_row = 1;
  for (int h = std::min(group, 128); h >= 1; --h) {
    // a wave's heads begin in other banks
    p.bias_row = g->bias ? places + (32 - places % 32 + (32 + h - 1) / h) % 32 : 0;
    p.heads = h;
    if (group % h == 0 && 128 / h * h >= 115 && h * p.bias_row <= 2240) break;
  }
  p.U = 128 / p.heads;
  p.tiles = tiles_of<kFromFirst>(g->tokens, g->batch, p.U);
  const int64_t columns = Hq / p.heads;
  double tile = g->cache.stored == g->dtype ? 2.25 : g->dtype == GEO_BF16 ? 2.6 : 3.9;
  if (DP == 128) tile *= 1.25;
  if (g->dtype == GEO_F32) tile = DP == 32 ? 6.2 : 0.13 * DP;
  const double rows = (std::floor(T / p.U) + 0.5 * B) * columns;            // tiles of queries that have any
  const double longest = most / 64.0, all = rows * std::max(longest - T / (128 * B), longest / 2);  // in tiles of keys
  // Weights rounded to the queries' type add an error as large as the output's own rounding: together 1.41 times it on the
  // average of many rows and keys, more in a short call's few.  A second part costs 20-25% of the products' time.  It is taken
  // where that is a small part: calls whose tiles of queries do not fill the card, and of those the sequences with which, were
  // they all like it, the call would be of 1024 products at most, of a tile with 64 keys.  Their lengths are known on the device
  // alone, and the table's width says nothing of them.  8 (2) heads of 64, bfloat16, one part | two: 500 tokens (250
  // products) 15.0 | 15.5 us, 1000 (500) 21.3 | 22.6, 16 behind 60,000 (940) 25.8 | 28.9, 400 behind 4000 (1600) 28.6 | 30.7,
  // 4 of 384 behind 20,000 (24,000) 109 | 137.  Where the kernel has to look, one part takes 1% longer, 4% over 8 bits.
  p.fine = rows > 512 ? 0 : static_cast<int>(64 * 1024 / rows);
  double least = 0;
  p.pieces = 1;
  for (int n = 1; n == 1 || (most >= 64 * n && rows * n <= 12 * 256 * waves); n *= 2) {  // tables may be far wider than streams are long
    const double groups = rows * n, len = longest / n + 1.3;
    double us = len * tile * (groups < 256 * (g->dtype == GEO_F32 ? 1 : waves - 1) ? 0.67 : 1);
    if (groups > 256 * waves) us = std::max(us, tile * ((all + 1.3 * groups) / (256 * waves) + 0.38 * len));
    if (n > 1) us += 6.3 + 0.06 * n + n * T * Hq * (DP + 4) * 8 / 6.6e6;
    if (n > 1 && us >= least) continue;
    least = us;
    p.pieces = n;
  }
  p.blocks = p.tiles * columns * p.pieces;
  return p;
}

template <typename T, typename C, int DP>
int launch_prompt(const Prompt& a, const PromptPlan& p, void* out, float* part, hipStream_t stream) {
  const size_t bytes = 2 * PromptLds<T, C, DP>::kBuffer + (a.bias.table ? static_cast<size_t>(a.heads) * a.bias_row * 4 : 0);
  constexpr bool kCanBeFine = Meet<T, C, true>::kFine;
  auto* const kernel = kCanBeFine && p.fine ? &paged_prompt<T, C, DP, kCanBeFine> : &paged_prompt<T, C, DP, false>;
  GEO_HIP_CHECK(attn::allow_lds(reinterpret_cast<const void*>(kernel), bytes));
  kernel<<<dim3(static_cast<uint32_t>(p.blocks)), dim3(kPromptThreads), bytes, stream>>>(a, p.tiles, p.pieces, a.pool.table, part,
                                                                                        static_cast<T*>(out));
  GEO_LAUNCH_CHECK("paged_prompt");
  if (p.pieces > 1) {
    constexpr int kSets = 8;
    const int64_t rows = a.T * a.Hq;
    const bool many = p.pieces > 8;
    const int64_t blocks = ceil_div(rows * (DP / 4) * (many ? kSets : 1), static_cast<int64_t>(kPromptThreads));
    GEO_REQUIRE(grid_fits(blocks, kPromptThreads), "paged attention: too many workgroups");
    if (many)
      paged_prompt_join<T, DP, kSets><<<dim3(static_cast<uint32_t>(blocks)), dim3(kPromptThreads), 0, stream>>>(a.pool.D, rows, p.pieces, part,
                                                                                                           static_cast<T*>(out));
    else
      paged_prompt_join<T, DP, 1><<<dim3(static_cast<uint32_t>(blocks)), dim3(kPromptThreads), 0, stream>>>(a.pool.D, rows, p.pieces, part,
                                                                                                       static_cast<T*>(out));
    GEO_LAUNCH_CHECK("paged_prompt_join");
  }
  return GEO_OK;
}
template <typename T, typename C>
int choose_prompt(const Prompt& a, const PromptPlan& p, void* out, float* part, hipStream_t stream) {
  switch (prompt_padded(a.pool.D)) {
    case 32: return launch_prompt<T, C, 32>(a, p, out, part, stream);
    case 64: return launch_prompt<T, C, 64>(a, p, out, part, stream);
    default: return launch_prompt<T, C, 128>(a, p, out, part, stream);
  }
}
// One query type's kernels, each in a file of its own.
template <typename T>
int prompt_of(int stored, const Prompt& a, const PromptPlan& p, void* out, float* part, hipStream_t stream) {
  if (stored == GEO_I8) return choose_prompt<T, I8>(a, p, out, part, stream);
  return stored == GEO_E4M3 ? choose_prompt<T, E4>(a, p, out, part, stream) : choose_prompt<T, T>(a, p, out, part, stream);
}

}  // namespace paged
}  // namespace geo
