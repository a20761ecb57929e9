// paged.hpp — keys and values of streams in pages of a shared pool: the layout, the 8-bit codes, and
// where the tokens of packed sequences lie.
//
// k [pages, Hk, page, D] row by row; v [pages, Hk, page / blk, D, blk], blk tokens to 64 bytes: a matrix
// instruction's operand of the values is 16 bytes of one dimension's tokens, so a wave's read of 16
// dimensions is one contiguous KiB and nothing is turned on the way.  Both take 64 D bytes for blk
// tokens, so a token block begins at the same offset in either.
#pragma once

#include <type_traits>
#include <utility>

#include "attention_args.hpp"

namespace geo {
namespace paged {

using attn::kInf;
using attn::exp2_hw;
using attn::kLog2e;

// Element types of 8-bit pools: whole numbers and e4m3 floats, each token and head with a scale.
struct I8 { uint8_t bits; };
struct E4 { uint8_t bits; };

template <typename C> struct Code { static constexpr bool kNarrow = false; };
template <> struct Code<I8> {
  static constexpr bool kNarrow = true;
  static constexpr float kMost = 127.f;
  // The product x rate, rounded once: the sum with 1.5 * 2^23 has steps of 1 (to even).
  static __device__ __forceinline__ float round(float x, float rate) {
    constexpr float kStep1 = 12582912.f;
    return fmaf(x, rate, kStep1) - kStep1;
  }
  static __device__ __forceinline__ uint8_t bits(float y) { return static_cast<uint8_t>(static_cast<int>(y)); }
  static __device__ __forceinline__ float value(uint8_t b) { return static_cast<float>(static_cast<int8_t>(b)); }
  // Four codes of such products: that sum's low byte is the code.
  static __device__ __forceinline__ uint32_t four(const float* x, float rate) {
    uint32_t y[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) y[n] = __float_as_uint(fmaf(x[n], rate, 12582912.f));
    return __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0400u) | __builtin_amdgcn_perm(y[3], y[2], 0x04000c0cu);
  }
};
template <> struct Code<E4> {
  static constexpr bool kNarrow = true;
  static constexpr float kMost = 448.f;
  // The same with steps of an eighth of the product's power of two, at least 2^-9.
  static __device__ __forceinline__ float round(float x, float rate) {
    const uint32_t power = max(__float_as_uint(x * rate) & 0x7f800000u, 0x3c800000u);
    const float big = __uint_as_float(power + ((20u << 23) | 0x400000u));
    return fmaf(x, rate, big) - big;
  }
  static __device__ __forceinline__ uint8_t bits(float y) {
    return static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false));
  }
  static __device__ __forceinline__ float value(uint8_t b) { return __builtin_amdgcn_cvt_f32_fp8(b, 0); }
  static __device__ __forceinline__ uint32_t four(const float* x, float rate) {
    const uint32_t lo = __builtin_amdgcn_cvt_pk_fp8_f32(round(x[0], rate), round(x[1], rate), 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(round(x[2], rate), round(x[3], rate), lo, true);
  }
};

using attn::bf16x8;
using attn::f16x8;
union Bytes16 {
  uint4 u;
  uint32_t w[4];
  float f[4];
  bf16x8 b;
  f16x8 h;
};
// Eight codes (two words) as bf16 or float16, which hold them exactly.
template <typename C>
__device__ __forceinline__ bf16x8 decode8(uint32_t lo, uint32_t hi) {
  Bytes16 y;
  // keeps the compiler from taking the bytes apart where they were loaded, an iteration earlier
  asm("" : "+v"(lo), "+v"(hi));
  if constexpr (__is_same(C, I8)) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const uint32_t x = n < 2 ? lo : hi;
      const float a = static_cast<float>(static_cast<int8_t>(x >> (16 * (n & 1))));
      const float b = static_cast<float>(static_cast<int8_t>(x >> (16 * (n & 1) + 8)));
      y.w[n] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);  // their upper halves
    }
  } else {
    y.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false));
    y.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true));
    y.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false));
    y.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true));
  }
  return y.b;
}
template <typename C>
__device__ __forceinline__ f16x8 decode8_f16(uint32_t lo, uint32_t hi) {
  Bytes16 y;
  if constexpr (__is_same(C, I8)) {
#pragma unroll
    for (int n = 0; n < 8; ++n)
      y.h[n] = static_cast<_Float16>(static_cast<float>(static_cast<int8_t>((n < 4 ? lo : hi) >> (8 * (n & 3)))));
  } else {
    y.w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, false));
    y.w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.f, true));
    y.w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, false));
    y.w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.f, true));
  }
  return y.h;
}

// Eight float32 values as the sum of PARTS bf16 operands: 8, 16 or all 24 bits of them.  Codes are exact in
// bf16, so products of 8-bit pools keep what the queries' type holds: one part for bfloat16, two for
// float16, three for float32.
template <int PARTS, typename F>
__device__ __forceinline__ void split8(const float (&x)[8], F (&y)[PARTS]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float r = x[e];
#pragma unroll
    for (int n = 0; n < PARTS; ++n) {
      y[n][e] = static_cast<std::remove_reference_t<decltype(y[n][0])>>(r);
      if (n + 1 < PARTS) r -= static_cast<float>(y[n][e]);
    }
  }
}
// The second of their parts alone.
template <typename F>
__device__ __forceinline__ F second8(const float (&x)[8]) {
  F y;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    using E = std::remove_reference_t<decltype(y[0])>;
    float r = x[e];
    asm volatile("" : "+v"(r));  // as in faint8
    y[e] = static_cast<E>(r - static_cast<float>(static_cast<E>(r)));
  }
  return y;
}
template <typename T> constexpr int parts_of() { return sizeof(T) == 4 ? 3 : __is_same(T, _Float16) ? 2 : 1; }

// Weights of operands of type V: kLazy is how far (in units of log 2) scores may exceed the maximum that weights refer to.
// Many keys 2^20 and more below one whose value is small are what a row consists of, and float16 has no digits for weights
// that small.  Its weights are formed 2^11 larger than those of other types, up to 2^15 then; of those that are still below
// 2^-14 (2^-9 where two parts are to keep 16 bits), what the parts leave is taken 2^38 larger, as a further
// operand whose products join sums brought up as far.  These are powers of two, so other rows' sums come back as they
// were.  Looking for such weights costs prompts 3-7% (8 pieces of up to 1024 behind 2048, 16 (4) heads of 64: 106 | 113 us; 32
// packets of up to 384 behind 4000 150 | 154), steps nothing.  Where scores spread so far that most tiles hold some, a deviation of 4,
// prompts take 1.4 to 1.5 times as long (heads of 128: 215 | 300 us; of 2 215 | 215, where weights 2^7 larger, and scores 8 above the maximum, took 237), steps 3%.
template <typename V>
struct Faint {
  static constexpr bool kHalf = __is_same(V, _Float16);
  static constexpr float kLift = kHalf ? 11.f : 0.f, kLazy = kHalf ? 4.f : 8.f, kUp = 0x1p38f, kDown = 0x1p-38f;
  static __host__ __device__ constexpr float below(int parts) { return parts > 1 ? 0x1p-9f : 0x1p-14f; }
  // What scores are taken less by, of the largest: itself where the difference would be rounded up past what V holds.
  static __device__ __forceinline__ float lifted(float most) { return kHalf && fabsf(most) < 0x1p20f ? most - kLift : most; }
};
// What PARTS float16 parts leave of eight weights, of those that are faint, 2^38 larger.
template <int PARTS>
__device__ __forceinline__ f16x8 faint8(const float (&x)[8]) {
  f16x8 y;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float r = x[e];
    asm volatile("" : "+v"(r));  // formed again: the parts' remainders kept for this would take the registers
    const bool small = r < Faint<_Float16>::below(PARTS);
#pragma unroll
    for (int n = 0; n < PARTS; ++n) r -= static_cast<float>(static_cast<_Float16>(r));
    y[e] = static_cast<_Float16>(small ? r * Faint<_Float16>::kUp : 0.f);
  }
  return y;
}

// How a row of largest magnitude a (its bits, so that NaN counts as most) is kept: values are code * scale,
// codes the exact products x * rate rounded once.  Rows below 2^-100 are kept as zeros; one with an
// infinity or a NaN has a scale of NaN and reads back so.
struct RowScale { float scale, rate; };
template <typename C>
__device__ __forceinline__ RowScale row_scale(uint32_t most_bits) {
  const float a = __uint_as_float(most_bits);
  if (most_bits >= 0x7f800000u) return {__builtin_nanf(""), 0.f};
  if (a < 0x1p-100f) return {0.f, 0.f};
  return {a / Code<C>::kMost, Code<C>::kMost / a};
}
template <typename C>
__device__ __forceinline__ float encode(float x, float rate) { return rate > 0.f ? Code<C>::round(x, rate) : 0.f; }

// Largest of unsigned numbers over a group of LW = 4, 8 or 16 lanes, in all of them.
template <int LW>
__device__ __forceinline__ uint32_t group_most(uint32_t x) {
  x = max(x, dpp_u32<kDppXor1>(x));
  x = max(x, dpp_u32<kDppXor2>(x));
  if constexpr (LW >= 8) x = max(x, dpp_u32<kDppHalfMirror>(x));
  if constexpr (LW >= 16) x = max(x, dpp_u32<kDppMirror>(x));
  return x;
}

// x[n] times what lane n of the 16 holds.
template <int... N>
__device__ __forceinline__ void by_group_of(float* x, float y, std::integer_sequence<int, N...>) {
  constexpr int kRowBroadcast = 0x150;
  ((x[N] *= __uint_as_float(dpp0_u32<kRowBroadcast + N>(__float_as_uint(y)))), ...);
}
template <int N>
__device__ __forceinline__ void by_group(float (&x)[N], float y) { by_group_of(x, y, std::make_integer_sequence<int, N>()); }

struct Pool {
  char *k, *v;
  float *ks, *vs;        // [pages, Hk, page], of 8-bit pools
  const int32_t* table;  // [streams, columns]: page of each `page` tokens
  int64_t table_st;
  int pages, columns, page, Hk, D;
};

template <typename C>
constexpr int block_tokens() { return 64 / static_cast<int>(sizeof(C)); }

// The packed sequences cut into tiles of U positions: at multiples of U (kCuts = 2), or from each sequence's
// first on (kCuts = 1).  Sequence b has at most n / U + kCuts of them, so its tiles are numbered from
// ptr[b] / U + kCuts b on; numbers without a tile are idle.
constexpr int kAtMultiples = 2, kFromFirst = 1;
template <int kCuts>
inline int64_t tiles_of(int64_t tokens, int64_t batch, int U) { return tokens / U + kCuts * batch; }

struct Span {
  int64_t first, start;  // row of the sequence's first token, and its position
  int64_t tile0;         // the tile's first position
  int b, lo, hi;         // the sequence; the tile's places that have tokens, lo .. hi - 1 (none: lo >= hi)
  int64_t before;        // on a sequence's first tile: how many of its tokens have negative positions
  int64_t middle;        // of a tile with tokens: the position halfway through the sequence's
};
// A start in a range in which nothing overflows; what lies as far out has no page either way.
__device__ __forceinline__ int64_t start_of(const int64_t* start, int b) {
  return start ? min(max(start[b], -(int64_t(1) << 60)), int64_t(1) << 60) : 0;
}
// Wave-wide: 64 sequences are looked at together.
template <int kCuts>
__device__ __forceinline__ Span span_of(const int64_t* ptr, const int64_t* start, int B, int64_t T, int64_t tile, int U) {
  const int lane = threadIdx.x & 63;
  auto offset = [&](int b) { return ptr ? min(max(ptr[b], int64_t(0)), T) : b ? T : int64_t(0); };
  auto tile_of = [&](int64_t first, int b) { return static_cast<uint32_t>(first) / static_cast<uint32_t>(U) + kCuts * static_cast<int64_t>(b); };
  int lo = 0, len = B;
  bool some = true;
  do {
    const int step = (len + 63) / 64, at = lo + lane * step;
    const bool ok = at < lo + len && tile_of(offset(at), at) <= tile;
    const int n = __popcll(__ballot(ok));
    some = some && n > 0;
    const int next = lo + max(n - 1, 0) * step;
    len = min(step, lo + len - next);
    lo = next;
  } while (len > 1);
  const int b = __builtin_amdgcn_readfirstlane(lo);
  Span s{offset(b), start_of(start, b), 0, b, 0, 0, 0, 0};
  const int64_t n = offset(b + 1) - s.first, from = max(s.start, int64_t(0)), end = s.start + n;
  const int64_t turn = tile - tile_of(s.first, b);
  s.tile0 = (kCuts == kAtMultiples ? from / U * U : from) + turn * U;
  if (some && turn == 0 && s.start < 0 && n > 0) s.before = s.start < -n ? n : -s.start;
  if (!some || n <= 0 || s.tile0 >= end) return s;
  s.middle = (from + end) / 2;
  s.lo = static_cast<int>(max(from - s.tile0, int64_t(0)));
  s.hi = static_cast<int>(min(end - s.tile0, static_cast<int64_t>(U)));
  return s;
}

// The page of a stream's column, or -1 where the table or the pool has none.
__device__ __forceinline__ int page_of(const Pool& p, int b, int64_t column) {
  if (column >= p.columns) return -1;
  const int n = p.table[b * p.table_st + column];
  return static_cast<uint32_t>(n) < static_cast<uint32_t>(p.pages) ? n : -1;
}

// Checks on the host; fills *pool.  Without streams there is no table: a tensor without elements has no address.
inline int pool_args(const char* name, const geo_paged_t* g, Pool* pool, bool streams = true) {
  GEO_REQUIRE(g, "%s: null arguments", name);
  const bool narrow = g->stored == GEO_I8 || g->stored == GEO_E4M3;
  GEO_REQUIRE(narrow || g->stored == GEO_F32 || g->stored == GEO_BF16 || g->stored == GEO_F16, "%s: pool type code %d", name,
              static_cast<int>(g->stored));
  GEO_REQUIRE(g->kv_heads >= 1 && g->kv_heads < (1 << 16), "%s: %d key heads", name, g->kv_heads);
  GEO_REQUIRE(g->head_dim >= 8 && g->head_dim <= 128 && g->head_dim % (narrow ? 16 : 8) == 0,
              "%s: head size %d (a multiple of %d up to 128)", name, g->head_dim, narrow ? 16 : 8);
  GEO_REQUIRE(g->page >= 64 && g->page % 64 == 0 && g->page <= (1 << 20), "%s: pages of %d tokens (a multiple of 64 up to 2^20)",
              name, g->page);
  GEO_REQUIRE(g->pages >= 1 && g->pages < (int64_t(1) << 31), "%s: %lld pages", name, static_cast<long long>(g->pages));
  GEO_REQUIRE(g->columns >= 1 && g->columns < (int64_t(1) << 30) && g->columns * g->page < (int64_t(1) << 30), "%s: a table of %lld columns of %d tokens (below 2^30)",
              name, static_cast<long long>(g->columns), g->page);
  auto aligned = [](const void* p) { return p && reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  GEO_REQUIRE(aligned(g->k) && aligned(g->v) && g->k != g->v, "%s: null pool, not on 16 bytes, or one for both", name);
  GEO_REQUIRE(!narrow || (aligned(g->k_scale) && aligned(g->v_scale) && g->k_scale != g->v_scale),
              "%s: an 8-bit pool needs scales, on 16 bytes", name);
  GEO_REQUIRE(g->table || !streams, "%s: null table", name);
  *pool = Pool{static_cast<char*>(g->k), static_cast<char*>(g->v), g->k_scale, g->v_scale, g->table, g->table_stream,
               static_cast<int>(g->pages), static_cast<int>(g->columns), g->page, g->kv_heads, g->head_dim};
  return GEO_OK;
}
// Numbers that a size can be formed of (the rest is checked where the call itself is).
inline bool sizes_ok(const geo_paged_t& c, int64_t batch, int heads) {
  return batch >= 1 && batch < (int64_t(1) << 31) && c.kv_heads >= 1 && c.kv_heads < (1 << 16) && heads >= c.kv_heads && heads < (1 << 20) &&
         heads % c.kv_heads == 0 && c.page >= 64 && c.page <= (1 << 20) && c.columns >= 1 && c.columns < (int64_t(1) << 30) &&
         c.columns * c.page < (int64_t(1) << 30);
}
inline bool type_ok(int dtype, int stored) {
  return (dtype == GEO_F32 || dtype == GEO_BF16 || dtype == GEO_F16) &&
         (stored == dtype || stored == GEO_I8 || stored == GEO_E4M3);
}

}  // namespace paged
}  // namespace geo
