// paged_cache.hip — tokens of packed sequences into the pages of a pool and out of them.
//
// A workgroup takes 64 positions of one sequence, at a multiple of 64, and one key head: a part of one
// page.  Keys are rows on both sides.  Values are turned in LDS, so that reads and writes of memory are
// contiguous on both sides.  An 8-bit row's largest magnitude is found by the lanes that hold it, and its codes
// are the products x * fl(M / a) rounded once: a fused multiply-add with 1.5 * 2^23 steps leaves them in the sum's
// last bits, so no product is rounded twice and ties are decided exactly.
//
// Bound by memory where pages are large: 131,072 tokens, 4 heads of 128, bfloat16, are written in 107 us (5.0 TB/s), 86,703 of
// 16 streams read from int8 in 52 us (5.2 TB/s).  Small heads and packets are bound by the way to the rows (offsets, page,
// rows, LDS, rows: 4 us for the least call) and e4m3 codes by vector instructions (64% of the cycles; codes in
// fours 11.9 us, one by one 14.6, for 32 packets of up to 384 tokens, 8 heads of 64).
#include <type_traits>

#include "paged.hpp"

namespace geo {
namespace paged {

constexpr int kTile = 64, kThreads = 256;

// Eight values of a row of type T, as words: unions and arrays of elements would go through memory.
using Words = uint32_t __attribute__((ext_vector_type(4)));
template <typename T>
struct Eight {
  static constexpr int kWords = sizeof(T) / 2;
  Words u[kWords];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int n = 0; n < kWords; ++n) u[n] = reinterpret_cast<const Words*>(p)[n];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int n = 0; n < kWords; ++n) reinterpret_cast<Words*>(p)[n] = u[n];
  }
  __device__ __forceinline__ float at(int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(u[e / 4][e % 4]);
    else return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(u[0][e / 2] >> (16 * (e % 2)))));
  }
  __device__ __forceinline__ void set(const float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e / 4][e % 4] = __float_as_uint(x[e]);
    } else {
#pragma unroll
      for (int n = 0; n < 4; ++n)
        u[0][n] = __builtin_bit_cast(uint16_t, static_cast<T>(x[2 * n])) | static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<T>(x[2 * n + 1]))) << 16;
    }
  }
  // Bits of the largest magnitude in float32, NaN above all; 16-bit types in pairs.
  __device__ __forceinline__ uint32_t most() const {
    if constexpr (sizeof(T) == 4) {
      uint32_t y = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) y = max(y, u[e / 4][e % 4] & 0x7fffffffu);
      return y;
    } else {
      using Pair = uint16_t __attribute__((ext_vector_type(2)));
      Pair y = {0, 0};
#pragma unroll
      for (int e = 0; e < 4; ++e) y = __builtin_elementwise_max(y, __builtin_bit_cast(Pair, u[0][e] & 0x7fff7fffu));
      const uint16_t z = max(y.x, y.y);
      return __float_as_uint(static_cast<float>(__builtin_bit_cast(T, z))) & 0x7fffffffu;
    }
  }
};
template <typename T, typename C>
struct Kept {  // eight values as the pool holds them
  static constexpr bool kNarrow = Code<C>::kNarrow;
  Eight<T> same;    // pools of the tokens' type
  uint32_t n[2];    // codes
  float scale;
  // from the row's values, by the LW lanes that share the row
  template <int LW>
  __device__ __forceinline__ void from(const Eight<T>& x) {
    if constexpr (kNarrow) {
      const RowScale s = row_scale<C>(group_most<LW>(x.most()));
      scale = s.scale;
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x.at(e);
      const uint32_t keep = s.rate > 0.f ? ~0u : 0u;
      n[0] = Code<C>::four(y, s.rate) & keep;
      n[1] = Code<C>::four(y + 4, s.rate) & keep;
    } else {
      same = x;
    }
  }
  __device__ __forceinline__ void to(Eight<T>& x) const {
    if constexpr (kNarrow) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = Code<C>::value(static_cast<uint8_t>(n[e / 4] >> (8 * (e % 4)))) * scale;
      x.set(y);
    } else {
      x = same;
    }
  }
  __device__ __forceinline__ void load(const C* p) {
    if constexpr (kNarrow) {
      const uint2 y = *reinterpret_cast<const uint2*>(p);
      n[0] = y.x;
      n[1] = y.y;
    } else {
      same.load(reinterpret_cast<const T*>(p));
    }
  }
  __device__ __forceinline__ void store(C* p) const {
    if constexpr (kNarrow) *reinterpret_cast<uint2*>(p) = uint2{n[0], n[1]};
    else same.store(reinterpret_cast<T*>(p));
  }
};

// Sixteen bytes of adjoining values of C, from and to places STRIDE apart.
template <typename C, int STRIDE>
__device__ __forceinline__ Words gather(const C* p) {
  Words y = {};
#pragma unroll
  for (int n = 0; n < static_cast<int>(16 / sizeof(C)); ++n) {
    constexpr int kBits = 8 * sizeof(C);
    using U = typename std::conditional<sizeof(C) == 4, uint32_t, typename std::conditional<sizeof(C) == 2, uint16_t, uint8_t>::type>::type;
    y[n * kBits / 32] |= static_cast<uint32_t>(reinterpret_cast<const U*>(p)[n * STRIDE]) << (n * kBits % 32);
  }
  return y;
}
template <typename C, int STRIDE>
__device__ __forceinline__ void scatter(C* p, const Words& y) {
#pragma unroll
  for (int n = 0; n < static_cast<int>(16 / sizeof(C)); ++n) {
    constexpr int kBits = 8 * sizeof(C);
    using U = typename std::conditional<sizeof(C) == 4, uint32_t, typename std::conditional<sizeof(C) == 2, uint16_t, uint8_t>::type>::type;
    reinterpret_cast<U*>(p)[n * STRIDE] = static_cast<U>(y[n * kBits / 32] >> (n * kBits % 32));
  }
}

// LDS rows of a tile's values: 16 bytes (8 of 8-bit types) more than the row, so that rows begin in other banks.
template <typename C, int LW>
constexpr int lds_row() { return 8 * LW + (sizeof(C) == 1 ? 8 : 16 / static_cast<int>(sizeof(C))); }

template <typename T, typename C, int LW>
__global__ __launch_bounds__(kThreads) void paged_write(const Pool p, const T* __restrict__ k, const T* __restrict__ v, int64_t k_st,
                                                        int64_t k_sh, int64_t v_st, int64_t v_sh, const int64_t* __restrict__ ptr,
                                                        const int64_t* __restrict__ start, int64_t T_all, int B) {
  constexpr int kRow = lds_row<C, LW>(), kGroups = kThreads / LW, kBlk = block_tokens<C>(), kPer = 16 / sizeof(C);
  __shared__ __attribute__((aligned(16))) C turned[kTile * kRow];
  const int h = static_cast<int>(blockIdx.x % p.Hk);
  const Span s = span_of<kAtMultiples>(ptr, start, B, T_all, blockIdx.x / p.Hk, kTile);
  if (s.lo >= s.hi) return;
  const int page = page_of(p, s.b, s.tile0 / p.page), off = static_cast<int>(s.tile0 % p.page);
  if (page < 0) return;
  const int64_t slot0 = (static_cast<int64_t>(page) * p.Hk + h) * p.page + off;
  C* const kp = reinterpret_cast<C*>(p.k) + slot0 * p.D;
  C* const vp = reinterpret_cast<C*>(p.v) + slot0 * p.D;
  const int lane = threadIdx.x % LW, g = threadIdx.x / LW, d = 8 * lane;
  const int64_t t0 = s.first + s.tile0 - s.start;
  Eight<T> kx[kTile / kGroups], vx[kTile / kGroups];
#pragma unroll
  for (int n = 0; n < kTile / kGroups; ++n) {
    const int r = g + n * kGroups;
    kx[n] = vx[n] = Eight<T>{};
    if (r >= s.lo && r < s.hi && d < p.D) {
      kx[n].load(k + (t0 + r) * k_st + h * k_sh + d);
      vx[n].load(v + (t0 + r) * v_st + h * v_sh + d);
    }
  }
#pragma unroll
  for (int n = 0; n < kTile / kGroups; ++n) {
    const int r = g + n * kGroups;
    const bool in = r >= s.lo && r < s.hi;
    Kept<T, C> ck, cv;
    ck.template from<LW>(kx[n]);
    cv.template from<LW>(vx[n]);
    if (in && d < p.D) ck.store(kp + r * p.D + d);
    if constexpr (Code<C>::kNarrow) {
      if (in && lane == 0) {
        p.ks[slot0 + r] = ck.scale;
        p.vs[slot0 + r] = cv.scale;
      }
    }
    cv.store(turned + r * kRow + d);
  }
  __syncthreads();
  const int pieces = kTile * p.D / kPer;
  for (int x = threadIdx.x; x < pieces; x += kThreads) {
    const int row = x / (kBlk / kPer), e = row % p.D, r0 = row / p.D * kBlk + x % (kBlk / kPer) * kPer;
    if (r0 >= s.hi || r0 + kPer <= s.lo) continue;
    if (r0 >= s.lo && r0 + kPer <= s.hi) {
      reinterpret_cast<Words*>(vp)[x] = gather<C, kRow>(turned + r0 * kRow + e);
    } else {
      for (int n = max(s.lo - r0, 0); n < min(s.hi - r0, kPer); ++n) vp[x * kPer + n] = turned[(r0 + n) * kRow + e];
    }
  }
}

template <typename T, typename C, int LW>
__global__ __launch_bounds__(kThreads) void paged_read(const Pool p, T* __restrict__ k, T* __restrict__ v,
                                                       const int64_t* __restrict__ ptr, const int64_t* __restrict__ start,
                                                       int64_t T_all, int B) {
  constexpr int kRow = lds_row<C, LW>(), kGroups = kThreads / LW, kBlk = block_tokens<C>(), kPer = 16 / sizeof(C);
  __shared__ __attribute__((aligned(16))) C turned[kTile * kRow];
  const int h = static_cast<int>(blockIdx.x % p.Hk);
  const int64_t tile = blockIdx.x / p.Hk;
  const int lane = threadIdx.x % LW, g = threadIdx.x / LW, d = 8 * lane;
  auto fill = [&](int64_t t, float x) {
    Eight<T> y;
    y.set({x, x, x, x, x, x, x, x});
    if (d < p.D) {
      y.store(k + (t * p.Hk + h) * p.D + d);
      y.store(v + (t * p.Hk + h) * p.D + d);
    }
  };
  if (ptr) {  // rows of no sequence, by the workgroups of the same number
    const int64_t first = ptr[0], end = ptr[B];
    for (int r = g; r < kTile; r += kGroups) {
      const int64_t t = tile * kTile + r;
      if (t < T_all && (t < first || t >= end)) fill(t, 0.f);
    }
  }
  const Span s = span_of<kAtMultiples>(ptr, start, B, T_all, tile, kTile);
  const int64_t t0 = s.first + s.tile0 - s.start;
  for (int64_t r = g; r < s.before; r += kGroups) fill(s.first + r, __builtin_nanf(""));
  if (s.lo >= s.hi) return;
  const int page = page_of(p, s.b, s.tile0 / p.page), off = static_cast<int>(s.tile0 % p.page);
  if (page < 0) {
    for (int r = g; r < kTile; r += kGroups)
      if (r >= s.lo && r < s.hi) fill(t0 + r, __builtin_nanf(""));
    return;
  }
  const int64_t slot0 = (static_cast<int64_t>(page) * p.Hk + h) * p.page + off;
  const C* const kp = reinterpret_cast<const C*>(p.k) + slot0 * p.D;
  const C* const vp = reinterpret_cast<const C*>(p.v) + slot0 * p.D;
  Kept<T, C> kx[kTile / kGroups];
#pragma unroll
  for (int n = 0; n < kTile / kGroups; ++n) {
    const int r = g + n * kGroups;
    if (r >= s.lo && r < s.hi && d < p.D) {
      kx[n].load(kp + r * p.D + d);
      if constexpr (Code<C>::kNarrow) kx[n].scale = p.ks[slot0 + r];
    }
  }
  const int pieces = kTile * p.D / kPer;
  for (int x = threadIdx.x; x < pieces; x += kThreads) {
    const int row = x / (kBlk / kPer), e = row % p.D, r0 = row / p.D * kBlk + x % (kBlk / kPer) * kPer;
    if (r0 >= s.hi || r0 + kPer <= s.lo) continue;
    scatter<C, kRow>(turned + r0 * kRow + e, reinterpret_cast<const Words*>(vp)[x]);
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kTile / kGroups; ++n) {
    const int r = g + n * kGroups;
    if (r >= s.lo && r < s.hi && d < p.D) {
      Eight<T> x;
      kx[n].to(x);
      x.store(k + ((t0 + r) * p.Hk + h) * p.D + d);
      Kept<T, C> cv;
      cv.load(turned + r * kRow + d);
      if constexpr (Code<C>::kNarrow) cv.scale = p.vs[slot0 + r];
      cv.to(x);
      x.store(v + ((t0 + r) * p.Hk + h) * p.D + d);
    }
  }
}

struct Move {  // arguments of either direction
  const void *k, *v;
  int64_t k_st, k_sh, v_st, v_sh;
  const int64_t *ptr, *start;
  int64_t T, B;
  bool write;
};
template <typename T, typename C, int LW>
int launch_move(const Pool& p, const Move& m, hipStream_t stream) {
  const int64_t blocks = tiles_of<kAtMultiples>(m.T, m.B, kTile) * p.Hk;
  GEO_REQUIRE(grid_fits(blocks, kThreads), "paged cache: too many workgroups");
  const dim3 grid(static_cast<uint32_t>(blocks));
  if (m.write)
    paged_write<T, C, LW><<<grid, dim3(kThreads), 0, stream>>>(p, static_cast<const T*>(m.k), static_cast<const T*>(m.v), m.k_st,
                                                              m.k_sh, m.v_st, m.v_sh, m.ptr, m.start, m.T, static_cast<int>(m.B));
  else
    paged_read<T, C, LW><<<grid, dim3(kThreads), 0, stream>>>(p, static_cast<T*>(const_cast<void*>(m.k)),
                                                             static_cast<T*>(const_cast<void*>(m.v)), m.ptr, m.start, m.T,
                                                             static_cast<int>(m.B));
  GEO_LAUNCH_CHECK(m.write ? "paged_write" : "paged_read");
  return GEO_OK;
}
template <typename T, typename C>
int choose_lanes(const Pool& p, const Move& m, hipStream_t stream) {
  if (p.D <= 32) return launch_move<T, C, 4>(p, m, stream);
  return p.D <= 64 ? launch_move<T, C, 8>(p, m, stream) : launch_move<T, C, 16>(p, m, stream);
}
template <typename T>
int choose_stored(int stored, const Pool& p, const Move& m, hipStream_t stream) {
  if (stored == GEO_I8) return choose_lanes<T, I8>(p, m, stream);
  return stored == GEO_E4M3 ? choose_lanes<T, E4>(p, m, stream) : choose_lanes<T, T>(p, m, stream);
}

int move(const char* name, const geo_paged_t* cache, int dtype, const Move& m, void* stream) {
  Pool p;
  if (const int rc = pool_args(name, cache, &p)) return rc;
  GEO_REQUIRE(type_ok(dtype, cache->stored), "%s: tokens of type code %d, a pool of %d", name, dtype, static_cast<int>(cache->stored));
  GEO_REQUIRE(m.T >= 0 && m.T < (int64_t(1) << 31) - 64 && m.B >= 0 && m.B < (int64_t(1) << 30) && (m.ptr || m.B <= 1),
              "%s: %lld tokens of %lld sequences%s", name, static_cast<long long>(m.T), static_cast<long long>(m.B),
              m.ptr ? "" : " without ptr");
  if (m.T == 0) return GEO_OK;
  GEO_REQUIRE(m.B >= 1, "%s: tokens of no sequence", name);
  const int size = dtype == GEO_F32 ? 4 : 2;
  auto in_pieces = [size](const void* x, int64_t st, int64_t sh) {
    return x && reinterpret_cast<uintptr_t>(x) % 16 == 0 && st * size % 16 == 0 && sh * size % 16 == 0;
  };
  GEO_REQUIRE(in_pieces(m.k, m.k_st, m.k_sh) && in_pieces(m.v, m.v_st, m.v_sh),
              "%s: null k or v, or rows not on multiples of 16 bytes", name);
  if (dtype == GEO_F32) return choose_stored<float>(cache->stored, p, m, as_stream(stream));
  if (dtype == GEO_BF16) return choose_stored<__bf16>(cache->stored, p, m, as_stream(stream));
  return choose_stored<_Float16>(cache->stored, p, m, as_stream(stream));
}

}  // namespace paged
}  // namespace geo

extern "C" int geo_paged_write(const geo_paged_t* cache, int dtype, const void* k, const void* v, int64_t k_token, int64_t k_head,
                               int64_t v_token, int64_t v_head, const int64_t* ptr, const int64_t* start, int64_t tokens,
                               int64_t batch, void* stream) {
  return geo::paged::move("paged write", cache, dtype,
                          {k, v, k_token, k_head, v_token, v_head, ptr, start, tokens, batch, true}, stream);
}

extern "C" int geo_paged_read(const geo_paged_t* cache, int dtype, const int64_t* ptr, const int64_t* start, int64_t tokens,
                              int64_t batch, void* k, void* v, void* stream) {
  GEO_REQUIRE(tokens == 0 || k != v, "paged read: one output for keys and values");
  return geo::paged::move("paged read", cache, dtype, {k, v, 0, 0, 0, 0, ptr, start, tokens, batch, false}, stream);
}
