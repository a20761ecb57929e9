// attention_tile.hpp — what the attention kernels share: element types and their matrix products,
// tiles of rows in LDS, which keys a query sees, the relative bias of a tile.
//
// Every product is one of two forms of D[m][n] += sum_k A[m][k] B[k][n] on 32x32 tiles, k in
// chunks of 16.  A lane holds column (A: row) lane % 32 and, with half = lane / 32, eight values
// of k: 8 half + 0..7 for operands read from memory.  The result's register r of a lane is row
// 8 (r / 4) + 4 half + r % 4 of column lane % 32, so a result turned operand without leaving its
// lane has the eight rows 16 c + 8 (j / 4) + 4 half + j % 4 as chunk c: the other operand of such
// a product is read in the same order of k (frag_down), and a softmax over keys is a loop over a
// lane's own registers and one exchange between the halves.
#pragma once

#include "common.hpp"

namespace geo {
namespace attn {

using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using f32x8 = float __attribute__((ext_vector_type(8)));
using f32x16 = float __attribute__((ext_vector_type(16)));
using i16x4 = short __attribute__((ext_vector_type(4)));

template <typename T> struct Type;
template <> struct Type<__bf16> {
  using Frag = bf16x8;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // x plus 0 times the packed values: x, or NaN where one of them is infinite or NaN
  static __device__ __forceinline__ float probe(uint32_t w, float x) {
    using Two = __bf16 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(Two, w), Two{}, x, false);
  }
};
template <> struct Type<_Float16> {
  using Frag = f16x8;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float probe(uint32_t w, float x) {
    using Two = _Float16 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(Two, w), Two{}, x, false);
  }
};
// float32: eight products with one k of each half, which cover the same sixteen k.
template <> struct Type<float> {
  using Frag = f32x8;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ float probe(uint32_t w, float x) { return fmaf(__uint_as_float(w), 0.f, x); }
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_huge_valf();
constexpr float kMost = 0x1.fffffep127f;  // the largest finite float32

// Log-sums above this are rounded by more than 2^-12, from 10^8 on they keep nothing of a sum of several weights.
// Biases that a query's keys share bring that about (scores as large leave it one key, and are rounded as much
// themselves), so with a bias the forward keeps the factor that such a row's exp2(score - log-sum) lack.
constexpr float kFarSum = 4096.f;
__device__ __forceinline__ bool far_sum(float lse) { return fabsf(lse) > kFarSum && lse < kInf; }

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// The value of the same column in the wave's other half combined with this lane's.
__device__ __forceinline__ float halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Rows row0 .. end - 1 of a head as a buffer: reads past them give zeros.  A row's offset is a
// multiple of the stride (at least D values), so a piece of row r lies inside iff r < end - row0.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const void* base, int64_t stride_bytes, int row0, int end) {
  const int64_t bytes = (end - row0) * stride_bytes;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(static_cast<const char*>(base)) + row0 * stride_bytes, 0,
                                           static_cast<int>(min(bytes, int64_t(0x7fffffff))), 0x00020000);
}

// A tile of ROWS rows in LDS, DP values each (a head's D, zeros beyond), in pieces of 16 bytes.  A
// row is padded so that one piece of eight neighbouring rows, which a read along the rows takes at a
// time, lies in eight different groups of the 64 banks, and the 64 bytes of four rows that a
// transposing read takes meet at most in pairs.  (Turning the pieces by row instead kept those apart
// too, but its addresses took registers that the products need: dq at D = 128 695 us, so 530.)
template <typename T, int DP, int ROWS, int NT>
struct Tile {
  static constexpr int kPer = 16 / sizeof(T);        // values in a piece
  static constexpr int kChunks = DP / kPer;          // pieces of a row
  static constexpr int kRow = DP * sizeof(T) + (DP * sizeof(T) == 256 ? 48 : 16);  // bytes from row to row
  static constexpr int kLoads = ROWS * kChunks / NT; // per thread
  static constexpr int kBytes = ROWS * kRow;
  static_assert(ROWS * kChunks % NT == 0, "a thread loads whole pieces");

  uint4 reg[kLoads];
  uint32_t off[kLoads];  // of the thread's pieces from the tile's first row, in bytes

  __device__ __forceinline__ void init(int64_t stride_bytes, int D) {
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int c = threadIdx.x + n * NT, row = c / kChunks, at = c % kChunks * kPer;
      off[n] = at < D ? static_cast<uint32_t>(row * static_cast<uint32_t>(stride_bytes) + at * sizeof(T)) : 0x80000000u;
    }
  }
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rows) {
#pragma unroll
    for (int n = 0; n < kLoads; ++n)
      reg[n] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rows, off[n], 0, 0));
  }
  static __device__ __forceinline__ uint4* place(T* lds, int n) {
    const int c = threadIdx.x + n * NT, row = c / kChunks, at = c % kChunks;
    return reinterpret_cast<uint4*>(reinterpret_cast<char*>(lds) + row * kRow + (at << 4));
  }
  // Rows whose bit is off as zeros (`some`: there may be such rows).
  __device__ __forceinline__ void drop(uint64_t rows, bool some) {
    if (!some) return;
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int row = (threadIdx.x + n * NT) / kChunks;
      if (!((rows >> row) & 1)) reg[n] = make_uint4(0, 0, 0, 0);
    }
  }
  __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
    for (int n = 0; n < kLoads; ++n) *place(lds, n) = reg[n];
  }
  // The same with zeros in the place of infinities and NaN, whose rows' bits go to `wild` (LDS): a
  // product down the rows gives every column's query or key a weight for every row, and a weight
  // of 0 would not keep them from the ones that do not see the row.  add_wild adds them where the
  // row is seen.
  __device__ __forceinline__ void store_finite(T* lds, unsigned long long* wild) const {
    float x = 0.f;
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      *place(lds, n) = reg[n];
      x = Type<T>::probe(reg[n].x, x);
      x = Type<T>::probe(reg[n].y, x);
      x = Type<T>::probe(reg[n].z, x);
      x = Type<T>::probe(reg[n].w, x);
    }
    if (x == 0.f) return;
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      union { uint4 u; T t[kPer]; } v;
      v.u = reg[n];
      bool any = false;
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (!(fabsf(static_cast<float>(v.t[e])) < kInf)) {
          v.t[e] = static_cast<T>(0.f);
          any = true;
        }
      if (any) {
        atomicOr(wild, 1ull << ((threadIdx.x + n * NT) / kChunks));
        *place(lds, n) = v.u;
      }
    }
  }
  // The stored pieces of this thread times by(row).
  template <typename By>
  static __device__ __forceinline__ void scale_rows(T* lds, By by) {
#pragma unroll 1
    for (int n = 0; n < kLoads; ++n) {
      const float x = by((threadIdx.x + n * NT) / kChunks);
      union { uint4 u; T t[kPer]; } v;
      v.u = *place(lds, n);
#pragma unroll
      for (int e = 0; e < kPer; ++e) v.t[e] = static_cast<T>(static_cast<float>(v.t[e]) * x);
      *place(lds, n) = v.u;
    }
  }
  // Operand with this lane's row `row0 + lane % 32` (row0 a multiple of 32), k = 16 kc + 8 half + 0..7
  // along the row.
  static __device__ __forceinline__ typename Type<T>::Frag frag_along(const T* lds, int row0, int kc) {
    const int lane = threadIdx.x & 63, half = lane >> 5, r = lane & 31;
    return *reinterpret_cast<const typename Type<T>::Frag*>(reinterpret_cast<const char*>(lds) + (row0 + r) * kRow +
                                                            (16 * kc + 8 * half) * sizeof(T));
  }
  // Operand with this lane's column `32 mt + lane % 32`, k down the rows in a result's order:
  // rows row0 + 8 (j / 4) + 4 half + j % 4 (row0 a multiple of 16).  For 2-byte types by the
  // transposing LDS read, which gives lane l of sixteen column l of the 4 x 16 values that the
  // sixteen address, four of a row each.
  static __device__ __forceinline__ typename Type<T>::Frag frag_down(const T* lds, int row0, int mt) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    typename Type<T>::Frag f;
    if constexpr (sizeof(T) == 2) {
      using LdsI16x4 = __attribute__((address_space(3))) i16x4;
      union { i16x4 h[2]; typename Type<T>::Frag f; } u;
      const char* p = reinterpret_cast<const char*>(lds) + (row0 + 4 * half + ((lane & 15) >> 2)) * kRow +
                      (32 * mt + (lane & 16) + 4 * (lane & 3)) * sizeof(T);
      u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4*)p);
      u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4*)(p + 8 * kRow));
      f = u.f;
    } else {
      const int x = 32 * mt + (lane & 31);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = 8 * (j >> 2) + 4 * half + (j & 3);
        f[j] = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(lds) + (row0 + r) * kRow + 4 * x);
      }
    }
    return f;
  }
};

// A value that all lanes hold, in scalar registers.
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
  return static_cast<uint64_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x >> 32))) << 32 |
         static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x)));
}

// x where bit n of `word` is set, else `other`: two instructions, with no condition mask.
__device__ __forceinline__ float keep_bit(float x, uint32_t word, int n, float other) {
  const uint32_t m = static_cast<uint32_t>(__builtin_amdgcn_sbfe(word, n, 1));
  return __uint_as_float((__float_as_uint(x) & m) | (__float_as_uint(other) & ~m));
}

// At the head of a branch on what the whole wave agrees on, with a value that the branch works from:
// keeps the compiler from carrying out the branch's instructions in every case.
__device__ __forceinline__ void stay_branch(uint32_t& x) { asm volatile("" : "+v"(x)); }

// The order of a product's LDS reads and matrix instructions, for the instructions written before it:
// AHEAD reads first, then one more behind each of the TOTAL matrix instructions that still has one to
// come (PER reads to an instruction).  Left alone the compiler, short of registers, reads one operand,
// waits for it (about 100 clocks), multiplies (32) and reads the next.
template <int TOTAL, int AHEAD, int PER>
__device__ __forceinline__ void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD * PER, 0);
#pragma unroll
  for (int n = 0; n < TOTAL - AHEAD; ++n) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}

// Registers 8 c .. 8 c + 7 of a result as an operand's chunk c.  Rounded to the inputs' type: the
// matrix units multiply 16-bit types only by their like, and a weight's relative error of half a
// unit is of the size of the output's own rounding.
template <typename T>
__device__ __forceinline__ typename Type<T>::Frag frag_of(const f32x16& x, int c) {
  typename Type<T>::Frag f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = static_cast<T>(x[8 * c + j]);
  return f;
}

// Operand with this lane's row of global memory, as frag_along; zero where !in or beyond D, the
// signs turned by `flip` (0 or the sign bit).
template <typename T>
__device__ __forceinline__ typename Type<T>::Frag frag_global(const T* row, int kc, int D, bool in, uint32_t flip = 0) {
  const int at = 16 * kc + 8 * ((threadIdx.x & 63) >> 5);
  const bool ok = in && at < D;
  union { uint4 u[sizeof(T) / 2]; typename Type<T>::Frag f; } x;
  const uint4* p = reinterpret_cast<const uint4*>(row + (ok ? at : 0));
#pragma unroll
  for (int n = 0; n < static_cast<int>(sizeof(T) / 2); ++n) {
    x.u[n] = p[n];
    if (!ok) x.u[n] = make_uint4(0, 0, 0, 0);
    if (flip) {
      const uint32_t m = sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
      x.u[n].x ^= m; x.u[n].y ^= m; x.u[n].z ^= m; x.u[n].w ^= m;
    }
  }
  return x.f;
}

// Infinities and NaN of a tile's rows to the columns that see their row (`vis`, whose lane holds
// column lane % 32): as they are, with weights that are never negative, or as NaN.
template <typename T, int MT, bool AS_NAN>
__device__ __forceinline__ void add_wild(const T* base, int64_t stride, int row0, uint64_t wild, uint64_t vis, int D,
                                         f32x16 (&acc)[MT]) {
  const int half = (threadIdx.x & 63) >> 5;
  for (; wild; wild &= wild - 1) {
    const int row = __builtin_ctzll(wild);
    const bool seen = (vis >> row) & 1;
    const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base + (row0 + row) * stride), 0,
                                                      static_cast<int>(D * sizeof(T)), 0x00020000);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int at = (32 * mt + 8 * g + 4 * half) * static_cast<int>(sizeof(T));
        union { uint4 u; decltype(__builtin_amdgcn_raw_buffer_load_b64(rs, 0, 0, 0)) w; T t[4]; } x;
        if constexpr (sizeof(T) == 2) x.w = __builtin_amdgcn_raw_buffer_load_b64(rs, at, 0, 0);
        else x.u = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, 0));
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float y = static_cast<float>(x.t[q]);
          if (!(fabsf(y) < kInf) && seen) acc[mt][4 * g + q] += AS_NAN ? __builtin_nanf("") : y;
        }
      }
  }
}

// A lane's register quads (four values along the row) of a transposed result, to a row of global
// memory: rows of the result are columns 32 mt + 8 g + 4 half + 0..3.  REST: what rounding to T takes
// from each value, in its place.
template <typename T, int MT, bool REST = false>
__device__ __forceinline__ void store_row(T* row, const f32x16 (&acc)[MT], float scale, int D) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * mt + 8 * g + 4 * half;
      if (d < D) {
        union { T t[4]; uint2 u2; uint4 u4; } w;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float x = acc[mt][4 * g + j] * scale;
          w.t[j] = static_cast<T>(x);
          if constexpr (REST) w.t[j] = static_cast<T>(x - static_cast<float>(w.t[j]));
        }
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(row + d) = w.u2;
        else *reinterpret_cast<uint4*>(row + d) = w.u4;
      }
    }
}

// Bits a..b of 64 (none where b < a), a and b any integers.
__device__ __forceinline__ uint64_t bit_range(int a, int b) {
  a = max(a, 0);
  b = min(b, 63);
  return b < a ? 0ull : (~0ull << a) & (~0ull >> (63 - b));
}

// The packed sequences: token i belongs to [ptr[b], ptr[b + 1]) of the last b with ptr[b] <= i.
struct Packing {
  const int64_t* ptr;  // B + 1 offsets, or null: one sequence of T tokens
  int B, T;
};
constexpr int kStagedPtr = 512;

// Copies up to kStagedPtr offsets into LDS (a barrier follows before the first seq_of).
__device__ __forceinline__ void stage_ptr(const Packing& s, int* lds) {
  if (s.ptr && s.B < kStagedPtr)
    for (int b = threadIdx.x; b <= s.B; b += blockDim.x)
      lds[b] = static_cast<int>(min(max(s.ptr[b], int64_t(0)), int64_t(s.T)));
}
// First token and end of token i's sequence; a token of no sequence is one of length zero at i.
__device__ __forceinline__ void seq_of(const Packing& s, const int* lds, int i, int& first, int& end) {
  if (!s.ptr) {
    first = 0;
    end = s.T;
  } else {
    const bool staged = s.B < kStagedPtr;
    auto at = [&](int b) -> int {
      return staged ? lds[b] : static_cast<int>(min(max(s.ptr[b], int64_t(0)), int64_t(s.T)));
    };
    int lo = 0, hi = s.B - 1;  // the last b in [0, B) with at(b) <= i, or 0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (at(mid) <= i) lo = mid; else hi = mid - 1;
    }
    first = at(lo);
    end = at(lo + 1);
  }
  if (i < first || i >= end) first = end = i;
}

// Element `at` of a bias table of any of the library's 16- and 32-bit types.
__device__ __forceinline__ float table_value(const void* table, int dtype, int64_t at) {
  if (dtype == GEO_F32) return static_cast<const float*>(table)[at];
  if (dtype == GEO_BF16) return static_cast<float>(static_cast<const __bf16*>(table)[at]);
  return static_cast<float>(static_cast<const _Float16*>(table)[at]);
}

// Largest and least over the wave's lanes, once per workgroup.
__device__ __forceinline__ int wave_most(int x) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x = max(x, __shfl_xor(x, d, 64));
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int wave_least(int x) { return -wave_most(-x); }

// The relative bias of one head, in LDS: times log2 e, for distances -maxd..maxd (any other has the
// bucket, and so the bias, of the nearer end).
struct Bias {
  const void* table;   // [buckets, Hq], or null
  const int32_t* lut;  // [2 maxd + 1]: bucket of each distance
  int dtype, buckets, maxd;
};
// An element of the table times log2 e.  A finite one stays finite: where the type's lowest value is all
// that a query's keys have, the factor would leave it keys of the weight exp(-inf) alone.
__device__ __forceinline__ float bias_value(const Bias& b, int64_t at) {
  const float x = table_value(b.table, b.dtype, at), y = x * kLog2e;
  return fabsf(x) < kInf ? fminf(fmaxf(y, -kMost), kMost) : y;
}
__device__ __forceinline__ void stage_bias(const Bias& b, int Hq, int h, float* lds) {
  for (int x = threadIdx.x; x <= 2 * b.maxd; x += blockDim.x)
    lds[x] = bias_value(b, static_cast<int64_t>(b.lut[x]) * Hq + h);
}

}  // namespace attn
}  // namespace geo
