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
  // nonzero iff one of the packed values is infinite or NaN
  static __device__ __forceinline__ uint32_t wild(uint32_t w) {
    return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
  }
};
template <> struct Type<_Float16> {
  using Frag = f16x8;
  static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t wild(uint32_t w) {
    return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
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
  static __device__ __forceinline__ uint32_t wild(uint32_t w) {
    return (w & 0x7f800000u) == 0x7f800000u;
  }
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kInf = __builtin_huge_valf();

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

// A tile of rows in LDS: ROWS rows of DP values (a head's D, zero beyond), 16 bytes of padding per
// row so that the rows of a column of 16-byte reads start in different banks.
template <typename T, int DP, int ROWS, int NT>
struct Tile {
  static constexpr int kPer = 16 / sizeof(T);            // values in 16 bytes
  static constexpr int kStride = DP + kPer;              // values from row to row
  static constexpr int kChunks = DP / kPer;              // 16-byte pieces of a row
  static constexpr int kLoads = ROWS * kChunks / NT;     // per thread
  static constexpr int kBytes = ROWS * kStride * sizeof(T);
  static_assert(ROWS * kChunks % NT == 0, "a thread loads whole pieces");

  uint4 reg[kLoads];

  // Rows row0.. of a head into registers; rows from `end` on and values from D on are not read
  // (their address is the last one's, in bounds: `end` >= 1).
  __device__ __forceinline__ void load(const T* base, int64_t stride, int row0, int end, int D) {
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int c = threadIdx.x + n * NT, row = c / kChunks, at = c % kChunks * kPer;
      const int r = min(row0 + row, end - 1), d = at < D ? at : 0;
      reg[n] = *reinterpret_cast<const uint4*>(base + r * stride + d);
    }
  }
  // The registers into LDS, rows whose bit is off and values from D on as zeros.
  __device__ __forceinline__ void store(T* lds, uint64_t rows, int D) const {
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int c = threadIdx.x + n * NT, row = c / kChunks, at = c % kChunks * kPer;
      *reinterpret_cast<uint4*>(lds + row * kStride + at) = piece(n, rows, D);
    }
  }
  // The same with zeros in the place of infinities and NaN, whose rows' bits go to `wild` (LDS): a
  // product down the rows gives every column's query or key a weight for every row, and a weight
  // of 0 would not keep them from the ones that do not see the row.  add_wild adds them where the
  // row is seen.
  __device__ __forceinline__ void store_finite(T* lds, uint64_t rows, int D, unsigned long long* wild) const {
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int c = threadIdx.x + n * NT, row = c / kChunks, at = c % kChunks * kPer;
      union { uint4 u; T t[kPer]; } v;
      v.u = piece(n, rows, D);
      if (Type<T>::wild(v.u.x) | Type<T>::wild(v.u.y) | Type<T>::wild(v.u.z) | Type<T>::wild(v.u.w)) {
        atomicOr(wild, 1ull << row);
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          v.t[e] = fabsf(static_cast<float>(v.t[e])) < kInf ? v.t[e] : static_cast<T>(0.f);
      }
      *reinterpret_cast<uint4*>(lds + row * kStride + at) = v.u;
    }
  }
  __device__ __forceinline__ uint4 piece(int n, uint64_t rows, int D) const {
    const int c = threadIdx.x + n * NT, row = c / kChunks, at = c % kChunks * kPer;
    const bool in = ((rows >> row) & 1) && at < D;
    uint4 v = reg[n];
    v.x = in ? v.x : 0; v.y = in ? v.y : 0; v.z = in ? v.z : 0; v.w = in ? v.w : 0;
    return v;
  }
  // Operand with this lane's row `row0 + lane % 32`, k = 16 kc + 8 half + 0..7 along the row.
  static __device__ __forceinline__ typename Type<T>::Frag frag_along(const T* lds, int row0, int kc) {
    const int lane = threadIdx.x & 63;
    const T* p = lds + (row0 + (lane & 31)) * kStride + 16 * kc + 8 * (lane >> 5);
    return *reinterpret_cast<const typename Type<T>::Frag*>(p);
  }
  // Operand with this lane's column `32 mt + lane % 32`, k down the rows in a result's order:
  // rows row0 + 8 (j / 4) + 4 half + j % 4.  For 2-byte types by the transposing LDS read, which
  // gives lane l of sixteen column l of the 4 x 16 values that the sixteen address, four of a row
  // each.
  static __device__ __forceinline__ typename Type<T>::Frag frag_down(const T* lds, int row0, int mt) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    typename Type<T>::Frag f;
    if constexpr (sizeof(T) == 2) {
      const int l = lane & 15;
      const T* p = lds + (row0 + 4 * half + (l >> 2)) * kStride + 32 * mt + (lane & 16) + 4 * (l & 3);
      using LdsI16x4 = __attribute__((address_space(3))) i16x4;
      const i16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4*)p);
      const i16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsI16x4*)(p + 8 * kStride));
      union { i16x4 h[2]; typename Type<T>::Frag f; } u;
      u.h[0] = a; u.h[1] = b;
      f = u.f;
    } else {
      const T* p = lds + (row0 + 4 * half) * kStride + 32 * mt + (lane & 31);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = p[(8 * (j >> 2) + (j & 3)) * kStride];
    }
    return f;
  }
};

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

// Operand with this lane's row of global memory, as frag_along; zero where !in or beyond D.
template <typename T>
__device__ __forceinline__ typename Type<T>::Frag frag_global(const T* row, int kc, int D, bool in) {
  const int at = 16 * kc + 8 * ((threadIdx.x & 63) >> 5);
  const bool ok = in && at < D;
  union { uint4 u[sizeof(T) / 2]; typename Type<T>::Frag f; } x;
  const uint4* p = reinterpret_cast<const uint4*>(row + (ok ? at : 0));
#pragma unroll
  for (int n = 0; n < static_cast<int>(sizeof(T) / 2); ++n) {
    x.u[n] = p[n];
    if (!ok) x.u[n] = make_uint4(0, 0, 0, 0);
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
    const T* p = base + (row0 + row) * stride;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = 32 * mt + 8 * (r >> 2) + 4 * half + (r & 3);
        const float x = d < D ? static_cast<float>(p[d]) : 0.f;
        if (!(fabsf(x) < kInf) && ((vis >> row) & 1)) acc[mt][r] += AS_NAN ? __builtin_nanf("") : x;
      }
  }
}

// A lane's register quads (four values along the row) of a transposed result, to a row of global
// memory: rows of the result are columns 32 mt + 8 g + 4 half + 0..3.
template <typename T, int MT>
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
        for (int j = 0; j < 4; ++j) w.t[j] = static_cast<T>(acc[mt][4 * g + j] * scale);
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

// The relative bias of one head, in LDS: times log2 e, for distances -maxd..maxd (any other has the
// bucket, and so the bias, of the nearer end).
struct Bias {
  const void* table;   // [buckets, Hq], or null
  const int32_t* lut;  // [2 maxd + 1]: bucket of each distance
  int dtype, buckets, maxd;
};
__device__ __forceinline__ void stage_bias(const Bias& b, int Hq, int h, float* lds) {
  for (int x = threadIdx.x; x <= 2 * b.maxd; x += blockDim.x)
    lds[x] = table_value(b.table, b.dtype, static_cast<int64_t>(b.lut[x]) * Hq + h) * kLog2e;
}

}  // namespace attn
}  // namespace geo
