// window_step.hip — one new token per stream of the window attention, over a cache that holds the
// first tokens and a ring of the window.
//
// The cache of a stream and key head is [sinks + ring, D]: token j lies in slot j for j < sinks, else
// in slot sinks + (j - sinks) mod ring.  The new token at position p is written to its slot and
// attends to the tokens j <= p that are held: the first ones and the last `ring` up to p itself.
#include <utility>

#include "attention_tile.hpp"

namespace geo {
namespace attn {

struct Step {
  const void *q, *k, *v;  // [B, Hq, D], [B, Hk, D], contiguous rows
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
  void *kc, *vc;          // [B, Hk, sinks + ring, D] by strides
  int64_t kc_b, kc_h, vc_b, vc_h;
  const int64_t* pos;     // [B]
  Bias bias;
  int B, Hq, Hk, D, sinks, ring, slots;
  float scale;
};

constexpr int kStepThreads = 256;
constexpr int kAhead = 4;  // keys of a lane group in flight

// Eight values of a row; their products are summed in float32 (pairs of 16-bit values by one
// instruction, exact products).
template <typename T>
struct Eight {
  union { uint4 u[sizeof(T) / 2]; T t[8]; };
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int n = 0; n < static_cast<int>(sizeof(T) / 2); ++n) u[n] = reinterpret_cast<const uint4*>(p)[n];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int n = 0; n < static_cast<int>(sizeof(T) / 2); ++n) reinterpret_cast<uint4*>(p)[n] = u[n];
  }
  __device__ __forceinline__ float operator[](int e) const { return static_cast<float>(t[e]); }
};
template <typename T>
__device__ __forceinline__ float dot(const Eight<T>& a, const Eight<T>& b) {
  float x = 0.f;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x = fmaf(a.t[e], b.t[e], x);
  } else {
    const uint32_t p[4] = {a.u[0].x, a.u[0].y, a.u[0].z, a.u[0].w}, q[4] = {b.u[0].x, b.u[0].y, b.u[0].z, b.u[0].w};
    using Two = T __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (__is_same(T, __bf16)) x = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(Two, p[e]), __builtin_bit_cast(Two, q[e]), x, false);
      else x = __builtin_amdgcn_fdot2(__builtin_bit_cast(Two, p[e]), __builtin_bit_cast(Two, q[e]), x, false);
    }
  }
  return x;
}
// Sum over a group of LW = 4, 8 or 16 lanes, in all of them: each mirrored half holds the same sums
// by the time that it is added.
template <int LW>
__device__ __forceinline__ float group_sum(float x) {
  x += __uint_as_float(dpp_u32<kDppXor1>(__float_as_uint(x)));
  x += __uint_as_float(dpp_u32<kDppXor2>(__float_as_uint(x)));
  if constexpr (LW >= 8) x += __uint_as_float(dpp_u32<kDppHalfMirror>(__float_as_uint(x)));
  if constexpr (LW >= 16) x += __uint_as_float(dpp_u32<kDppMirror>(__float_as_uint(x)));
  return x;
}

// One workgroup: a piece of the slots of one stream and key head, for GB of the query heads that
// share it.  LW lanes hold a key, 8 values each (D / 8 rounded up to a power of two); every lane group
// takes kAhead keys at a time, their reads in flight together, and keeps its own running maximum, sum
// and output, which are joined through LDS at the end.  Partial results of the pieces go to the
// workspace.  The work is the reading of the cache: 256 streams, 4112 slots, 16 (4) heads of 128 in
// bfloat16 409-415 us, 4.55 TB/s with the join (a large copy: 5.19); 712 us with one key at a time and
// its lane sums through LDS.
template <typename T, int LW, int GB>
__global__ __launch_bounds__(kStepThreads) void step_piece(const Step a, int pieces, float* __restrict__ part,
                                                           T* __restrict__ out) {
  constexpr int kGroups = kStepThreads / LW;  // lane groups
  constexpr int kDp = 8 * LW;
  __shared__ float sm[4][GB], sl[4][GB];
  __shared__ float so[4][GB][kDp];
  extern __shared__ float sbias[];  // [GB][maxd + 1]: biases of distances 0 .. maxd back, times log2 e
  const int group = a.Hq / a.Hk, chunks = (group + GB - 1) / GB;
  int64_t w = blockIdx.x;
  const int piece = static_cast<int>(w % pieces); w /= pieces;
  const int gc = static_cast<int>(w % chunks); w /= chunks;
  const int hk = static_cast<int>(w % a.Hk);
  const int64_t b = w / a.Hk;
  const int64_t p = a.pos[b];
  const int lane = threadIdx.x % LW, kg = threadIdx.x / LW, d = 8 * lane;
  // lanes past the head size repeat its first values, which count as zeros on both sides: an infinity
  // times a query's zero would be NaN
  const bool wide = d < a.D, idle = a.D < kDp;
  const int heads = min(GB, group - gc * GB), h0 = hk * group + gc * GB;

  T* const kc = static_cast<T*>(a.kc) + b * a.kc_b + hk * a.kc_h;
  T* const vc = static_cast<T*>(a.vc) + b * a.vc_b + hk * a.vc_h;
  const T* const kn = static_cast<const T*>(a.k) + b * a.k_st + hk * a.k_sh;
  const T* const vn = static_cast<const T*>(a.v) + b * a.v_st + hk * a.v_sh;
  const int now = p < a.sinks ? -1 : static_cast<int>((p - a.sinks) % a.ring);  // the new token's place in the ring
  const int fresh = p < 0 ? -1 : now < 0 ? static_cast<int>(p) : a.sinks + now;
  // slots in use: all once the window is full
  const int used = p < 0 ? 0 : static_cast<int>(min(p + 1, int64_t(a.slots)));
  const int per = (used + pieces - 1) / pieces;
  const int s0 = piece * per, s1 = min(used, s0 + per);
  const int ds = wide ? d : 0;

  Eight<T> kx[kAhead], vx[kAhead];
  auto fetch = [&](int s) {
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const int at = min(s + n * kGroups, s1 - 1);
      kx[n].load((at == fresh ? kn : kc + static_cast<int64_t>(at) * a.D) + ds);
      vx[n].load((at == fresh ? vn : vc + static_cast<int64_t>(at) * a.D) + ds);
    }
  };
  if (s0 < s1) fetch(s0 + kg);
  Eight<T> q[GB];
  float o[GB][8] = {}, m[GB], l[GB];
#pragma unroll
  for (int g = 0; g < GB; ++g) {
    m[g] = -kInf;
    l[g] = 0.f;
    q[g].load(static_cast<const T*>(a.q) + b * a.q_st + (h0 + min(g, heads - 1)) * a.q_sh + ds);
    if (!wide) q[g] = Eight<T>{};
  }
  if (a.bias.table) {
    for (int x = threadIdx.x; x <= a.bias.maxd; x += kStepThreads) {
      const int64_t row = static_cast<int64_t>(a.bias.lut[a.bias.maxd - x]) * a.Hq + h0;
#pragma unroll
      for (int g = 0; g < GB; ++g)
        sbias[g * (a.bias.maxd + 1) + x] = bias_value(a.bias, row + min(g, heads - 1));
    }
    __syncthreads();
  }
  const float scale2 = a.scale * kLog2e;
  for (int s = s0 + kg; s - kg < s1; s += kAhead * kGroups) {
    float x[kAhead][GB];
#pragma unroll
    for (int n = 0; n < kAhead; ++n) {
      const int at = s + n * kGroups;
      const bool in = at < s1;
      if (at == fresh && gc == 0 && wide && in) {
        kx[n].store(kc + static_cast<int64_t>(at) * a.D + d);
        vx[n].store(vc + static_cast<int64_t>(at) * a.D + d);
      }
      if (idle && !wide) kx[n] = Eight<T>{};
      const float* bias = nullptr;
      if (a.bias.table) {
        // how far back the slot's token lies (at most maxd): the ring is read backwards from `now`
        const int ring = at - a.sinks <= now ? now - (at - a.sinks) : now + a.ring - (at - a.sinks);
        const int64_t back = at < a.sinks ? p - at : ring;
        bias = sbias + static_cast<int>(min(max(back, int64_t(0)), int64_t(a.bias.maxd)));
      }
#pragma unroll
      for (int g = 0; g < GB; ++g) {
        const float y = group_sum<LW>(dot(q[g], kx[n])) * scale2;
        x[n][g] = in ? (bias ? y + bias[g * (a.bias.maxd + 1)] : y) : -kInf;
      }
    }
#pragma unroll
    for (int g = 0; g < GB; ++g) {
      float top = m[g];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) top = fmaxf(top, x[n][g]);
      const float shift = top == -kInf ? 0.f : top, keep = exp2_hw(m[g] - shift);
      m[g] = top;
      l[g] *= keep;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[g][e] *= keep;
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        x[n][g] = exp2_hw(x[n][g] - shift);
        l[g] += x[n][g];
      }
    }
#pragma unroll
    for (int n = 0; n < kAhead; ++n)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // a repeated last key (no key of this place) has the weight 0, its values may be anything
        const float y = s + n * kGroups < s1 ? vx[n][e] : 0.f;
#pragma unroll
        for (int g = 0; g < GB; ++g) o[g][e] = fmaf(x[n][g], y, o[g][e]);
      }
    if (s - kg + kAhead * kGroups < s1) fetch(s + kAhead * kGroups);
  }
  // the groups' results joined: the wave's first, then the four waves'
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int g = 0; g < GB; ++g) {
    float top = m[g];
#pragma unroll
    for (int n = LW; n < 64; n *= 2) top = fmaxf(top, __shfl_xor(top, n, 64));
    const float keep = m[g] == -kInf ? 0.f : exp2_hw(m[g] - top);
    float sum = l[g] * keep;
#pragma unroll
    for (int n = LW; n < 64; n *= 2) sum += __shfl_xor(sum, n, 64);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float x = o[g][e] * keep;
#pragma unroll
      for (int n = LW; n < 64; n *= 2) x += __shfl_xor(x, n, 64);
      if ((threadIdx.x & 63) < LW) so[wave][g][d + e] = x;
    }
    if ((threadIdx.x & 63) == 0) {
      sm[wave][g] = top;
      sl[wave][g] = sum;
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < heads * kDp; x += kStepThreads) {
    const int g = x / kDp, e = x % kDp;
    float top = sm[0][g];
    for (int n = 1; n < 4; ++n) top = fmaxf(top, sm[n][g]);
    float sum = 0.f, y = 0.f;
    for (int n = 0; n < 4; ++n) {
      const float keep = sm[n][g] == -kInf ? 0.f : exp2_hw(sm[n][g] - top);
      sum += sl[n][g] * keep;
      y += so[n][g][e] * keep;
    }
    if (pieces == 1) {
      if (e < a.D) out[(b * a.Hq + h0 + g) * a.D + e] = static_cast<T>(used == 0 ? 0.f : y / sum);
    } else {
      float* row = part + ((b * a.Hq + h0 + g) * pieces + piece) * (kDp + 2);
      row[2 + e] = y;
      if (e == 0) {
        row[0] = top;
        row[1] = sum;
      }
    }
  }
}

template <typename T, int LW>
__global__ __launch_bounds__(8 * LW) void step_join(int D, int Hq, int pieces, const int64_t* __restrict__ pos,
                                                    const float* __restrict__ part, T* __restrict__ out) {
  constexpr int kDp = 8 * LW;
  const float* row = part + static_cast<int64_t>(blockIdx.x) * pieces * (kDp + 2);
  const int e = threadIdx.x;
  float top = -kInf, sum = 0.f, y = 0.f;
  for (int n = 0; n < pieces; ++n) top = fmaxf(top, row[n * (kDp + 2)]);
  for (int n = 0; n < pieces; ++n) {
    const float m = row[n * (kDp + 2)], keep = m == -kInf ? 0.f : exp2_hw(m - top);
    sum += row[n * (kDp + 2) + 1] * keep;
    y += row[n * (kDp + 2) + 2 + e] * keep;
  }
  if (e < D) out[static_cast<int64_t>(blockIdx.x) * D + e] = static_cast<T>(pos[blockIdx.x / Hq] < 0 ? 0.f : y / sum);
}

// Tokens into caches: one thread per 16 bytes of a token's and head's row, k and v.  131,072 tokens of 8 heads of
// 64 in bfloat16: 100 us, 5.35 TB/s (a large copy: 5.19).
template <int SIZE>
__global__ __launch_bounds__(256) void cache_fill(const char* __restrict__ k, const char* __restrict__ v, int64_t k_st,
                                                  int64_t k_sh, int64_t v_st, int64_t v_sh, const int64_t* __restrict__ ptr,
                                                  const int64_t* __restrict__ start, int64_t T, int64_t B, int Hk, int D,
                                                  char* __restrict__ kc, char* __restrict__ vc, int64_t kc_b, int64_t kc_h,
                                                  int64_t vc_b, int64_t vc_h, int64_t sinks, int64_t ring) {
  const int per = D * SIZE / 16;
  int64_t n = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (n >= T * Hk * per) return;
  const int e = static_cast<int>(n % per) * 16;
  n /= per;
  const int h = static_cast<int>(n % Hk);
  const int64_t t = n / Hk;
  int64_t lo = 0, hi = B - 1, first = 0, end = T;
  if (ptr) {
    while (lo < hi) {
      const int64_t mid = (lo + hi + 1) >> 1;
      if (ptr[mid] <= t) lo = mid; else hi = mid - 1;
    }
    first = ptr[lo];
    end = min(ptr[lo + 1], T);
  }
  if (t < first || t >= end) return;
  const int64_t at = start ? start[lo] : 0, j = at + t - first, last = at + end - 1 - first;
  if (j < 0 || (j >= sinks && j <= last - ring)) return;
  const int64_t slot = j < sinks ? j : sinks + (j - sinks) % ring;
  *reinterpret_cast<uint4*>(kc + (lo * kc_b + h * kc_h + slot * D) * SIZE + e) =
      *reinterpret_cast<const uint4*>(k + (t * k_st + h * k_sh) * SIZE + e);
  *reinterpret_cast<uint4*>(vc + (lo * vc_b + h * vc_h + slot * D) * SIZE + e) =
      *reinterpret_cast<const uint4*>(v + (t * v_st + h * v_sh) * SIZE + e);
}

// The heads of all streams lie apart, so that what is written to one is read from no other.
inline bool apart(int64_t batch, int64_t stream, int64_t heads, int64_t head, int64_t block) {
  if (batch > 1 && heads > 1 && stream < head) {  // heads outside
    std::swap(batch, heads);
    std::swap(stream, head);
  }
  if (heads > 1 && head < block) return false;
  return batch <= 1 || stream >= (heads > 1 ? head * (heads - 1) : 0) + block;
}

inline int lanes_of(int D) { return D <= 32 ? 4 : D <= 64 ? 8 : 16; }

// Pieces of a stream's slots: sixteen workgroups for each of the 256 CUs where there is work, at least
// four rounds of a workgroup's keys each (a stream of 260 slots of 32 values in two pieces and a
// join 9.8 us, in one 6 us).
inline int step_pieces(int64_t rows, int64_t slots, int D) {
  const int64_t least = 4 * kAhead * kStepThreads / lanes_of(D);
  int64_t n = 1;
  while (rows * n < 4096 && slots / (2 * n) >= least) n *= 2;
  return static_cast<int>(n);
}

template <typename T, int LW, int GB>
int launch_step(const Step& a, void* out, float* part, hipStream_t stream) {
  const int group = a.Hq / a.Hk;
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hk * ceil_div(group, GB);
  const int pieces = step_pieces(rows, a.slots, a.D);
  GEO_REQUIRE(grid_fits(rows * pieces, kStepThreads) && grid_fits(static_cast<int64_t>(a.B) * a.Hq, 8 * LW),
              "window attention step: too many workgroups");
  const size_t lds = a.bias.table ? sizeof(float) * GB * (a.bias.maxd + 1) : 0;
  step_piece<T, LW, GB><<<dim3(static_cast<uint32_t>(rows * pieces)), dim3(kStepThreads), lds, stream>>>(a, pieces, part, static_cast<T*>(out));
  GEO_LAUNCH_CHECK("step_piece");
  if (pieces > 1) {
    step_join<T, LW><<<dim3(static_cast<uint32_t>(static_cast<int64_t>(a.B) * a.Hq)), dim3(8 * LW), 0, stream>>>(a.D, a.Hq, pieces, a.pos, part, static_cast<T*>(out));
    GEO_LAUNCH_CHECK("step_join");
  }
  return GEO_OK;
}
inline int group_block(int group) { return group >= 4 ? 4 : group >= 2 ? 2 : 1; }
template <typename T, int LW>
int choose_group(const Step& a, void* out, float* part, hipStream_t stream) {
  switch (group_block(a.Hq / a.Hk)) {
    case 4: return launch_step<T, LW, 4>(a, out, part, stream);
    case 2: return launch_step<T, LW, 2>(a, out, part, stream);
    default: return launch_step<T, LW, 1>(a, out, part, stream);
  }
}
template <typename T>
int choose_step(const Step& a, void* out, float* part, hipStream_t stream) {
  switch (lanes_of(a.D)) {
    case 4: return choose_group<T, 4>(a, out, part, stream);
    case 8: return choose_group<T, 8>(a, out, part, stream);
    default: return choose_group<T, 16>(a, out, part, stream);
  }
}

}  // namespace attn
}  // namespace geo

extern "C" size_t geo_window_attention_step_workspace_bytes(int64_t batch, int64_t heads, int64_t kv_heads, int64_t slots,
                                                            int64_t head_dim) {
  if (batch < 1 || heads < 1 || kv_heads < 1 || slots < 1 || head_dim < 1) return 0;
  const int64_t rows = batch * kv_heads * geo::ceil_div(heads / kv_heads, geo::attn::group_block(static_cast<int>(heads / kv_heads)));
  const int pieces = geo::attn::step_pieces(rows, slots, static_cast<int>(head_dim));
  return pieces == 1 ? 0 : static_cast<size_t>(batch * heads) * pieces * (8 * geo::attn::lanes_of(static_cast<int>(head_dim)) + 2) * sizeof(float);
}

extern "C" int geo_window_attention_step(const geo_window_step_t* g, void* out, void* workspace, size_t workspace_bytes,
                                         void* stream) {
  using namespace geo;
  GEO_REQUIRE(g, "window attention step: null arguments");
  GEO_REQUIRE(g->dtype == GEO_F32 || g->dtype == GEO_BF16 || g->dtype == GEO_F16, "window attention step: dtype code %d",
              static_cast<int>(g->dtype));
  GEO_REQUIRE(g->batch >= 0 && g->batch < (int64_t(1) << 31) && g->kv_heads >= 1 && g->heads >= 1 && g->heads % g->kv_heads == 0,
              "window attention step: %d heads are no multiple of %d key heads", g->heads, g->kv_heads);
  GEO_REQUIRE(g->head_dim >= 8 && g->head_dim <= 128 && g->head_dim % 8 == 0,
              "window attention step: head size %d (a multiple of 8 up to 128)", g->head_dim);
  GEO_REQUIRE(g->sinks >= 0 && g->slots > g->sinks && g->slots < (int64_t(1) << 30),
              "window attention step: %lld slots, %lld of them first tokens", static_cast<long long>(g->slots),
              static_cast<long long>(g->sinks));
  if (g->bias) {
    GEO_REQUIRE(g->bias_dtype == GEO_F32 || g->bias_dtype == GEO_BF16 || g->bias_dtype == GEO_F16,
                "window attention step: bias dtype code %d", static_cast<int>(g->bias_dtype));
    GEO_REQUIRE(g->bias_lut && g->buckets >= 1 && g->max_distance >= 1 && g->max_distance <= 1024,
                "window attention step: bias of %d buckets up to distance %d (at most 1024)", g->buckets, g->max_distance);
  }
  if (g->batch == 0) return GEO_OK;
  const int size = g->dtype == GEO_F32 ? 4 : 2;
  auto in_pieces = [size](const void* p, int64_t st, int64_t sh) {
    return p && reinterpret_cast<uintptr_t>(p) % 16 == 0 && st * size % 16 == 0 && sh * size % 16 == 0;
  };
  GEO_REQUIRE(in_pieces(g->q, g->q_stream, g->q_head) && in_pieces(g->k, g->k_stream, g->k_head) &&
                  in_pieces(g->v, g->v_stream, g->v_head) && in_pieces(g->k_cache, g->k_cache_stream, g->k_cache_head) &&
                  in_pieces(g->v_cache, g->v_cache_stream, g->v_cache_head),
              "window attention step: null tensor, or rows not on multiples of 16 bytes");
  GEO_REQUIRE(attn::apart(g->batch, g->k_cache_stream, g->kv_heads, g->k_cache_head, g->slots * g->head_dim) &&
                  attn::apart(g->batch, g->v_cache_stream, g->kv_heads, g->v_cache_head, g->slots * g->head_dim) && g->k_cache != g->v_cache,
              "window attention step: heads or streams of a cache share memory");
  GEO_REQUIRE(out && g->positions, "window attention step: null output or positions");
  const size_t need = geo_window_attention_step_workspace_bytes(g->batch, g->heads, g->kv_heads, g->slots, g->head_dim);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(GEO_ERR_WORKSPACE, "window attention step: workspace of %zu bytes, %zu needed",
                     workspace ? workspace_bytes : size_t(0), need);
  const attn::Step a{g->q, g->k, g->v, g->q_stream, g->q_head, g->k_stream, g->k_head, g->v_stream, g->v_head,
                     g->k_cache, g->v_cache, g->k_cache_stream, g->k_cache_head, g->v_cache_stream, g->v_cache_head,
                     g->positions, {g->bias, g->bias_lut, g->bias_dtype, g->buckets, g->max_distance},
                     static_cast<int>(g->batch), g->heads, g->kv_heads, g->head_dim, static_cast<int>(g->sinks),
                     static_cast<int>(g->slots - g->sinks), static_cast<int>(g->slots), g->scale};
  const hipStream_t s = as_stream(stream);
  float* part = static_cast<float*>(workspace);
  if (g->dtype == GEO_F32) return attn::choose_step<float>(a, out, part, s);
  if (g->dtype == GEO_BF16) return attn::choose_step<__bf16>(a, out, part, s);
  return attn::choose_step<_Float16>(a, out, part, s);
}

extern "C" int geo_window_cache_fill(int dtype, const void* k, const void* v, int64_t k_token, int64_t k_head, int64_t v_token,
                                     int64_t v_head, const int64_t* ptr, const int64_t* start, int64_t tokens, int64_t batch,
                                     int64_t kv_heads, int64_t head_dim, void* k_cache, void* v_cache, int64_t k_cache_stream,
                                     int64_t k_cache_head, int64_t v_cache_stream, int64_t v_cache_head, int64_t slots,
                                     int64_t sinks, void* stream) {
  using namespace geo;
  GEO_REQUIRE(dtype == GEO_F32 || dtype == GEO_BF16 || dtype == GEO_F16, "window cache: dtype code %d", dtype);
  GEO_REQUIRE(tokens >= 0 && batch >= 0 && kv_heads >= 1 && kv_heads < (1 << 20) && head_dim >= 8 && head_dim <= 128 && head_dim % 8 == 0,
              "window cache: %lld tokens, %lld streams, %lld heads of %lld", static_cast<long long>(tokens),
              static_cast<long long>(batch), static_cast<long long>(kv_heads), static_cast<long long>(head_dim));
  GEO_REQUIRE(sinks >= 0 && slots > sinks, "window cache: %lld slots, %lld of them first tokens",
              static_cast<long long>(slots), static_cast<long long>(sinks));
  GEO_REQUIRE(ptr || batch <= 1, "window cache: %lld streams without ptr", static_cast<long long>(batch));
  if (tokens == 0 || batch == 0) return GEO_OK;
  const int size = dtype == GEO_F32 ? 4 : 2;
  auto in_pieces = [size](const void* p, int64_t st, int64_t sh) {
    return p && reinterpret_cast<uintptr_t>(p) % 16 == 0 && st * size % 16 == 0 && sh * size % 16 == 0;
  };
  GEO_REQUIRE(in_pieces(k, k_token, k_head) && in_pieces(v, v_token, v_head) &&
                  in_pieces(k_cache, k_cache_stream, k_cache_head) && in_pieces(v_cache, v_cache_stream, v_cache_head),
              "window cache: null tensor, or rows not on multiples of 16 bytes");
  GEO_REQUIRE(attn::apart(batch, k_cache_stream, kv_heads, k_cache_head, slots * head_dim) &&
                  attn::apart(batch, v_cache_stream, kv_heads, v_cache_head, slots * head_dim) && k_cache != v_cache,
              "window cache: heads or streams of a cache share memory");
  const int64_t blocks = ceil_div(tokens * kv_heads * (head_dim * size / 16), 256);
  GEO_REQUIRE(grid_fits(blocks, 256), "window cache: too many workgroups");
  auto launch = [&](auto kernel) {
    kernel<<<dim3(static_cast<uint32_t>(blocks)), dim3(256), 0, as_stream(stream)>>>(
        static_cast<const char*>(k), static_cast<const char*>(v), k_token, k_head, v_token, v_head, ptr, start, tokens, batch,
        static_cast<int>(kv_heads), static_cast<int>(head_dim), static_cast<char*>(k_cache), static_cast<char*>(v_cache),
        k_cache_stream, k_cache_head, v_cache_stream, v_cache_head, sinks, slots - sinks);
  };
  if (size == 4) launch(attn::cache_fill<4>);
  else launch(attn::cache_fill<2>);
  GEO_LAUNCH_CHECK("cache_fill");
  return GEO_OK;
}
