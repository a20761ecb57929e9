// window_attention.hip — softmax attention within a window over packed sequences, forward.
//
// Token i of the sequence [first, end) sees key j iff first <= j < end, j <= i + right,
// (j >= i - left or j < first + sinks) and mask[j].  With s_ij = scale q_i.k_j + bias(j - i):
// o_i = sum_j exp(s_ij) v_j / sum_j exp(s_ij) over the keys it sees, 0 where it sees none.
#include "attention_args.hpp"
#include "attention_tile.hpp"

namespace geo {
namespace attn {

// One workgroup holds 32 NW queries of one head, 32 a wave, one a lane (twice, once in each half),
// and walks the keys that any of them sees in tiles of BN: first the leading tokens of the sequence
// that the first query belongs to, as far as they lie before its window, then all from the first
// query's first key to the last query's last.  Products are transposed, S^T = K Q^T and
// O^T = V^T P^T, so that a query's weights, running maximum and sum stay in one lane.
//
// Which of a tile's keys a query sees is a 64-bit word per lane: the tile is skipped by a wave
// whose words are all zero, and takes no select where all bits are set.
//
// A wave forms a tile's scores, their softmax and the product with V one after the other, per score a scale, a
// maximum, an exponential, a sum and half a conversion against 4 D operations of the matrix units.
// 131,072 tokens, 8 heads of 64 in bfloat16, window 512 to both sides: 430-446 us, 615-639 TFLOP/s (a large
// matrix product: 1122); vector instructions are active in 64% of a SIMD's cycles, matrix instructions in
// 33%, so neither alone is the bound, but how little of the one runs beside the other.
template <typename T, int DP, int NW, int BN, bool BIAS, int WAVES>
__global__ __launch_bounds__(64 * NW, WAVES) void attend_fwd(const Attend a, T* __restrict__ out, T* __restrict__ rest,
                                                            float* __restrict__ lse) {
  using Tl = Tile<T, DP, BN, 64 * NW>;
  using Frag = typename Type<T>::Frag;
  constexpr int kSub = BN / 32, kMt = DP / 32, kKc = DP / 16, kBm = 32 * NW;
  constexpr float kSlack = 8.f;
  extern __shared__ __align__(16) unsigned char lds[];
  T* const ks = reinterpret_cast<T*>(lds);
  T* const vs = reinterpret_cast<T*>(lds + Tl::kBytes);
  float* const near = reinterpret_cast<float*>(lds + 2 * Tl::kBytes);  // the tile's biases by distance
  float* const base = near + (BIAS ? kBm + BN : 0);                    // the head's, -maxd..maxd
  __shared__ int sptr[kStagedPtr];
  __shared__ unsigned long long wild[2];

  const int64_t w = xcd_block();
  const int h = static_cast<int>(w % a.Hq), q0 = static_cast<int>(w / a.Hq) * kBm;
  const int hk = h / (a.Hq / a.Hk);
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
  const T* const kbase = static_cast<const T*>(a.k) + hk * a.k_sh;
  const T* const vbase = static_cast<const T*>(a.v) + hk * a.v_sh;

  stage_ptr(a.seq, sptr);
  if (BIAS) stage_bias(a.bias, a.Hq, h, base);
  if (threadIdx.x < 2) wild[threadIdx.x] = 0;
  __syncthreads();

  // what this lane's query sees: keys lo..hi, and first..far
  const int iw = q0 + 32 * wave, i = iw + (lane & 31);
  const bool real = i < a.seq.T;
  int first, end;
  seq_of(a.seq, sptr, real ? i : a.seq.T - 1, first, end);
  const int lo = max(first, i - a.left), hi = real ? min(end - 1, i + a.right) : -1;
  const int far = min(first + a.sinks - 1, hi);
  // keys that all of the wave's queries see (both ends grow with the query), or none
  const int all_lo = __builtin_amdgcn_readlane(lo, max(min(a.seq.T - 1 - iw, 31), 0)), all_hi = __builtin_amdgcn_readlane(hi, 0);
  const Span k = span_of(a, sptr, q0, kBm);
  const int sink_tiles = k.sink_end > k.first ? (k.sink_end - k.first + BN - 1) / BN : 0;
  const int tiles = sink_tiles + (k.jend > k.jlo ? (k.jend - k.jlo + BN - 1) / BN : 0);

  Frag qf[kKc];
  {
    const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(real ? i : 0) * a.q_st + h * a.q_sh;
#pragma unroll
    for (int kc = 0; kc < kKc; ++kc) qf[kc] = frag_global(q, kc, a.D, real && a.scale != 0.f, a.scale < 0.f);
  }
  f32x16 o[kMt] = {};
  float m = -kInf, l = 0.f;
  uint64_t looked = 0;  // lanes whose query has seen a key
  // positive, so that the products' maximum is the scores': the queries carry its sign, or are zeros
  const float scale2 = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;

  auto tile_at = [&](int t, int& j0, int& jlim) {
    const bool s = t < sink_tiles;
    j0 = s ? k.first + t * BN : k.jlo + (t - sink_tiles) * BN;
    jlim = s ? k.sink_end : k.jend;
  };
  Tl kt, vt;
  kt.init(a.k_st * sizeof(T), a.D);
  vt.init(a.v_st * sizeof(T), a.D);
  uint32_t seen_byte = 1;
  auto fetch = [&](int t) {
    int j0, jlim;
    tile_at(t, j0, jlim);
    kt.load(rows_at(kbase, a.k_st * sizeof(T), j0, jlim));
    vt.load(rows_at(vbase, a.v_st * sizeof(T), j0, jlim));
    if (a.mask) seen_byte = a.mask[min(j0 + lane, jlim - 1)];
  };
  if (tiles > 0) fetch(0);
  for (int t = 0; t < tiles; ++t) {
    int j0, jlim;
    tile_at(t, j0, jlim);
    uint64_t rows = bit_range(0, min(jlim - j0, BN) - 1);
    if (a.mask) rows &= __ballot(seen_byte != 0);
    __syncthreads();
    kt.drop(rows, a.mask);
    vt.drop(rows, a.mask);
    kt.store(ks);
    vt.store_finite(vs, &wild[t & 1]);
    if (threadIdx.x == 0) wild[(t + 1) & 1] = 0;
    if (BIAS)
      for (int x = threadIdx.x; x < kBm + BN - 1; x += 64 * NW)
        near[x] = base[min(max(j0 - q0 + x - (kBm - 1), -a.bias.maxd), a.bias.maxd) + a.bias.maxd];
    __syncthreads();
    if (t + 1 < tiles) fetch(t + 1);

    const bool whole = rows == (~0ull >> (64 - BN)) && j0 >= all_lo && j0 + BN - 1 <= all_hi;
    uint64_t vis = ~0ull;
    if (!whole) {
      vis = bit_range(lo - j0, hi - j0);
      if (a.sinks) vis |= bit_range(first - j0, far - j0);
      vis &= rows;
      const uint64_t any = __ballot(vis != 0);
      if (any == 0) continue;
      looked |= any;
    } else {
      looked = ~0ull;
    }
    f32x16 s[kSub];
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      s[u] = f32x16{};
#pragma unroll
      for (int kc = 0; kc < kKc; ++kc) s[u] = Type<T>::mma(Tl::frag_along(ks, 32 * u, kc), qf[kc], s[u]);
    }
    if (sizeof(T) == 2) reads_ahead<kSub * kKc, 4, 1>();
    if (BIAS) {
      const float* bias = near + 4 * half + kBm - 1 - 32 * wave - (lane & 31);
#pragma unroll
      for (int u = 0; u < kSub; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[u][r] = fmaf(s[u][r], scale2, bias[32 * u + 8 * (r >> 2) + (r & 3)]);
    }
    if (!whole) {
#pragma unroll
      for (int u = 0; u < kSub; ++u) {
        uint32_t word = static_cast<uint32_t>(vis >> (32 * u + 4 * half));
        stay_branch(word);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[u][r] = keep_bit(s[u][r], word, 8 * (r >> 2) + (r & 3), -kInf);
      }
    }
    float top = s[0][0];
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][r]);
    top = halves_max(top) * (BIAS ? 1.f : scale2);
    // The exponentials' reference moves only when a score passes it by more than kSlack: they stay
    // below 2^kSlack, which loses nothing in any of the types, and most tiles leave the sums alone.
    const bool up = top > m + kSlack;
    if (__ballot(up)) {
      const float keep = up ? exp2_hw(m - top) : 1.f;
      m = up ? top : m;
      l *= keep;
#pragma unroll
      for (int mt = 0; mt < kMt; ++mt) o[mt] *= keep;
    }
    const float shift = m == -kInf ? 0.f : m;  // no key so far: every exponential below is 0
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[u][r] = exp2_hw(BIAS ? s[u][r] - shift : fmaf(s[u][r], scale2, -shift));
        l += s[u][r];
      }
#pragma unroll
    for (int u = 0; u < kSub; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Frag p = frag_of<T>(s[u], c);
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt) o[mt] = Type<T>::mma(Tl::frag_down(vs, 32 * u + 16 * c, mt), p, o[mt]);
      }
    if (sizeof(T) == 2) reads_ahead<kSub * 2 * kMt, 4, 2>();
    if (wild[t & 1]) add_wild<T, kMt, false>(vbase, a.v_st, j0, wild[t & 1], vis, a.D, o);
  }
  l = halves_sum(l);
  if (real) {
    const int64_t row = (static_cast<int64_t>(i) * a.Hq + h) * a.D;
    // keys are seen, but with scores of -inf alone: 0 / 0
    if (l == 0.f && (looked >> lane) & 1) l = __builtin_nanf("");
    const float inv = l == 0.f ? 0.f : 1.f / l;
    store_row<T>(out + row, o, inv, a.D);
    if (sizeof(T) == 2 && rest) store_row<T, kMt, true>(rest + row, o, inv, a.D);
    // +inf where no key is seen: the backward's exp2(s - lse) is 0 there
    if (lse && half == 0) {
      const int64_t at = static_cast<int64_t>(h) * a.seq.T + i;
      const float sum = log2f(l);
      float x = m + sum;
      // a factor of at most 1: times what is near float16's largest value it has to stay one
      if (BIAS && far_sum(x) && x - m > sum) x = nextafterf(x, -kInf);
      lse[at] = l == 0.f ? kInf : x;
      if (BIAS) lse[static_cast<int64_t>(a.Hq) * a.seq.T + at] = far_sum(x) ? exp2_hw(x - m - sum) : 1.f;
    }
  }
}

// Waves per SIMD that the registers are bounded for: while one waits for LDS or forms exponentials
// another keeps the matrix unit busy.
template <typename T, int DP, int NW>
constexpr int fwd_waves() {
  return NW == 1 ? 1 : sizeof(T) == 4 ? (DP <= 32 ? 2 : 1) : DP <= 32 ? 4 : DP <= 64 ? 3 : 2;
}

template <typename T, int DP, int NW, int BN, bool BIAS>
int launch_fwd(const Attend& a, void* out, void* rest, float* lse, hipStream_t stream) {
  const int64_t blocks = ceil_div(a.seq.T, 32 * NW) * a.Hq;
  GEO_REQUIRE(grid_fits(blocks, 64 * NW), "window attention: too many workgroups (%lld)", static_cast<long long>(blocks));
  const size_t lds = 2 * Tile<T, DP, BN, 64 * NW>::kBytes +
                     (BIAS ? sizeof(float) * (32 * NW + BN + 2 * a.bias.maxd + 1) : 0);
  GEO_HIP_CHECK(allow_lds(reinterpret_cast<const void*>(attend_fwd<T, DP, NW, BN, BIAS, fwd_waves<T, DP, NW>()>), lds));
  attend_fwd<T, DP, NW, BN, BIAS, fwd_waves<T, DP, NW>()><<<dim3(static_cast<uint32_t>(blocks)), dim3(64 * NW), lds, stream>>>(
      a, static_cast<T*>(out), static_cast<T*>(rest), lse);
  GEO_LAUNCH_CHECK("attend_fwd");
  return GEO_OK;
}

template <typename T, int DP>
int choose_fwd(const Attend& a, void* out, void* rest, float* lse, hipStream_t stream) {
  const bool lone = lone_wave(a, a.Hq, sizeof(T) == 4);
  if (a.bias.table)
    return lone ? launch_fwd<T, DP, 1, 32, true>(a, out, rest, lse, stream) : launch_fwd<T, DP, 4, 64, true>(a, out, rest, lse, stream);
  return lone ? launch_fwd<T, DP, 1, 32, false>(a, out, rest, lse, stream) : launch_fwd<T, DP, 4, 64, false>(a, out, rest, lse, stream);
}

template <typename T>
int choose_width(const Attend& a, void* out, void* rest, float* lse, hipStream_t stream) {
  if (a.D <= 32) return choose_fwd<T, 32>(a, out, rest, lse, stream);
  if (a.D <= 64) return choose_fwd<T, 64>(a, out, rest, lse, stream);
  if (a.D <= 96) return choose_fwd<T, 96>(a, out, rest, lse, stream);
  return choose_fwd<T, 128>(a, out, rest, lse, stream);
}

}  // namespace attn
}  // namespace geo

extern "C" int geo_window_attention_fwd(const geo_window_attention_t* args, void* out, void* rest, float* lse,
                                        void* stream) {
  geo::attn::Attend a;
  const int rc = geo::attn::attend_args(args, &a);
  if (rc != GEO_OK || args->tokens == 0) return rc;
  GEO_REQUIRE(out, "window attention: null output");
  const hipStream_t s = geo::as_stream(stream);
  if (args->dtype == GEO_F32) return geo::attn::choose_width<float>(a, out, rest, lse, s);
  if (args->dtype == GEO_BF16) return geo::attn::choose_width<__bf16>(a, out, rest, lse, s);
  return geo::attn::choose_width<_Float16>(a, out, rest, lse, s);
}
