// window_attention_bwd.hip — gradients of the window attention (window_attention.hip).
//
// With p_ij the weights, g_i the output's gradient and delta_i = g_i.o_i:
//   dv_j = sum_i p_ij g_i,  ds_ij = p_ij (g_i.v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dbias(d) = sum of ds_ij, j - i = d.
// delta is formed from the output before its rounding (out + rest): the rounding would cost as much
// again as the rounding of ds does.  The weights are formed again from the scores and the forward's
// log-sums, once for dq (and the bias) and once for dk and dv: seven products instead of five, for sums
// that no two workgroups share, so every gradient is the same from run to run.
#include "attention_args.hpp"
#include "attention_tile.hpp"

namespace geo {
namespace attn {

// ------------------------------------------------------------------ dq, bias ---

// Slots of a bias gradient's sums by distance: -maxd..maxd and, at both ends, the distances of a
// 32 x 32 tile that reaches inside.
constexpr int kPast = 64;
__host__ __device__ inline int bias_slots(int maxd) { return 2 * maxd + 1 + 2 * kPast; }

// A result's sums along its diagonals: lane l < 63 gets the sum over key c and query n (row and
// column) with c - n = 31 - l.  The sums move up a lane from key to key while each key's values are
// added, so a value of key c ends 31 - c lanes above its query; a key's values of the 32 queries are
// first moved to the lower half, the upper one left empty for them to move into.  Three
// instructions per 64 values; an LDS atomic for each took as long as forty.
__device__ __forceinline__ float sum_by_distance(const f32x16& x) {
  float sum = 0.f;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    float low[4], high[4];  // keys 8 g + 0..3 (of the lower half), 8 g + 4..7 (of the upper)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[4 * g + r]), 0u, false, false);
      low[r] = __uint_as_float(p[0]);
      high[r] = __uint_as_float(p[1]);
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int up = __builtin_amdgcn_update_dpp(0, __float_as_int(sum), 0x138, 0xF, 0xF, true);  // from the lane below
      sum = __int_as_float(up) + (c < 4 ? low[c & 3] : high[c & 3]);
    }
  }
  return sum;
}

// As the forward, a wave's 32 queries over tiles of keys.  The bias gradient is summed by distance,
// each wave into its own places; sub-tiles with no distance inside the ends go to two registers.  The
// workgroup's sums leave by bucket.
//
// 32,768 tokens, 8 (2) heads of 128 in bfloat16, window 2047 back: 525 us, 767 TFLOP/s of its three
// products; matrix instructions 41% of a SIMD's cycles, vector instructions 34%.  With the bias, 65,536
// tokens, 8 heads of 32, window 128 to both sides: 145 us, vector instructions.
template <typename T, int DP, int NW, int BN, bool BIAS, int WAVES>
__global__ __launch_bounds__(64 * NW, WAVES) void attend_bwd_q(const Attend a, const T* __restrict__ out,
                                                        const T* __restrict__ rest,
                                                        const T* __restrict__ grad, const float* __restrict__ lse,
                                                        float* __restrict__ delta, T* __restrict__ dq,
                                                        const int32_t* __restrict__ range, float* __restrict__ part) {
  using Tl = Tile<T, DP, BN, 64 * NW>;
  using Frag = typename Type<T>::Frag;
  constexpr int kSub = BN / 32, kMt = DP / 32, kKc = DP / 16, kBm = 32 * NW;
  extern __shared__ __align__(16) unsigned char lds[];
  T* const ks = reinterpret_cast<T*>(lds);
  T* const vs = reinterpret_cast<T*>(lds + Tl::kBytes);
  float* const near = reinterpret_cast<float*>(lds + 2 * Tl::kBytes);
  float* const base = near + (BIAS ? kBm + BN : 0);
  const int slots = bias_slots(a.bias.maxd);
  float* const sums = base + (BIAS ? 2 * a.bias.maxd + 1 : 0);  // [NW][slots]
  __shared__ int sptr[kStagedPtr];
  __shared__ unsigned long long wild[2];

  const int64_t w = xcd_block();
  const int h = static_cast<int>(w % a.Hq), block = static_cast<int>(w / a.Hq), q0 = block * kBm;
  const int hk = h / (a.Hq / a.Hk);
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
  const T* const kbase = static_cast<const T*>(a.k) + hk * a.k_sh;
  const T* const vbase = static_cast<const T*>(a.v) + hk * a.v_sh;

  stage_ptr(a.seq, sptr);
  if (BIAS) {
    stage_bias(a.bias, a.Hq, h, base);
    for (int x = threadIdx.x; x < NW * slots; x += 64 * NW) sums[x] = 0.f;
  }
  if (threadIdx.x < 2) wild[threadIdx.x] = 0;
  __syncthreads();

  const int iw = q0 + 32 * wave, i = iw + (lane & 31);
  const bool real = i < a.seq.T;
  int first, end;
  seq_of(a.seq, sptr, real ? i : a.seq.T - 1, first, end);
  const int lo = max(first, i - a.left), hi = real ? min(end - 1, i + a.right) : -1;
  const int far = min(first + a.sinks - 1, hi);
  const int all_lo = __builtin_amdgcn_readlane(lo, max(min(a.seq.T - 1 - iw, 31), 0)), all_hi = __builtin_amdgcn_readlane(hi, 0);
  const Span k = span_of(a, sptr, q0, kBm);
  const int sink_tiles = k.sink_end > k.first ? (k.sink_end - k.first + BN - 1) / BN : 0;
  const int tiles = sink_tiles + (k.jend > k.jlo ? (k.jend - k.jlo + BN - 1) / BN : 0);

  Frag qf[kKc], gf[kKc];
  float dl = 0.f;
  {
    const T* q = static_cast<const T*>(a.q) + static_cast<int64_t>(real ? i : 0) * a.q_st + h * a.q_sh;
    const int64_t row = (static_cast<int64_t>(real ? i : 0) * a.Hq + h) * a.D;
#pragma unroll
    for (int kc = 0; kc < kKc; ++kc) {
      qf[kc] = frag_global(q, kc, a.D, real);
      gf[kc] = frag_global(grad + row, kc, a.D, real);
      const Frag of = frag_global(out + row, kc, a.D, real);
      Frag rf{};
      if (sizeof(T) == 2 && rest) rf = frag_global(rest + row, kc, a.D, real);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float y = static_cast<float>(of[j]);
        if (sizeof(T) == 2 && rest) y += static_cast<float>(rf[j]);
        dl = fmaf(static_cast<float>(gf[kc][j]), y, dl);
      }
    }
    dl = halves_sum(dl);
    if (real && half == 0) delta[static_cast<int64_t>(h) * a.seq.T + i] = dl;
  }
  if (!dq && !(BIAS && range)) return;  // delta alone
  const float ls = real ? lse[static_cast<int64_t>(h) * a.seq.T + i] : kInf;
  if (BIAS && far_sum(ls)) {  // the factor of the row's weights, as one of what they are multiplied with
    const float norm = lse[static_cast<int64_t>(a.Hq + h) * a.seq.T + i];
    dl *= norm;
#pragma unroll
    for (int kc = 0; kc < kKc; ++kc)
#pragma unroll
      for (int j = 0; j < 8; ++j) gf[kc][j] = static_cast<T>(static_cast<float>(gf[kc][j]) * norm);
  }
  f32x16 o[kMt] = {};
  float below = 0.f, above = 0.f;
  const float scale2 = a.scale * kLog2e;

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
    kt.store_finite(ks, &wild[t & 1]);
    vt.store(vs);
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
      if (__ballot(vis != 0) == 0) continue;
    }
    // The scores below take infinities and NaN of K for zeros.  A query with a number as its log-sum
    // can see such a key only at a score of -inf, with the weight 0 (any other leaves NaN there).
    const uint64_t odd = uniform(wild[t & 1]);
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      uint32_t word = static_cast<uint32_t>(vis >> (32 * u + 4 * half));
      if (!whole && __ballot((word & 0x0f0f0f0fu) != 0) == 0) continue;
      f32x16 s{}, dp{};
#pragma unroll
      for (int kc = 0; kc < kKc; ++kc) {
        s = Type<T>::mma(Tl::frag_along(ks, 32 * u, kc), qf[kc], s);
        dp = Type<T>::mma(Tl::frag_along(vs, 32 * u, kc), gf[kc], dp);
      }
      if (sizeof(T) == 2) reads_ahead<2 * kKc, 4, 1>();
      const float* bias = near + 4 * half + kBm - 1 - 32 * wave - (lane & 31) + 32 * u;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int kk = 8 * (r >> 2) + (r & 3);
        s[r] = exp2_hw(BIAS ? fmaf(s[r], scale2, bias[kk]) - ls : fmaf(s[r], scale2, -ls)) * (dp[r] - dl);
      }
      if (!whole || odd) {
        if (odd && ls == ls) word = static_cast<uint32_t>((vis & ~odd) >> (32 * u + 4 * half));
        stay_branch(word);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          s[r] = keep_bit(s[r], word, 8 * (r >> 2) + (r & 3), 0.f);
      }
      if (BIAS) {
        const int d0 = j0 + 32 * u - iw;  // this sub-tile's distances: d0 - 31 .. d0 + 31
        if (d0 + 31 <= -a.bias.maxd) {
#pragma unroll
          for (int r = 0; r < 16; ++r) below += s[r];
        } else if (d0 - 31 >= a.bias.maxd) {
#pragma unroll
          for (int r = 0; r < 16; ++r) above += s[r];
        } else {
          const float x = sum_by_distance(s);
          if (lane < 63)
            __hip_atomic_fetch_add(sums + wave * slots + a.bias.maxd + kPast + d0 + 31 - lane, x, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_WORKGROUP);
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Frag p = frag_of<T>(s, c);
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt) o[mt] = Type<T>::mma(Tl::frag_down(ks, 32 * u + 16 * c, mt), p, o[mt]);
      }
      if (sizeof(T) == 2) reads_ahead<2 * kMt, 4 < 2 * kMt ? 4 : 2 * kMt, 2>();
    }
    if (odd) add_wild<T, kMt, true>(kbase, a.k_st, j0, odd, vis, a.D, o);
  }
  if (real && dq) store_row<T>(dq + (static_cast<int64_t>(i) * a.Hq + h) * a.D, o, a.scale, a.D);
  if (BIAS && range) {
    below = wave_sum(below);
    above = wave_sum(above);
    if (lane == 0) {
      sums[wave * slots] += below;
      sums[wave * slots + slots - 1] += above;
    }
    __syncthreads();
    for (int b = threadIdx.x; b < a.bias.buckets; b += 64 * NW) {
      float x = 0.f;
      // the bucket's places among the distances; the first and the last extend past the ends
      const int n = 2 * a.bias.maxd + 1, r0 = max(range[2 * b], 0), r1 = min(range[2 * b + 1], n);
      const int x0 = r0 == 0 ? 0 : r0 + kPast, x1 = r1 == n ? slots : r1 + kPast;
      if (r0 >= r1) {
        part[(static_cast<int64_t>(h) * gridDim.x / a.Hq + block) * a.bias.buckets + b] = 0.f;
        continue;
      }
      for (int at = x0; at < x1; ++at)
#pragma unroll
        for (int q = 0; q < NW; ++q) x += sums[q * slots + at];
      part[(static_cast<int64_t>(h) * gridDim.x / a.Hq + block) * a.bias.buckets + b] = x;
    }
  }
}

// The workgroups' bucket sums of one head and bucket, added in their order by one wave.
__global__ __launch_bounds__(64) void attend_bwd_bias(const float* __restrict__ part, int64_t blocks, int buckets,
                                                      int Hq, int dtype, void* __restrict__ dbias) {
  const int b = blockIdx.x % buckets, h = blockIdx.x / buckets, lane = threadIdx.x;
  double x = 0.0;
  for (int64_t n = lane; n < blocks; n += 64) x += part[(h * blocks + n) * buckets + b];
  x = wave_sum(x);
  if (lane == 0) {
    const int64_t at = static_cast<int64_t>(b) * Hq + h;
    const float y = static_cast<float>(x);
    if (dtype == GEO_F32) static_cast<float*>(dbias)[at] = y;
    else if (dtype == GEO_BF16) static_cast<__bf16*>(dbias)[at] = static_cast<__bf16>(y);
    else static_cast<_Float16*>(dbias)[at] = static_cast<_Float16>(y);
  }
}

// -------------------------------------------------------------------- dk, dv ---

// Queries far behind a leading token still see it, so such a key's gradient is a sum over the rest
// of its sequence.  That is cut at multiples of `len` tokens: the key's own workgroup adds the
// queries up to the first cut past its window, workgroups of their own (PART) add one piece each,
// per query head, and attend_bwd_join adds the sums of a key in their order.
struct Far {
  int len;       // 0: no leading tokens beyond a window
  float* own;    // [pieces][Hk][sinks][2][D]: by the piece that the sequence begins in
  float* part;   // [pieces][Hq][sinks][2][D]: by the piece of the queries
};
__device__ __forceinline__ int own_end(const Far& f, int j, int left) { return (j + left) / f.len * f.len + f.len; }

// Stores a transposed result's row as float32.
template <int MT>
__device__ __forceinline__ void store_sums(float* row, const f32x16 (&acc)[MT], int D) {
  store_row<float>(row, acc, 1.f, D);
}

// Wide heads keep their rows of V in LDS: with K's, V's and both sums in registers one wave fits a
// SIMD, and nothing hides its waits.
template <int DP>
constexpr bool kv_lds() { return DP >= 96; }

// One workgroup holds 32 NW keys of one key head, a lane one of them, and walks the queries of all
// heads that share it in tiles of BN.  S = Q K^T and dP = G V^T leave a key's weights of 16 queries
// in a lane's registers, where dV^T = G^T P and dK^T = Q^T dS take them as operands; the sums over
// heads and queries stay in registers.
//
// 32,768 tokens, 8 (2) heads of 128 in bfloat16, window 2047 back: 1030 us, 521 TFLOP/s of its four
// products.  With one wave a SIMD, LDS reads, matrix (25% of the cycles) and vector instructions (21%)
// follow one another.  65,536 tokens, 8 (2) heads of 64, window 255 back, two waves a SIMD: 140 us.
template <typename T, int DP, int NW, int BN, bool BIAS, bool PART, int WAVES>
__global__ __launch_bounds__(64 * NW, WAVES) void attend_bwd_kv(const Attend a, const T* __restrict__ grad,
                                                         const float* __restrict__ lse, const float* __restrict__ delta,
                                                         T* __restrict__ dk, T* __restrict__ dv, const Far f) {
  using Tl = Tile<T, DP, BN, 64 * NW>;
  using Frag = typename Type<T>::Frag;
  constexpr int kSub = BN / 32, kMt = DP / 32, kKc = DP / 16, kBk = 32 * NW;
  constexpr bool kVLds = kv_lds<DP>();
  using Vl = Tile<T, DP, kBk, 64 * NW>;
  extern __shared__ __align__(16) unsigned char lds[];
  T* const qs = reinterpret_cast<T*>(lds);
  T* const gs = reinterpret_cast<T*>(lds + Tl::kBytes);
  float* const rowl = reinterpret_cast<float*>(lds + 2 * Tl::kBytes);  // the tile's log-sums and deltas
  float* const rowd = rowl + BN;
  T* const vl = reinterpret_cast<T*>(rowd + BN);  // kVLds: the workgroup's rows of V
  float* const near = reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(vl) + (kVLds ? Vl::kBytes : 0));
  float* const base = near + (BIAS ? kBk + BN : 0);
  __shared__ int sptr[kStagedPtr];
  __shared__ unsigned long long wildq[2], wildg[2];
  __shared__ int last, far[2];  // far: a row of the tile has a far_sum

  const int group = a.Hq / a.Hk;
  const int lane = threadIdx.x & 63, half = lane >> 5, wave = threadIdx.x >> 6;
  int hk, key0, g0 = 0, heads = group, cut = 0;
  if constexpr (PART) {  // (piece - 1, query head, 32 NW of the leading tokens)
    const int64_t w = blockIdx.x;
    const int h = static_cast<int>(w % a.Hq);
    const int blocks = (a.sinks + kBk - 1) / kBk;
    cut = static_cast<int>(w / a.Hq / blocks + 1) * f.len;
    key0 = static_cast<int>(w / a.Hq % blocks) * kBk;
    hk = h / group;
    g0 = h % group;
    heads = 1;
  } else {
    const int64_t w = xcd_block();
    hk = static_cast<int>(w % a.Hk);
    key0 = static_cast<int>(w / a.Hk) * kBk;
  }

  stage_ptr(a.seq, sptr);
  if (threadIdx.x < 2) wildq[threadIdx.x] = wildg[threadIdx.x] = 0;
  if (BIAS && threadIdx.x < 2) far[threadIdx.x] = 0;
  if (threadIdx.x == 0) last = -1;
  __syncthreads();

  int first, end;
  if constexpr (PART) {  // the leading tokens of the sequence that holds the cut
    seq_of(a.seq, sptr, cut, first, end);
    if (first >= cut || end <= cut || own_end(f, first, a.left) > cut) return;
    key0 += first;
  }
  const int j = key0 + 32 * wave + (lane & 31);
  bool real = j < a.seq.T;
  if constexpr (PART) real = j < min(end, first + a.sinks);
  else seq_of(a.seq, sptr, real ? j : a.seq.T - 1, first, end);
  const bool sink = real && j - first < a.sinks;
  int ilo = max(first, j - a.right), ihi = min(end - 1, j + a.left);
  bool more = false;  // sums of other workgroups are added to this key's
  if constexpr (PART) {
    ilo = cut;
    ihi = own_end(f, j, a.left) <= cut ? min(end, cut + f.len) - 1 : -1;
  } else if (f.len && sink) {
    more = own_end(f, j, a.left) < end;
    ihi = more ? own_end(f, j, a.left) - 1 : end - 1;
  } else if (sink) {
    ihi = end - 1;
  }
  const bool on = real && (!a.mask || a.mask[j]);
  if (!on) ihi = -1;
  // queries of the workgroup: from its first key's on (they grow with the key), to the last of any
  int i0, ilast;
  if constexpr (PART) {
    i0 = cut;
  } else {
    int first0, end0;
    seq_of(a.seq, sptr, key0, first0, end0);
    i0 = max(first0, key0 - a.right);
  }
  atomicMax(&last, ihi);
  __syncthreads();
  ilast = __builtin_amdgcn_readfirstlane(last);
  i0 = __builtin_amdgcn_readfirstlane(i0);
  // queries that see all of the wave's keys
  const int all_lo = wave_most(real ? ilo : 0), all_hi = wave_least(real ? ihi : a.seq.T);
  const int span = ilast >= i0 ? (ilast - i0) / BN + 1 : 0;
  const int tiles = span * heads;

  Frag kf[kKc], vf[kVLds ? 1 : kKc];
  {
    const T* kr = static_cast<const T*>(a.k) + static_cast<int64_t>(real ? j : 0) * a.k_st + hk * a.k_sh;
    const T* vr = static_cast<const T*>(a.v) + static_cast<int64_t>(real ? j : 0) * a.v_st + hk * a.v_sh;
#pragma unroll
    for (int kc = 0; kc < kKc; ++kc) {
      kf[kc] = frag_global(kr, kc, a.D, on);
      if constexpr (kVLds) {  // its own wave reads a row only: no barrier
        *reinterpret_cast<Frag*>(reinterpret_cast<char*>(vl) + (32 * wave + (lane & 31)) * Vl::kRow +
                                 (16 * kc + 8 * half) * sizeof(T)) = frag_global(vr, kc, a.D, on);
      } else {
        vf[kc] = frag_global(vr, kc, a.D, on);
      }
    }
  }
  f32x16 dka[kMt] = {}, dva[kMt] = {};
  const float scale2 = a.scale * kLog2e;

  Tl qt, gt;
  qt.init(a.q_st * sizeof(T), a.D);
  gt.init(static_cast<int64_t>(a.Hq) * a.D * sizeof(T), a.D);
  float row_value = 0.f;
  auto fetch = [&](int h, int it) {
    qt.load(rows_at(static_cast<const T*>(a.q) + h * a.q_sh, a.q_st * sizeof(T), it, ilast + 1));
    gt.load(rows_at(grad + static_cast<int64_t>(h) * a.D, static_cast<int64_t>(a.Hq) * a.D * sizeof(T), it, ilast + 1));
    const int n = threadIdx.x % (2 * BN);
    row_value = (n < BN ? lse : delta)[static_cast<int64_t>(h) * a.seq.T + min(it + n % BN, ilast)];
  };
  static_assert(2 * BN <= 64 * NW, "one thread for each of a tile's log-sums and deltas");
  int h = hk * group + g0, it = i0;
  if (tiles > 0) fetch(h, it);
  for (int t = 0; t < tiles; ++t) {
    const int now = it, head = h;
    const uint64_t rows = bit_range(0, min(ilast + 1 - now, BN) - 1);
    if (BIAS && now == i0) stage_bias(a.bias, a.Hq, head, base);
    if (BIAS && threadIdx.x < BN && far_sum(row_value)) far[t & 1] = 1;
    __syncthreads();
    const int any_far = BIAS ? far[t & 1] : 0;
    qt.store_finite(qs, &wildq[t & 1]);
    gt.store_finite(gs, &wildg[t & 1]);
    if (threadIdx.x < 2 * BN) rowl[threadIdx.x] = row_value;
    if (threadIdx.x == 0) wildq[(t + 1) & 1] = wildg[(t + 1) & 1] = 0;
    if (BIAS) {
      if (threadIdx.x == 0) far[(t + 1) & 1] = 0;
      for (int x = threadIdx.x; x < kBk + BN - 1; x += 64 * NW)
        near[x] = base[min(max(key0 - now + x - (BN - 1), -a.bias.maxd), a.bias.maxd) + a.bias.maxd];
    }
    __syncthreads();
    if (BIAS && __builtin_amdgcn_readfirstlane(any_far)) {  // the rows' factors, as in attend_bwd_q
      const float* norm = lse + static_cast<int64_t>(a.Hq + head) * a.seq.T;
      gt.scale_rows(gs, [&](int n) { return far_sum(rowl[n]) ? norm[min(now + n, ilast)] : 1.f; });
      if (threadIdx.x < BN && far_sum(rowl[threadIdx.x])) rowd[threadIdx.x] *= norm[min(now + static_cast<int>(threadIdx.x), ilast)];
      __syncthreads();
    }
    it += BN;
    if (it > ilast) {
      it = i0;
      ++h;
    }
    if (t + 1 < tiles) fetch(h, it);

    const bool whole = rows == (~0ull >> (64 - BN)) && now >= all_lo && now + BN - 1 <= all_hi;
    uint64_t vis = ~0ull;
    if (!whole) {
      vis = bit_range(ilo - now, ihi - now) & rows;
      if (__ballot(vis != 0) == 0) continue;
    }
#pragma unroll
    for (int u = 0; u < kSub; ++u) {
      uint32_t word = static_cast<uint32_t>(vis >> (32 * u + 4 * half));
      if (!whole && __ballot((word & 0x0f0f0f0fu) != 0) == 0) continue;
      f32x16 s{}, dp{};
#pragma unroll
      for (int kc = 0; kc < kKc; ++kc) {
        s = Type<T>::mma(Tl::frag_along(qs, 32 * u, kc), kf[kc], s);
        if constexpr (!kVLds) dp = Type<T>::mma(Tl::frag_along(gs, 32 * u, kc), vf[kc], dp);
      }
      if constexpr (kVLds) {
#pragma unroll
        for (int kc = 0; kc < kKc; ++kc) dp = Type<T>::mma(Tl::frag_along(gs, 32 * u, kc), Vl::frag_along(vl, 32 * wave, kc), dp);
        if (sizeof(T) == 2) {
          reads_ahead<kKc, 2, 1>();
          reads_ahead<kKc, 2, 2>();
        }
      } else if (sizeof(T) == 2) {
        reads_ahead<2 * kKc, 4, 1>();
      }
      const float* bias = near + (lane & 31) + 32 * wave - 4 * half + (BN - 32 * u - 28);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const float4 ls = *reinterpret_cast<const float4*>(rowl + 32 * u + 8 * g + 4 * half);
        const float4 dl = *reinterpret_cast<const float4*>(rowd + 32 * u + 8 * g + 4 * half);
        const float lsv[4] = {ls.x, ls.y, ls.z, ls.w}, dlv[4] = {dl.x, dl.y, dl.z, dl.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = 4 * g + q, kk = 8 * g + q;
          s[r] = exp2_hw(BIAS ? fmaf(s[r], scale2, bias[27 - kk]) - lsv[q] : fmaf(s[r], scale2, -lsv[q]));
          dp[r] = s[r] * (dp[r] - dlv[q]);
        }
      }
      if (!whole) {
        stay_branch(word);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[r] = keep_bit(s[r], word, 8 * (r >> 2) + (r & 3), 0.f);
          dp[r] = keep_bit(dp[r], word, 8 * (r >> 2) + (r & 3), 0.f);
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Frag p = frag_of<T>(s, c), ds = frag_of<T>(dp, c);
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt) {
          dva[mt] = Type<T>::mma(Tl::frag_down(gs, 32 * u + 16 * c, mt), p, dva[mt]);
          dka[mt] = Type<T>::mma(Tl::frag_down(qs, 32 * u + 16 * c, mt), ds, dka[mt]);
        }
      }
      if (sizeof(T) == 2) reads_ahead<4 * kMt, 4, 2>();
    }
    if (wildq[t & 1] | wildg[t & 1]) {
      add_wild<T, kMt, false>(grad + static_cast<int64_t>(head) * a.D, static_cast<int64_t>(a.Hq) * a.D, now, wildg[t & 1],
                              vis, a.D, dva);
      add_wild<T, kMt, true>(static_cast<const T*>(a.q) + head * a.q_sh, a.q_st, now, wildq[t & 1], vis, a.D, dka);
    }
  }
  if (!real) return;
  if constexpr (PART) {
    const int h0 = hk * group + g0;
    float* row = f.part + ((static_cast<int64_t>(cut / f.len) * a.Hq + h0) * a.sinks + (j - first)) * 2 * a.D;
    store_sums(row, dka, a.D);
    store_sums(row + a.D, dva, a.D);
  } else if (more) {
    float* row = f.own + ((static_cast<int64_t>(first / f.len) * a.Hk + hk) * a.sinks + (j - first)) * 2 * a.D;
    store_sums(row, dka, a.D);
    store_sums(row + a.D, dva, a.D);
  } else {
    const int64_t at = (static_cast<int64_t>(j) * a.Hk + hk) * a.D;
    store_row<T>(dk + at, dka, a.scale, a.D);
    store_row<T>(dv + at, dva, 1.f, a.D);
  }
}

// The sums of leading token s of a sequence that reaches past the piece c that it begins in (one alone
// does): the key's own and each later piece's and head's, in kJoinRuns runs that are added in their
// order.  A workgroup for 64 of dk's and dv's values of every sequence, or where there are more of them
// of every piece (by_piece).  A chain of reads behind one another, hence the runs: 17 us for 128 pieces
// of 8 (2) heads of 128 and 16 leading tokens.
constexpr int kJoinRuns = 16;
template <typename T>
__global__ __launch_bounds__(64 * kJoinRuns) void attend_bwd_join(const Attend a, T* __restrict__ dk, T* __restrict__ dv, const Far f,
                                                        bool by_piece) {
  __shared__ int sptr[kStagedPtr];
  __shared__ float runs[kJoinRuns][64];
  const int blocks = (2 * a.D + 63) / 64;
  const int64_t w = blockIdx.x / blocks;
  const int s = static_cast<int>(w % a.sinks), hk = static_cast<int>(w / a.sinks % a.Hk);
  const int n = static_cast<int>(w / a.sinks / a.Hk);
  int first = 0, end = a.seq.T;
  if (by_piece) {
    stage_ptr(a.seq, sptr);
    __syncthreads();
    seq_of(a.seq, sptr, (n + 1) * f.len, first, end);
    if (first / f.len != n) return;
  } else if (a.seq.ptr) {
    first = static_cast<int>(min(max(a.seq.ptr[n], int64_t(0)), int64_t(a.seq.T)));
    end = static_cast<int>(min(max(a.seq.ptr[n + 1], int64_t(0)), int64_t(a.seq.T)));
  }
  const int j = first + s;
  const int64_t c = first / f.len;
  if (j >= end || own_end(f, j, a.left) >= end) return;
  const int column = threadIdx.x & 63, x = static_cast<int>(blockIdx.x % blocks) * 64 + column, run = threadIdx.x >> 6;
  const int group = a.Hq / a.Hk;
  const int64_t p0 = own_end(f, j, a.left) / f.len, terms = ((end - 1) / f.len - p0 + 1) * group;
  const int64_t per = (terms + kJoinRuns - 1) / kJoinRuns, t0 = min(run * per, terms), t1 = min(t0 + per, terms);
  float sum = 0.f;
  if (x < 2 * a.D) {
    auto term = [&](int64_t t) {
      return f.part[(((p0 + t / group) * a.Hq + hk * group + t % group) * a.sinks + s) * 2 * a.D + x];
    };
    for (int64_t t = t0; t < t1; t += 16) {
      float y[16];
#pragma unroll
      for (int q = 0; q < 16; ++q) y[q] = term(min(t + q, t1 - 1));
#pragma unroll
      for (int q = 0; q < 16; ++q) sum += t + q < t1 ? y[q] : 0.f;
    }
  }
  runs[run][column] = sum;
  __syncthreads();
  if (run || x >= 2 * a.D) return;
  sum = f.own[((c * a.Hk + hk) * a.sinks + s) * 2 * a.D + x];
  for (int q = 0; q < kJoinRuns; ++q) sum += runs[q][column];
  const int64_t row = (static_cast<int64_t>(j) * a.Hk + hk) * a.D;
  if (x < a.D) dk[row + x] = static_cast<T>(sum * a.scale);
  else dv[row + x - a.D] = static_cast<T>(sum);
}

// ---------------------------------------------------------------------- host ---

// Pieces of the queries past a leading token's window: 256 tokens, longer where that would be more than
// 512 pieces or their sums (`each` bytes a piece) more than kFarBytes.  131,072 tokens, 16 (4) heads of 128 in
// bfloat16, window 511, backward in us at 16 | 64 | 256 MiB | no bound: 64 leading tokens 5996 | 4168 | 4147 |
// 4350, 256 of them (2.7 GB without a bound) 19,920 | 6500 | 5640 | 6510; up to 64 MiB nothing changes.
constexpr int64_t kFarBytes = int64_t(64) << 20;
inline int far_len(int T, int left, int sinks, int64_t each) {
  if (sinks == 0 || T - 1 <= left) return 0;
  int len = 256;
  while (len < T && (ceil_div(T, len) > 512 || ceil_div(T, len) * each > kFarBytes)) len *= 2;
  return (left / len + 1) * static_cast<int64_t>(len) < T ? len : 0;
}

struct Plan {
  int64_t q_blocks;
  float *delta, *part;
  Far far;
  int64_t pieces;
};
inline size_t plan(const geo_window_attention_t& g, const Attend& a, void* workspace, Plan* p) {
  const int T = a.seq.T, sinks = a.sinks;
  Carver c(workspace);
  p->q_blocks = ceil_div(T, lone_wave(a, a.Hq, g.dtype == GEO_F32) ? 32 : 128);
  p->delta = c.take<float>(static_cast<size_t>(g.heads) * T);
  p->part = c.take<float>(g.bias ? static_cast<size_t>(p->q_blocks) * g.heads * g.buckets : 0);
  p->far.len = far_len(T, a.left, sinks, int64_t(g.heads + g.kv_heads) * sinks * 2 * g.head_dim * sizeof(float));
  p->pieces = p->far.len ? ceil_div(T, p->far.len) : 0;
  p->far.own = c.take<float>(static_cast<size_t>(p->pieces) * g.kv_heads * sinks * 2 * g.head_dim);
  p->far.part = c.take<float>(static_cast<size_t>(p->pieces) * g.heads * sinks * 2 * g.head_dim);
  return c.used;
}

struct Grads {
  const void *out, *rest, *grad;
  const float* lse;
  void *dq, *dk, *dv, *dbias;
  const int32_t* range;
};

// Waves per SIMD that the registers are bounded for.  dk and dv with heads of 128 keep 128 registers of
// sums and take a SIMD for themselves: two waves there spilled into the loop (1166 us against 1009 at
// 32,768 tokens, 8 (2) heads of 128, window 2047).
template <typename T, int DP, int NW>
constexpr int q_waves() {
  return NW == 1 ? 1 : sizeof(T) == 4 ? (DP <= 32 ? 2 : 1) : DP <= 32 ? 4 : DP <= 64 ? 3 : 2;
}
template <typename T, int DP, int NW>
constexpr int kv_waves() {
  return NW == 1 ? 1 : sizeof(T) == 4 ? (DP <= 32 ? 2 : 1) : DP <= 32 ? 3 : DP <= 96 ? 2 : 1;
}
// Rows of a tile: 64, or 32 where the next tile's would not find registers.
template <int DP>
constexpr int q_rows() { return DP == 128 ? 32 : 64; }
template <typename T, int DP>
constexpr int kv_rows() { return DP == 128 && sizeof(T) == 4 ? 32 : 64; }

template <typename T, int DP, int NW, int BN, bool BIAS>
int launch_q(const Attend& a, const Grads& g, const Plan& p, hipStream_t stream) {
  const size_t lds = 2 * Tile<T, DP, BN, 64 * NW>::kBytes +
                     (BIAS ? sizeof(float) * (32 * NW + BN + 2 * a.bias.maxd + 1 + NW * bias_slots(a.bias.maxd)) : 0);
  GEO_HIP_CHECK(allow_lds(reinterpret_cast<const void*>(attend_bwd_q<T, DP, NW, BN, BIAS, q_waves<T, DP, NW>()>), lds));
  attend_bwd_q<T, DP, NW, BN, BIAS, q_waves<T, DP, NW>()><<<dim3(static_cast<uint32_t>(p.q_blocks * a.Hq)), dim3(64 * NW), lds, stream>>>(
      a, static_cast<const T*>(g.out), static_cast<const T*>(g.rest), static_cast<const T*>(g.grad), g.lse, p.delta, static_cast<T*>(g.dq), g.range,
      p.part);
  GEO_LAUNCH_CHECK("attend_bwd_q");
  if (g.dbias) {
    attend_bwd_bias<<<dim3(a.bias.buckets * a.Hq), dim3(64), 0, stream>>>(p.part, p.q_blocks, a.bias.buckets, a.Hq,
                                                                          a.bias.dtype, g.dbias);
    GEO_LAUNCH_CHECK("attend_bwd_bias");
  }
  return GEO_OK;
}

template <typename T, int DP, int NW, int BN, bool BIAS, bool PART>
int launch_kv(const Attend& a, const Grads& g, const Plan& p, int64_t blocks, hipStream_t stream) {
  const size_t lds = 2 * Tile<T, DP, BN, 64 * NW>::kBytes + 2 * BN * sizeof(float) +
                     (kv_lds<DP>() ? Tile<T, DP, 32 * NW, 64 * NW>::kBytes : 0) +
                     (BIAS ? sizeof(float) * (32 * NW + BN + 2 * a.bias.maxd + 1) : 0);
  GEO_HIP_CHECK(allow_lds(reinterpret_cast<const void*>(attend_bwd_kv<T, DP, NW, BN, BIAS, PART, kv_waves<T, DP, NW>()>), lds));
  attend_bwd_kv<T, DP, NW, BN, BIAS, PART, kv_waves<T, DP, NW>()><<<dim3(static_cast<uint32_t>(blocks)), dim3(64 * NW), lds, stream>>>(
      a, static_cast<const T*>(g.grad), g.lse, p.delta, static_cast<T*>(g.dk), static_cast<T*>(g.dv), p.far);
  GEO_LAUNCH_CHECK("attend_bwd_kv");
  return GEO_OK;
}

template <typename T, int DP, bool BIAS>
int all_grads(const Attend& a, const Grads& g, const Plan& p, hipStream_t stream) {
  int rc = lone_wave(a, a.Hq, sizeof(T) == 4) ? launch_q<T, DP, 1, 32, BIAS>(a, g, p, stream)
                                              : launch_q<T, DP, 4, q_rows<DP>(), BIAS>(a, g, p, stream);
  if (!g.dk) return rc;
  if (rc == GEO_OK && p.far.len)
    rc = launch_kv<T, DP, 1, 32, BIAS, true>(a, g, p, (p.pieces - 1) * ceil_div(a.sinks, 32) * a.Hq, stream);
  if (rc == GEO_OK)
    rc = lone_wave(a, a.Hk, sizeof(T) == 4)
             ? launch_kv<T, DP, 1, 32, BIAS, false>(a, g, p, ceil_div(a.seq.T, 32) * a.Hk, stream)
             : launch_kv<T, DP, 4, kv_rows<T, DP>(), BIAS, false>(a, g, p, ceil_div(a.seq.T, 128) * a.Hk, stream);
  if (rc == GEO_OK && p.far.len) {
    const bool by_piece = a.seq.B > p.pieces - 1;
    const int64_t each = by_piece ? p.pieces - 1 : a.seq.B;
    attend_bwd_join<T><<<dim3(static_cast<uint32_t>(each * a.Hk * a.sinks * ceil_div(2 * a.D, 64))), dim3(64 * kJoinRuns), 0, stream>>>(
        a, static_cast<T*>(g.dk), static_cast<T*>(g.dv), p.far, by_piece);
    GEO_LAUNCH_CHECK("attend_bwd_join");
  }
  return rc;
}

template <typename T, int DP>
int choose_bias(const Attend& a, const Grads& g, const Plan& p, hipStream_t stream) {
  return a.bias.table ? all_grads<T, DP, true>(a, g, p, stream) : all_grads<T, DP, false>(a, g, p, stream);
}
template <typename T>
int choose_grads(const Attend& a, const Grads& g, const Plan& p, hipStream_t stream) {
  if (a.D <= 32) return choose_bias<T, 32>(a, g, p, stream);
  if (a.D <= 64) return choose_bias<T, 64>(a, g, p, stream);
  if (a.D <= 96) return choose_bias<T, 96>(a, g, p, stream);
  return choose_bias<T, 128>(a, g, p, stream);
}

}  // namespace attn
}  // namespace geo

extern "C" size_t geo_window_attention_bwd_workspace_bytes(const geo_window_attention_t* args) {
  geo::attn::Attend a;
  if (geo::attn::attend_args(args, &a) != GEO_OK || args->tokens == 0) return 0;
  geo::attn::Plan p;
  return geo::attn::plan(*args, a, nullptr, &p);
}

extern "C" int geo_window_attention_bwd(const geo_window_attention_t* args, const void* out, const void* rest, const void* grad,
                                        const float* lse, void* dq, void* dk, void* dv, const int32_t* bucket_range,
                                        void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  geo::attn::Attend a;
  const int rc = geo::attn::attend_args(args, &a);
  if (rc != GEO_OK || args->tokens == 0) return rc;
  GEO_REQUIRE(out && grad && lse && !dk == !dv, "window attention backward: null tensor");
  GEO_REQUIRE(reinterpret_cast<uintptr_t>(grad) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(rest) % 16 == 0,
              "window attention backward: out, rest and grad must lie on multiples of 16 bytes");
  GEO_REQUIRE(!dbias || (args->bias && bucket_range), "window attention backward: null bias or bucket_range");
  geo::attn::Plan p;
  const size_t need = geo::attn::plan(*args, a, workspace, &p);
  if (!workspace || workspace_bytes < need)
    return geo::set_error(GEO_ERR_WORKSPACE, "window attention backward: workspace of %zu bytes, %zu needed",
                          workspace ? workspace_bytes : size_t(0), need);
  const int64_t far = p.pieces * a.sinks;
  GEO_REQUIRE(geo::grid_fits(geo::ceil_div(a.seq.T, 128) * a.Hq, 256) && geo::grid_fits(far * a.Hq, 64) &&
                  geo::grid_fits(far * a.Hk * 4, 64 * geo::attn::kJoinRuns),
              "window attention backward: too many workgroups");
  const geo::attn::Grads g{out, rest, grad, lse, dq, dk, dv, dbias, dbias ? bucket_range : nullptr};
  const hipStream_t s = geo::as_stream(stream);
  if (args->dtype == GEO_F32) return geo::attn::choose_grads<float>(a, g, p, s);
  if (args->dtype == GEO_BF16) return geo::attn::choose_grads<__bf16>(a, g, p, s);
  return geo::attn::choose_grads<_Float16>(a, g, p, s);
}
