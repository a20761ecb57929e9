// attention_args.hpp — the attention kernels' arguments, and their checks on the host.
#pragma once

#include "attention_tile.hpp"

namespace geo {
namespace attn {

struct Attend {
  const void *q, *k, *v;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;  // elements from token to token and from head to head
  Packing seq;
  const uint8_t* mask;
  Bias bias;
  int Hq, Hk, D, left, right, sinks;
  float scale;
};

// The keys of a workgroup's queries q0 .. q0 + rows - 1: the first and last queries' bound them, for
// both ends grow with the query; and the leading tokens of the first query's sequence, as far as
// they lie before those.  Wave-uniform.
struct Span {
  int first, sink_end, jlo, jend;
};
__device__ __forceinline__ Span span_of(const Attend& a, const int* sptr, int q0, int rows) {
  int first0, end0, first1, end1;
  seq_of(a.seq, sptr, q0, first0, end0);
  const int q1 = min(q0 + rows, a.seq.T) - 1;
  seq_of(a.seq, sptr, q1, first1, end1);
  Span k;
  k.first = __builtin_amdgcn_readfirstlane(first0);
  k.jlo = __builtin_amdgcn_readfirstlane(max(first0, q0 - a.left));
  k.jend = __builtin_amdgcn_readfirstlane(min(end1, q1 + a.right + 1));
  k.sink_end = __builtin_amdgcn_readfirstlane(min(min(first0 + a.sinks, k.jlo), end0));
  return k;
}

// Reads of 16 bytes begin at any token and head: pointer and strides are multiples of that.  Tokens
// do not overlap, and a tile's offsets stay below 2^31.
inline bool in_pieces(const void* p, int64_t st, int64_t sh, int D, int size) {
  return p && reinterpret_cast<uintptr_t>(p) % 16 == 0 && st * size % 16 == 0 && sh * size % 16 == 0 && st >= D &&
         st < (int64_t(1) << 22);
}

inline int attend_args(const geo_window_attention_t* g, Attend* a) {
  GEO_REQUIRE(g, "window attention: null arguments");
  GEO_REQUIRE(g->dtype == GEO_F32 || g->dtype == GEO_BF16 || g->dtype == GEO_F16, "window attention: dtype code %d",
              static_cast<int>(g->dtype));
  GEO_REQUIRE(g->tokens >= 0 && g->tokens < (int64_t(1) << 30), "window attention: %lld tokens (at most 2^30 - 1)",
              static_cast<long long>(g->tokens));
  GEO_REQUIRE(g->kv_heads >= 1 && g->heads >= 1 && g->heads % g->kv_heads == 0,
              "window attention: %d heads are no multiple of %d key heads", g->heads, g->kv_heads);
  GEO_REQUIRE(g->head_dim >= 8 && g->head_dim <= 128 && g->head_dim % 8 == 0,
              "window attention: head size %d (a multiple of 8 up to 128)", g->head_dim);
  GEO_REQUIRE(g->left >= 0 && g->right >= 0 && g->sinks >= 0 && g->sinks <= 256,
              "window attention: window of %lld and %lld, %lld first tokens (none negative, at most 256 of these)",
              static_cast<long long>(g->left), static_cast<long long>(g->right), static_cast<long long>(g->sinks));
  GEO_REQUIRE(!g->ptr || (g->sequences >= 1 && g->sequences < (int64_t(1) << 30)), "window attention: %lld sequences",
              static_cast<long long>(g->sequences));
  if (g->bias) {
    GEO_REQUIRE(g->bias_dtype == GEO_F32 || g->bias_dtype == GEO_BF16 || g->bias_dtype == GEO_F16,
                "window attention: bias dtype code %d", static_cast<int>(g->bias_dtype));
    GEO_REQUIRE(g->bias_lut && g->buckets >= 1 && g->buckets <= 256 && g->max_distance >= 1 && g->max_distance <= 1024,
                "window attention: bias of %d buckets up to distance %d (at most 256 and 1024)", g->buckets, g->max_distance);
  }
  if (g->tokens == 0) return GEO_OK;
  const int size = g->dtype == GEO_F32 ? 4 : 2;
  GEO_REQUIRE(in_pieces(g->q, g->q_token, g->q_head, g->head_dim, size) &&
                  in_pieces(g->k, g->k_token, g->k_head, g->head_dim, size) &&
                  in_pieces(g->v, g->v_token, g->v_head, g->head_dim, size),
              "window attention: null q, k or v, rows not on multiples of 16 bytes, or a token stride below the head size "
              "or from 2^22 on");
  const int T = static_cast<int>(g->tokens);
  auto up_to = [T](int64_t x) { return static_cast<int>(x < T ? x : T); };
  *a = Attend{g->q, g->k, g->v, g->q_token, g->q_head, g->k_token, g->k_head, g->v_token, g->v_head,
              {g->ptr, static_cast<int>(g->ptr ? g->sequences : 1), T}, g->mask,
              {g->bias, g->bias_lut, g->bias_dtype, g->buckets, g->max_distance},
              g->heads, g->kv_heads, g->head_dim, up_to(g->left), up_to(g->right), up_to(g->sinks), g->scale};
  return GEO_OK;
}

// Rows are taken by workgroups of four waves, which share tiles of 64 rows of the other side, or by one
// wave alone with tiles of 32.  Alone, a wave loads little that it does not need: better where four would
// leave CUs without a workgroup and the window is narrow.  1024 tokens of 8 heads of 64, windows to both
// sides, forward and backward in us, four waves | one:
//   bfloat16, 129 keys   9.1  25.7 |  8.3  21.5      float32, 129 keys   24.2   76.5 | 18.4   54.8
//             385       13.6  38.8 | 15.4  37.8               513        52.3  170.9 | 50.3  161.1
//             769       20.3  57.0 | 25.3  61.2              2049        82.0  265.4 | 92.2  293.1
// and at 8192 tokens, 512 workgroups of four waves, with 257 keys 16.7 49.9 | 18.9 53.1 and 63.7 214.4 |
// 79.8 200.6.
inline bool lone_wave(const Attend& a, int heads, bool f32) {
  const int64_t keys = int64_t(a.left) + a.right + 1;
  return ceil_div(a.seq.T, 128) * heads < 256 && keys <= (f32 ? 512 : 256);
}

// Dynamic LDS beyond 64 KB has to be asked for.
inline hipError_t allow_lds(const void* kernel, size_t bytes) {
  return bytes <= 60 * 1024 ? hipSuccess
                            : hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
}

}  // namespace attn
}  // namespace geo
