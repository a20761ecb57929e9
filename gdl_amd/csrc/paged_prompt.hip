// paged_prompt.hip — the C entry of attention of prompts over paged caches, and its bfloat16 kernels.
#include "paged_prompt.hpp"

namespace geo {
namespace paged {
extern template int prompt_of<float>(int, const Prompt&, const PromptPlan&, void*, float*, hipStream_t);
extern template int prompt_of<_Float16>(int, const Prompt&, const PromptPlan&, void*, float*, hipStream_t);
}  // namespace paged
}  // namespace geo

extern "C" size_t geo_paged_attention_workspace_bytes(const geo_paged_prompt_t* g) {
  using namespace geo::paged;
  if (!g || g->tokens < 1 || g->tokens >= (int64_t(1) << 31) || !sizes_ok(g->cache, g->batch, g->heads)) return 0;
  const PromptPlan p = plan_prompt(g);
  return p.pieces == 1 ? 0 : static_cast<size_t>(g->tokens) * g->heads * p.pieces * (prompt_padded(g->cache.head_dim) + 4) * sizeof(float);
}

extern "C" int geo_paged_attention(const geo_paged_prompt_t* g, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace geo;
  const char* const name = "paged attention";
  GEO_REQUIRE(g, "%s: null arguments", name);
  paged::Prompt a;
  if (const int rc = paged::pool_args(name, &g->cache, &a.pool)) return rc;
  GEO_REQUIRE(paged::type_ok(g->dtype, g->cache.stored), "%s: queries of type code %d, a pool of %d", name,
              static_cast<int>(g->dtype), static_cast<int>(g->cache.stored));
  GEO_REQUIRE(g->heads >= 1 && g->heads < (1 << 20) && g->heads % g->cache.kv_heads == 0,
              "%s: %d heads are no multiple of %d key heads (below 2^20)", name, g->heads, g->cache.kv_heads);
  GEO_REQUIRE(g->tokens >= 0 && g->tokens < (int64_t(1) << 31) - 64 && g->batch >= 0 && g->batch < (int64_t(1) << 30) &&
                  (g->ptr || g->batch <= 1),
              "%s: %lld tokens of %lld sequences%s", name, static_cast<long long>(g->tokens), static_cast<long long>(g->batch),
              g->ptr ? "" : " without ptr");
  if (g->bias) {
    GEO_REQUIRE(g->bias_dtype == GEO_F32 || g->bias_dtype == GEO_BF16 || g->bias_dtype == GEO_F16, "%s: bias dtype code %d", name,
                static_cast<int>(g->bias_dtype));
    GEO_REQUIRE(g->bias_lut && g->buckets >= 1 && g->buckets <= 256 && g->max_distance >= 1 && g->max_distance <= 1024,
                "%s: bias of %d buckets up to distance %d (at most 256 and 1024)", name, g->buckets, g->max_distance);
  }
  if (g->tokens == 0) return GEO_OK;
  GEO_REQUIRE(g->batch >= 1, "%s: tokens of no sequence", name);
  const int size = g->dtype == GEO_F32 ? 4 : 2;
  GEO_REQUIRE(g->q && reinterpret_cast<uintptr_t>(g->q) % 16 == 0 && g->q_token * size % 16 == 0 && g->q_head * size % 16 == 0 && out,
              "%s: null q or output, or rows not on multiples of 16 bytes", name);
  const paged::PromptPlan p = paged::plan_prompt(g);
  GEO_REQUIRE(grid_fits(p.blocks, paged::kPromptThreads), "%s: too many workgroups", name);
  const size_t need = geo_paged_attention_workspace_bytes(g);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(GEO_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, workspace ? workspace_bytes : size_t(0), need);
  a.q = g->q, a.q_st = g->q_token, a.q_sh = g->q_head, a.ptr = g->ptr, a.start = g->start;
  a.bias = {g->bias, g->bias_lut, g->bias_dtype, g->buckets, g->max_distance};
  a.T = g->tokens, a.B = static_cast<int>(g->batch), a.Hq = g->heads, a.heads = p.heads, a.U = p.U, a.bias_row = p.bias_row, a.fine = p.fine, a.scale = g->scale;
  float* const part = static_cast<float*>(workspace);
  const hipStream_t on = as_stream(stream);
  if (g->dtype == GEO_F32) return paged::prompt_of<float>(g->cache.stored, a, p, out, part, on);
  if (g->dtype == GEO_BF16) return paged::prompt_of<__bf16>(g->cache.stored, a, p, out, part, on);
  return paged::prompt_of<_Float16>(g->cache.stored, a, p, out, part, on);
}
