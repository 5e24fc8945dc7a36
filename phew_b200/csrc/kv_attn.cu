// Attention over a quantised key/value cache (4-bit codes), queries against
// pages read in place.
//
//   o[b, h, i] = softmax_j(scale * q[b, h, i] . k[b, h / per, j]) v[b, h / per, j]
//
// over the keys j < lengths[b] that token i sees, k and v the values
// scale * code + bias of the cache.  The serving form of
// mx.fast.quantized_scaled_dot_product_attention (phew emit/codegen.py:428-449).
#include "kv_attn_tc.cuh"

using namespace phew;

extern "C" size_t phew_kv_attention_workspace(const phew_kv_cache* cache, int64_t batch, int64_t heads,
                                              int64_t tokens, int64_t columns) {
  if (!cache || cache->kv_heads <= 0 || batch <= 0 || heads <= 0 || tokens <= 0 || columns <= 0) return 0;
  const int64_t rows = tokens * (heads / cache->kv_heads);
  size_t few = 0, many = 0;
  switch (cache->dtype) {
    case PHEW_F32: few = kv::attn_bytes<float>(batch, cache->kv_heads, cache->head_dim, cache->group_size, rows); break;
    case PHEW_F16: few = kv::attn_bytes<f16>(batch, cache->kv_heads, cache->head_dim, cache->group_size, rows); break;
    default: few = kv::attn_bytes<bf16>(batch, cache->kv_heads, cache->head_dim, cache->group_size, rows);
  }
  const int64_t cap = columns * cache->page_size;
  if (kv::takes_tc(batch, cache->kv_heads, cache->head_dim, cache->dtype, rows, cap))
    many = kv::tc_bytes(batch, cache->kv_heads, cache->head_dim, rows, cap);
  return few > many ? few : many;
}

extern "C" int phew_kv_attention(const phew_kv_cache* cache, const void* q, const int64_t* q_strides, void* o,
                                 int64_t batch, int64_t heads, int64_t tokens, const int* lengths, const int* counts,
                                 const int* block_table, int64_t table_stride, int64_t columns, float scale,
                                 int causal, void* workspace, size_t workspace_bytes, int* error_flag, void* stream) {
  kv::AttnParams p;
  if (int s = kv::make_cache(cache, block_table, table_stride, columns, batch, "phew_kv_attention", &p.c)) return s;
  PHEW_REQUIRE(q && q_strides && o && lengths && error_flag, "phew_kv_attention: null pointer");
  PHEW_REQUIRE(cache->bits == 4, "phew_kv_attention: the cache must hold 4-bit codes");
  PHEW_REQUIRE(tokens > 0 && tokens < (1ll << 31), "phew_kv_attention: bad token count");
  PHEW_REQUIRE(heads > 0 && heads % cache->kv_heads == 0 && heads < (1ll << 31),
               "phew_kv_attention: heads must be a multiple of the cache's kv_heads");
  PHEW_REQUIRE(heads / cache->kv_heads < ((1ll << 31) - (1 << 16)) / tokens, "phew_kv_attention: too many query rows");
  // (the kernels count keys a few tiles past the last one, and a sequence's tiles over its heads, in 32 bits)
  const int64_t cap = kv::capacity(p.c.map);
  PHEW_REQUIRE(cap <= (1ll << 31) - 1024 && (cap / kv::kTile + 1 + kv::kBegin) * cache->kv_heads < (1ll << 32),
               "phew_kv_attention: a sequence's pages hold too many tokens");
  PHEW_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o)) & 15) == 0,
               "phew_kv_attention: pointers must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    PHEW_REQUIRE(q_strides[i] * dtype_bytes(cache->dtype) % 16 == 0,
                 "phew_kv_attention: strides must be multiples of 16 bytes");
  PHEW_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0,
               "phew_kv_attention: pointers must be 16-byte aligned");
  PHEW_REQUIRE(workspace_bytes >= phew_kv_attention_workspace(cache, batch, heads, tokens, block_table ? columns : 1) &&
                   (workspace || workspace_bytes == 0),
               "phew_kv_attention: the workspace is too small");
  p.q = q;
  for (int i = 0; i < 3; ++i) p.st[i] = q_strides[i];
  p.o = o;
  p.lengths = lengths;
  p.counts = counts;
  p.batch = static_cast<int>(batch);
  p.heads = static_cast<int>(heads);
  p.tokens = static_cast<int>(tokens);
  p.per = static_cast<int>(heads / cache->kv_heads);
  p.by_per = kv::fast_div(static_cast<uint32_t>(p.per));
  p.scale_log2 = scale * 1.4426950408889634f;
  p.causal = causal != 0;
  p.error_flag = error_flag;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // (the tcgen05 kernel takes its maxima over unscaled scores)
  if (p.scale_log2 > 0.f && kv::takes_tc(batch, cache->kv_heads, cache->head_dim, cache->dtype,
                                         static_cast<int64_t>(p.tokens) * p.per, cap))
    return kv::run_attn_tc(p, cache->dtype == PHEW_BF16, workspace, st);
  switch (cache->dtype) {
    case PHEW_F32: return kv::run_attn<float>(p, workspace, st);
    case PHEW_F16: return kv::run_attn<f16>(p, workspace, st);
    default: return kv::run_attn<bf16>(p, workspace, st);
  }
}
