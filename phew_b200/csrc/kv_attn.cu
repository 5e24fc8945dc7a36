// Attention over a quantised key/value cache (4-bit codes), queries against
// pages read in place.
//
//   o[b, h, i] = softmax_j(scale * q[b, h, i] . k[b, h / per, j]) v[b, h / per, j]
//
// over the keys j < lengths[b] that token i sees, k and v the values
// scale * code + bias of the cache.  The serving form of
// mx.fast.quantized_scaled_dot_product_attention (phew emit/codegen.py:428-449).
#include "kv_cache.cuh"

namespace phew {
namespace kv {
namespace {

struct AttnParams {
  Cache c;
  const void* q;
  int64_t st[3];  // q's token, head and batch strides (elements)
  void* o;        // [batch][heads][tokens][D]
  const int32_t* lengths;
  const int32_t* counts;  // null: all `tokens`
  int batch, heads, tokens;
  float scale_log2;
  bool causal;
  int* error_flag;
};

__device__ __forceinline__ float value_at(const Cache& c, int side, uint32_t row, int d, float sc, float bi) {
  const uint32_t word = c.codes[side][static_cast<int64_t>(row) * (c.head_dim / 8) + (d >> 3)];
  return fmaf(sc, static_cast<float>((word >> ((d & 7) * 4)) & 15), bi);
}

// The simplest right form: one warp per query row, lanes along the head
// dimension, one key at a time with a running maximum and sum.
template <typename T, int D>
__global__ void __launch_bounds__(128) attn_kernel(const AttnParams p) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= static_cast<int64_t>(p.batch) * p.heads * p.tokens) return;
  const int tok = static_cast<int>(row % p.tokens);
  const int h = static_cast<int>(row / p.tokens % p.heads);
  const int b = static_cast<int>(row / p.tokens / p.heads);
  const int kvh = h / (p.heads / p.c.map.kv_heads);
  const int count = p.counts ? clamp_count(p.counts[b], p.tokens) : p.tokens;
  const int length = clamp_count(p.lengths[b], capacity(p.c.map));
  if (length != p.lengths[b] && lane == 0) atomicExch(p.error_flag, PHEW_ERR_INVALID);
  const int end = seen_end(length, count, tok, p.causal);
  const T* q = static_cast<const T*>(p.q) + b * p.st[2] + h * p.st[1] + tok * p.st[0];
  const int ng = D / p.c.group;
  float qv[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    qv[e] = end > 0 ? to_f32(q[lane * E + e]) : 0.f;
    o[e] = 0.f;
  }
  const int grp = lane * E / p.c.group;
  for (int j = 0; j < end; ++j) {
    const uint32_t at = row_of(p.c.map, b, kvh, j);
    if (at == kNoRow) {
      if (lane == 0) atomicExch(p.error_flag, PHEW_ERR_INVALID);
      continue;
    }
    const int64_t s_at = static_cast<int64_t>(at) * ng + grp;
    const float ks = to_f32(static_cast<const T*>(p.c.scales[0])[s_at]), kb = to_f32(static_cast<const T*>(p.c.biases[0])[s_at]);
    const float vs = to_f32(static_cast<const T*>(p.c.scales[1])[s_at]), vb = to_f32(static_cast<const T*>(p.c.biases[1])[s_at]);
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(qv[e], value_at(p.c, 0, at, lane * E + e, ks, kb), s);
    s = warp_sum(s) * p.scale_log2;
    const float m_new = fmaxf(m, s);
    const float alpha = exp2f(m - m_new), w = exp2f(s - m_new);
    m = m_new;
    l = fmaf(l, alpha, w);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(w, value_at(p.c, 1, at, lane * E + e, vs, vb), o[e] * alpha);
  }
  T* out = static_cast<T*>(p.o) + row * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = from_f32<T>(end > 0 ? o[e] / l : 0.f);
}

template <typename T>
int launch(const AttnParams& p, cudaStream_t st) {
  const int64_t blocks = (static_cast<int64_t>(p.batch) * p.heads * p.tokens + 3) / 4;
  PHEW_REQUIRE(blocks < (1ll << 31), "phew_kv_attention: too many query rows");
  const unsigned grid = static_cast<unsigned>(blocks);
  switch (p.c.head_dim) {
    case 64: attn_kernel<T, 64><<<grid, 128, 0, st>>>(p); break;
    case 128: attn_kernel<T, 128><<<grid, 128, 0, st>>>(p); break;
    default: attn_kernel<T, 256><<<grid, 128, 0, st>>>(p); break;
  }
  return launch_status("kv attn_kernel");
}

}  // namespace
}  // namespace kv
}  // namespace phew

using namespace phew;

extern "C" size_t phew_kv_attention_workspace(const phew_kv_cache* cache, int64_t batch, int64_t heads, int64_t tokens) {
  return 0;
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
  PHEW_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o)) & 15) == 0,
               "phew_kv_attention: pointers must be 16-byte aligned");
  for (int i = 0; i < 3; ++i)
    PHEW_REQUIRE(q_strides[i] * dtype_bytes(cache->dtype) % 16 == 0,
                 "phew_kv_attention: strides must be multiples of 16 bytes");
  PHEW_REQUIRE(workspace_bytes >= phew_kv_attention_workspace(cache, batch, heads, tokens) &&
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
  p.scale_log2 = scale * 1.4426950408889634f;
  p.causal = causal != 0;
  p.error_flag = error_flag;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (cache->dtype) {
    case PHEW_F32: return kv::launch<float>(p, st);
    case PHEW_F16: return kv::launch<f16>(p, st);
    default: return kv::launch<bf16>(p, st);
  }
}
