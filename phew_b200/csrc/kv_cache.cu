// Quantised key/value cache: writing tokens into it and reading them back.
//
// The serving form of the packed k and v that
// mx.fast.quantized_scaled_dot_product_attention takes (phew
// emit/codegen.py:428-449, node FastQuantizedScaledDotProductAttention
// ir/ops.py:191-200): the same affine group-wise codes as phew_quantize /
// phew_dequantize, kept in pages and written in place one step at a time.
//
// Per group of g values along the head dimension
//   scale = T(max((max - min) / (2^bits - 1), 1e-8)),  bias = T(min),
//   code  = clamp(rint((x - bias) / scale), 0, 2^bits - 1)       (fp32, IEEE divide)
//   value = T(scale * code + bias)                               (fp32 fma)
// so a written row is bit for bit what phew_quantize gives for it and a read
// row what phew_dequantize gives.
#include "common.cuh"
#include "kv_cache.cuh"

namespace phew {
namespace kv {
namespace {

constexpr int kThreads = 256;

struct UpdateParams {
  Cache c;
  const void* x[2];      // k, v
  int64_t st[2][3];      // their token, head and batch strides (elements)
  void* dense[2];        // values written back, [batch][kv_heads][tokens][D]; null: none
  const int32_t* offsets;
  const int32_t* counts;  // null: all `tokens`
  int batch, tokens;
  int* error_flag;
};

// One thread per group of one token row: the simplest right form.
template <typename T>
__global__ void __launch_bounds__(kThreads) update_kernel(const UpdateParams p) {
  const int g = p.c.group, ng = p.c.head_dim / g, per = 32 / p.c.bits, top = (1 << p.c.bits) - 1;
  const int64_t rows = static_cast<int64_t>(p.batch) * p.c.map.kv_heads * p.tokens;
  const int64_t total = 2 * rows * ng;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int side = i >= rows * ng;
    const int64_t j = i - side * rows * ng;
    const int64_t row = j / ng;
    const int grp = static_cast<int>(j % ng);
    const int tok = static_cast<int>(row % p.tokens);
    const int h = static_cast<int>(row / p.tokens % p.c.map.kv_heads);
    const int b = static_cast<int>(row / p.tokens / p.c.map.kv_heads);
    const int count = p.counts ? clamp_count(p.counts[b], p.tokens) : p.tokens;
    T* dense = p.dense[side] ? static_cast<T*>(p.dense[side]) + row * p.c.head_dim + grp * g : nullptr;
    if (tok >= count) {
      if (dense)
        for (int e = 0; e < g; ++e) dense[e] = from_f32<T>(0.f);
      continue;
    }
    const T* x = static_cast<const T*>(p.x[side]) + b * p.st[side][2] + h * p.st[side][1] + tok * p.st[side][0] + grp * g;
    float lo = to_f32(x[0]), hi = lo;
    for (int e = 1; e < g; ++e) {
      lo = fminf(lo, to_f32(x[e]));
      hi = fmaxf(hi, to_f32(x[e]));
    }
    const float sc = round_to<T>(fmaxf(__fdiv_rn(hi - lo, static_cast<float>(top)), 1e-8f));
    const float bi = round_to<T>(lo);
    const uint32_t at = row_of(p.c.map, b, h, static_cast<int64_t>(p.offsets[b]) + tok);
    if (at == kNoRow)
      atomicExch(p.error_flag, PHEW_ERR_INVALID);
    else {
      static_cast<T*>(p.c.scales[side])[static_cast<int64_t>(at) * ng + grp] = from_f32<T>(sc);
      static_cast<T*>(p.c.biases[side])[static_cast<int64_t>(at) * ng + grp] = from_f32<T>(bi);
    }
    for (int w = 0; w < g / per; ++w) {
      uint32_t word = 0;
      for (int e = 0; e < per; ++e) {
        const float q = fminf(fmaxf(rintf(__fdiv_rn(to_f32(x[w * per + e]) - bi, sc)), 0.f), static_cast<float>(top));
        word |= static_cast<uint32_t>(q) << (e * p.c.bits);
        if (dense) dense[w * per + e] = from_f32<T>(fmaf(sc, q, bi));
      }
      if (at != kNoRow) p.c.codes[side][static_cast<int64_t>(at) * (p.c.head_dim / per) + grp * (g / per) + w] = word;
    }
  }
}

struct FetchParams {
  Cache c;
  void* dense[2];  // [batch][kv_heads][out_len][D]
  const int32_t* lengths;
  int batch, out_len;
  int* error_flag;
};

// One thread per word of codes.
template <typename T>
__global__ void __launch_bounds__(kThreads) fetch_kernel(const FetchParams p) {
  const int per = 32 / p.c.bits, words = p.c.head_dim / per, top = (1 << p.c.bits) - 1;
  const int ng = p.c.head_dim / p.c.group;
  const int64_t rows = static_cast<int64_t>(p.batch) * p.c.map.kv_heads * p.out_len;
  const int64_t total = 2 * rows * words;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int side = i >= rows * words;
    const int64_t j = i - side * rows * words;
    const int64_t row = j / words;
    const int w = static_cast<int>(j % words);
    const int pos = static_cast<int>(row % p.out_len);
    const int h = static_cast<int>(row / p.out_len % p.c.map.kv_heads);
    const int b = static_cast<int>(row / p.out_len / p.c.map.kv_heads);
    T* dense = static_cast<T*>(p.dense[side]) + row * p.c.head_dim + w * per;
    uint32_t at = kNoRow;
    if (pos < p.lengths[b]) {
      at = row_of(p.c.map, b, h, pos);
      if (at == kNoRow) atomicExch(p.error_flag, PHEW_ERR_INVALID);
    }
    if (at == kNoRow) {
      for (int e = 0; e < per; ++e) dense[e] = from_f32<T>(0.f);
      continue;
    }
    const int grp = w * per / p.c.group;
    const float sc = to_f32(static_cast<const T*>(p.c.scales[side])[static_cast<int64_t>(at) * ng + grp]);
    const float bi = to_f32(static_cast<const T*>(p.c.biases[side])[static_cast<int64_t>(at) * ng + grp]);
    const uint32_t word = p.c.codes[side][static_cast<int64_t>(at) * words + w];
    for (int e = 0; e < per; ++e)
      dense[e] = from_f32<T>(fmaf(sc, static_cast<float>((word >> (e * p.c.bits)) & top), bi));
  }
}

unsigned grid_for(int64_t threads) {
  const int64_t blocks = (threads + kThreads - 1) / kThreads, cap = static_cast<int64_t>(sm_count_current()) * 64;
  return static_cast<unsigned>(blocks < cap ? blocks : cap);
}

}  // namespace

int make_cache(const phew_kv_cache* c, const int* table, int64_t table_stride, int64_t columns, int64_t batch,
               const char* who, Cache* out) {
  const std::string name(who);
  PHEW_REQUIRE(c != nullptr, name + ": null cache");
  PHEW_REQUIRE(c->k_codes && c->k_scales && c->k_biases && c->v_codes && c->v_scales && c->v_biases,
               name + ": null cache array");
  PHEW_REQUIRE(c->bits == 4 || c->bits == 8, name + ": bits must be 4 or 8");
  PHEW_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, name + ": head_dim must be 64, 128 or 256");
  PHEW_REQUIRE((c->group_size == 32 || c->group_size == 64 || c->group_size == 128) && c->head_dim % c->group_size == 0,
               name + ": group_size must be 32, 64 or 128 and divide head_dim");
  PHEW_REQUIRE(dtype_bytes(c->dtype) != 0, name + ": bad dtype");
  PHEW_REQUIRE(c->pages > 0 && c->kv_heads > 0 && c->page_size > 0, name + ": empty cache");
  PHEW_REQUIRE(c->pages < (1ll << 31) && c->page_size < (1ll << 31) &&
                   c->pages * c->kv_heads < (1ll << 32) / c->page_size,
               name + ": the cache has too many rows");
  PHEW_REQUIRE(batch > 0 && batch < (1ll << 31), name + ": bad batch");
  if (table) {
    PHEW_REQUIRE(columns > 0 && columns < (1ll << 31) && columns * c->page_size < (1ll << 31) && table_stride >= 0,
                 name + ": bad block table (a sequence's pages hold at most 2^31 - 1 tokens)");
  } else {
    PHEW_REQUIRE(batch <= c->pages, name + ": without a block table the cache needs a page per sequence");
  }
  for (const void* q : {c->k_codes, c->k_scales, c->k_biases, c->v_codes, c->v_scales, c->v_biases})
    PHEW_REQUIRE((reinterpret_cast<uintptr_t>(q) & 15) == 0, name + ": cache arrays must be 16-byte aligned");
  out->codes[0] = static_cast<uint32_t*>(c->k_codes);
  out->codes[1] = static_cast<uint32_t*>(c->v_codes);
  out->scales[0] = c->k_scales;
  out->scales[1] = c->v_scales;
  out->biases[0] = c->k_biases;
  out->biases[1] = c->v_biases;
  out->head_dim = c->head_dim;
  out->group = c->group_size;
  out->bits = c->bits;
  out->map.table = table;
  out->map.table_stride = table_stride;
  out->map.columns = table ? static_cast<int32_t>(columns) : 1;
  out->map.pages = static_cast<int32_t>(c->pages);
  out->map.kv_heads = c->kv_heads;
  out->map.page_size = static_cast<int32_t>(c->page_size);
  out->map.by_page = fast_div(static_cast<uint32_t>(c->page_size));
  return PHEW_OK;
}

}  // namespace kv
}  // namespace phew

using namespace phew;

extern "C" int phew_kv_update(const phew_kv_cache* cache, const void* k, const void* v, const int64_t* k_strides,
                              const int64_t* v_strides, int64_t batch, int64_t tokens, const int* offsets,
                              const int* counts, const int* block_table, int64_t table_stride, int64_t columns,
                              void* k_out, void* v_out, int* error_flag, void* stream) {
  kv::UpdateParams p;
  if (int s = kv::make_cache(cache, block_table, table_stride, columns, batch, "phew_kv_update", &p.c)) return s;
  PHEW_REQUIRE(k && v && k_strides && v_strides && offsets && error_flag, "phew_kv_update: null pointer");
  PHEW_REQUIRE((k_out == nullptr) == (v_out == nullptr), "phew_kv_update: k_out and v_out go together");
  PHEW_REQUIRE(tokens > 0 && tokens < (1ll << 31), "phew_kv_update: bad token count");
  const int size = dtype_bytes(cache->dtype);
  for (const void* q : {k, v, static_cast<const void*>(k_out), static_cast<const void*>(v_out)})
    PHEW_REQUIRE((reinterpret_cast<uintptr_t>(q) & 15) == 0, "phew_kv_update: pointers must be 16-byte aligned");
  for (const int64_t* st : {k_strides, v_strides})
    for (int i = 0; i < 3; ++i)
      PHEW_REQUIRE(st[i] * size % 16 == 0, "phew_kv_update: strides must be multiples of 16 bytes");
  p.x[0] = k;
  p.x[1] = v;
  for (int i = 0; i < 3; ++i) {
    p.st[0][i] = k_strides[i];
    p.st[1][i] = v_strides[i];
  }
  p.dense[0] = k_out;
  p.dense[1] = v_out;
  p.offsets = offsets;
  p.counts = counts;
  p.batch = static_cast<int>(batch);
  p.tokens = static_cast<int>(tokens);
  p.error_flag = error_flag;
  const unsigned grid = kv::grid_for(2 * batch * tokens * cache->kv_heads * (cache->head_dim / cache->group_size));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (cache->dtype) {
    case PHEW_F32: kv::update_kernel<float><<<grid, kv::kThreads, 0, st>>>(p); break;
    case PHEW_F16: kv::update_kernel<f16><<<grid, kv::kThreads, 0, st>>>(p); break;
    default: kv::update_kernel<bf16><<<grid, kv::kThreads, 0, st>>>(p); break;
  }
  return launch_status("kv update_kernel");
}

extern "C" int phew_kv_fetch(const phew_kv_cache* cache, void* k_out, void* v_out, int64_t batch, int64_t out_len,
                             const int* lengths, const int* block_table, int64_t table_stride, int64_t columns,
                             int* error_flag, void* stream) {
  kv::FetchParams p;
  if (int s = kv::make_cache(cache, block_table, table_stride, columns, batch, "phew_kv_fetch", &p.c)) return s;
  PHEW_REQUIRE(k_out && v_out && lengths && error_flag, "phew_kv_fetch: null pointer");
  PHEW_REQUIRE(out_len > 0 && out_len < (1ll << 31), "phew_kv_fetch: bad output length");
  for (const void* q : {k_out, v_out})
    PHEW_REQUIRE((reinterpret_cast<uintptr_t>(q) & 15) == 0, "phew_kv_fetch: pointers must be 16-byte aligned");
  p.dense[0] = k_out;
  p.dense[1] = v_out;
  p.lengths = lengths;
  p.batch = static_cast<int>(batch);
  p.out_len = static_cast<int>(out_len);
  p.error_flag = error_flag;
  const unsigned grid = kv::grid_for(2 * batch * out_len * cache->kv_heads * (cache->head_dim * cache->bits / 32));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (cache->dtype) {
    case PHEW_F32: kv::fetch_kernel<float><<<grid, kv::kThreads, 0, st>>>(p); break;
    case PHEW_F16: kv::fetch_kernel<f16><<<grid, kv::kThreads, 0, st>>>(p); break;
    default: kv::fetch_kernel<bf16><<<grid, kv::kThreads, 0, st>>>(p); break;
  }
  return launch_status("kv fetch_kernel");
}
