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
constexpr int64_t kMaxRows = (1ll << 31) - (1 << 16);  // row numbers of a block past the last one stay 32-bit

// Eight consecutive elements of a token row: one thread's share.
template <typename T> struct alignas(16) Eight {
  T v[8];
};

template <typename T> __device__ __forceinline__ Eight<T> load8(const T* p) {
  Eight<T> e;
  const uint4* q = reinterpret_cast<const uint4*>(p);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) reinterpret_cast<uint4*>(&e)[i] = __ldg(q + i);
  return e;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const Eight<T>& e) {
  uint4* q = reinterpret_cast<uint4*>(p);
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) q[i] = reinterpret_cast<const uint4*>(&e)[i];
}

// A row number in [0, 2^31) of a [batch][kv_heads][n] array, taken apart.
struct RowSplit {
  FastDiv by_n, by_heads;
};
__device__ __forceinline__ void split_row(const RowSplit& s, int row, int& b, int& h, int& i) {
  const int bh = static_cast<int>(div_by(s.by_n, static_cast<uint32_t>(row)));
  i = row - bh * static_cast<int>(s.by_n.d);
  b = static_cast<int>(div_by(s.by_heads, static_cast<uint32_t>(bh)));
  h = bh - b * static_cast<int>(s.by_heads.d);
}

// Token rows a thread works on at once: their loads are in flight together.
constexpr int kRows = 4;

struct UpdateParams {
  Cache c;
  const void* x[2];      // k, v
  int64_t st[2][3];      // their token, head and batch strides (elements)
  void* dense[2];        // values written back, [batch][kv_heads][tokens][D]; null: none
  const int32_t* offsets;
  const int32_t* counts;  // null: all `tokens`
  RowSplit split;
  int rows, tokens;
  int* error_flag;
};

// Codes of eight values.  (x - bias) / scale is taken as a product with the
// reciprocal, which lies within 3 roundings (q 2^-22.4) of the IEEE quotient:
// only where that could cross a border between two codes, or is no number,
// are the eight divided again, so the codes are phew_quantize's bit for bit
// at a third of the instructions of eight divisions.
template <int BITS>
__device__ __forceinline__ void codes8(const float* x, float bi, float sc, float* q) {
  constexpr float top = (1 << BITS) - 1;
  constexpr float near = 0.5f - (BITS == 4 ? 1.f / (1 << 17) : 1.f / (1 << 13));  // > 3 roundings of 2 top
  const float inv = __frcp_rn(sc);
  bool sure = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = __fmul_rn(x[e] - bi, inv);
    const float r = __fadd_rn(__fadd_rn(v, 12582912.f), -12582912.f);  // nearest even, |v| < 2^22
    sure = sure && fabsf(v - r) < near;
    q[e] = fminf(fmaxf(r, 0.f), top);
  }
  if (!sure) {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = fminf(fmaxf(rintf(__fdiv_rn(x[e] - bi, sc)), 0.f), top);
  }
}

// Bound by HBM: one 16-byte load of x per eight 16-bit values, 4 or 8 bytes of
// codes out (and 16 of values).  Eight values to a thread make a code word of
// one thread and a group of 4, 8 or 16 neighbouring lanes.
template <typename T, int BITS, int G>
__global__ void __launch_bounds__(kThreads) update_kernel(const UpdateParams p) {
  constexpr int LG = G / 8;
  constexpr float top = (1 << BITS) - 1;
  const int side = blockIdx.y;
  const int lanes = p.c.head_dim / 8;                  // threads to a row
  const int per_pass = kThreads / lanes;               // rows to a pass of the block
  const int c = threadIdx.x & (lanes - 1);             // which eight of the row
  const int row0 = blockIdx.x * (per_pass * kRows) + static_cast<int>(threadIdx.x) / lanes;
  const int ng = p.c.head_dim / G;
  const T* xs = static_cast<const T*>(p.x[side]);
  Eight<T> in[kRows];
  int b[kRows], h[kRows], tok[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int row = row0 + u * per_pass;
    if (row < p.rows) {
      split_row(p.split, row, b[u], h[u], tok[u]);
      in[u] = load8(xs + b[u] * p.st[side][2] + h[u] * p.st[side][1] + tok[u] * p.st[side][0] + c * 8);
    } else {
      tok[u] = -1;
      in[u] = Eight<T>{};
    }
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    float x[8], q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = to_f32(in[u].v[e]);
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      lo = fminf(lo, x[e]);
      hi = fmaxf(hi, x[e]);
    }
#pragma unroll
    for (int o = LG / 2; o > 0; o >>= 1) {  // a group's lanes lie side by side
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (tok[u] < 0) continue;
    const int row = row0 + u * per_pass;
    const int count = p.counts ? clamp_count(__ldg(p.counts + b[u]), p.tokens) : p.tokens;
    T* dense = p.dense[side] ? static_cast<T*>(p.dense[side]) + static_cast<int64_t>(row) * p.c.head_dim + c * 8 : nullptr;
    if (tok[u] >= count) {
      if (dense) store8(dense, Eight<T>{});
      continue;
    }
    const float sc = round_to<T>(fmaxf(__fdiv_rn(hi - lo, top), 1e-8f));
    const float bi = round_to<T>(lo);
    codes8<BITS>(x, bi, sc, q);
    const uint32_t at = row_of(p.c.map, b[u], h[u], static_cast<int64_t>(__ldg(p.offsets + b[u])) + tok[u]);
    if (at == kNoRow) {
      atomicExch(p.error_flag, PHEW_ERR_INVALID);
    } else {
      uint32_t w[BITS / 4] = {};
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e * BITS / 32] |= static_cast<uint32_t>(q[e]) << (e * BITS % 32);
      uint32_t* dst = p.c.codes[side] + (static_cast<int64_t>(at) * lanes + c) * (BITS / 4);
      if (BITS == 4)
        dst[0] = w[0];
      else
        *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[BITS / 4 - 1]);
      if ((c & (LG - 1)) == 0) {
        const int64_t s_at = static_cast<int64_t>(at) * ng + c / LG;
        static_cast<T*>(p.c.scales[side])[s_at] = from_f32<T>(sc);
        static_cast<T*>(p.c.biases[side])[s_at] = from_f32<T>(bi);
      }
    }
    if (dense) {
      Eight<T> out;
#pragma unroll
      for (int e = 0; e < 8; ++e) out.v[e] = from_f32<T>(fmaf(sc, q[e], bi));
      store8(dense, out);
    }
  }
}

struct FetchParams {
  Cache c;
  void* dense[2];  // [batch][kv_heads][out_len][D]
  const int32_t* lengths;
  RowSplit split;
  int rows;
  int* error_flag;
};

// Bound by HBM, mostly by the values written: eight codes (one or two words)
// and their group's scale and bias to a thread, 16 bytes of 16-bit values out.
template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads) fetch_kernel(const FetchParams p) {
  const int side = blockIdx.y;
  const int lanes = p.c.head_dim / 8;
  const int per_pass = kThreads / lanes;
  const int c = threadIdx.x & (lanes - 1);
  const int row0 = blockIdx.x * (per_pass * kRows) + static_cast<int>(threadIdx.x) / lanes;
  const int ng = p.c.head_dim / p.c.group, grp = c * 8 / p.c.group;
  uint32_t at[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int row = row0 + u * per_pass;
    at[u] = kNoRow;
    if (row < p.rows) {
      int b, h, pos;
      split_row(p.split, row, b, h, pos);
      if (pos < __ldg(p.lengths + b)) {
        at[u] = row_of(p.c.map, b, h, pos);
        if (at[u] == kNoRow) atomicExch(p.error_flag, PHEW_ERR_INVALID);
      }
    }
  }
  uint32_t w[kRows][BITS / 4];
  T sc[kRows], bi[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    if (at[u] == kNoRow) continue;
    const uint32_t* src = p.c.codes[side] + (static_cast<int64_t>(at[u]) * lanes + c) * (BITS / 4);
    if (BITS == 4) {
      w[u][0] = __ldg(src);
    } else {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
      w[u][0] = v.x;
      w[u][BITS / 4 - 1] = v.y;
    }
    const int64_t s_at = static_cast<int64_t>(at[u]) * ng + grp;
    sc[u] = static_cast<const T*>(p.c.scales[side])[s_at];
    bi[u] = static_cast<const T*>(p.c.biases[side])[s_at];
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int row = row0 + u * per_pass;
    if (row >= p.rows) continue;
    Eight<T> out{};
    if (at[u] != kNoRow) {
      const float s = to_f32(sc[u]), z = to_f32(bi[u]);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        out.v[e] = from_f32<T>(fmaf(s, static_cast<float>((w[u][e * BITS / 32] >> (e * BITS % 32)) & ((1 << BITS) - 1)), z));
    }
    store8(static_cast<T*>(p.dense[side]) + static_cast<int64_t>(row) * p.c.head_dim + c * 8, out);
  }
}

// Blocks along x for `rows` token rows of a side.
dim3 grid_for(int64_t rows, int head_dim) {
  const int64_t per_block = static_cast<int64_t>(kThreads / (head_dim / 8)) * kRows;
  return dim3(static_cast<unsigned>((rows + per_block - 1) / per_block), 2);
}

template <typename T, int BITS> void launch_update(const UpdateParams& p, cudaStream_t st) {
  const dim3 grid = grid_for(p.rows, p.c.head_dim);
  switch (p.c.group) {
    case 32: update_kernel<T, BITS, 32><<<grid, kThreads, 0, st>>>(p); break;
    case 64: update_kernel<T, BITS, 64><<<grid, kThreads, 0, st>>>(p); break;
    default: update_kernel<T, BITS, 128><<<grid, kThreads, 0, st>>>(p); break;
  }
}

template <typename T> int update_typed(const UpdateParams& p, cudaStream_t st) {
  if (p.c.bits == 4)
    launch_update<T, 4>(p, st);
  else
    launch_update<T, 8>(p, st);
  return launch_status("kv update_kernel");
}

template <typename T> int fetch_typed(const FetchParams& p, cudaStream_t st) {
  const dim3 grid = grid_for(p.rows, p.c.head_dim);
  if (p.c.bits == 4)
    fetch_kernel<T, 4><<<grid, kThreads, 0, st>>>(p);
  else
    fetch_kernel<T, 8><<<grid, kThreads, 0, st>>>(p);
  return launch_status("kv fetch_kernel");
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
  PHEW_REQUIRE(tokens > 0 && tokens < (1ll << 31) && batch * cache->kv_heads < kv::kMaxRows / tokens,
               "phew_kv_update: bad token count (batch * kv_heads * tokens must stay below 2^31 - 2^16)");
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
  p.split = {kv::fast_div(static_cast<uint32_t>(tokens)), kv::fast_div(static_cast<uint32_t>(cache->kv_heads))};
  p.rows = static_cast<int>(batch * cache->kv_heads * tokens);
  p.tokens = static_cast<int>(tokens);
  p.error_flag = error_flag;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (cache->dtype) {
    case PHEW_F32: return kv::update_typed<float>(p, st);
    case PHEW_F16: return kv::update_typed<f16>(p, st);
    default: return kv::update_typed<bf16>(p, st);
  }
}

extern "C" int phew_kv_fetch(const phew_kv_cache* cache, void* k_out, void* v_out, int64_t batch, int64_t out_len,
                             const int* lengths, const int* block_table, int64_t table_stride, int64_t columns,
                             int* error_flag, void* stream) {
  kv::FetchParams p;
  if (int s = kv::make_cache(cache, block_table, table_stride, columns, batch, "phew_kv_fetch", &p.c)) return s;
  PHEW_REQUIRE(k_out && v_out && lengths && error_flag, "phew_kv_fetch: null pointer");
  PHEW_REQUIRE(out_len > 0 && out_len < (1ll << 31) && batch * cache->kv_heads < kv::kMaxRows / out_len,
               "phew_kv_fetch: bad output length (batch * kv_heads * length must stay below 2^31 - 2^16)");
  for (const void* q : {k_out, v_out})
    PHEW_REQUIRE((reinterpret_cast<uintptr_t>(q) & 15) == 0, "phew_kv_fetch: pointers must be 16-byte aligned");
  p.dense[0] = k_out;
  p.dense[1] = v_out;
  p.lengths = lengths;
  p.split = {kv::fast_div(static_cast<uint32_t>(out_len)), kv::fast_div(static_cast<uint32_t>(cache->kv_heads))};
  p.rows = static_cast<int>(batch * cache->kv_heads * out_len);
  p.error_flag = error_flag;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (cache->dtype) {
    case PHEW_F32: return kv::fetch_typed<float>(p, st);
    case PHEW_F16: return kv::fetch_typed<f16>(p, st);
    default: return kv::fetch_typed<bf16>(p, st);
  }
}
