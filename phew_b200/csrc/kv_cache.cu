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
// row what phew_dequantize gives.  But a group that holds a NaN gets NaN for
// scale and bias (codes 0), so that it reads back as NaN, where phew_quantize
// passes over it.
#include <type_traits>

#include "common.cuh"
#include "kv_cache.cuh"

namespace phew {
namespace kv {
namespace {

constexpr int kThreads = 128;

// Two floats in one 64-bit register, for the packed fp32 instructions (each half rounds like the scalar one).
__device__ __forceinline__ uint64_t two(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float lo_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float hi_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
// Eight consecutive elements of a token row, as they lie in memory.
template <typename T> struct Eight {
  uint32_t w[2 * sizeof(T)];
};
template <typename T> __device__ __forceinline__ Eight<T> load8(const T* p) {
  Eight<T> e;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
    e.w[4 * i] = v.x;
    e.w[4 * i + 1] = v.y;
    e.w[4 * i + 2] = v.z;
    e.w[4 * i + 3] = v.w;
  }
  return e;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const Eight<T>& e) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i)
    reinterpret_cast<uint4*>(p)[i] = make_uint4(e.w[4 * i], e.w[4 * i + 1], e.w[4 * i + 2], e.w[4 * i + 3]);
}
template <typename T> __device__ __forceinline__ uint32_t pack(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack<bf16>(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
template <> __device__ __forceinline__ uint32_t pack<f16>(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// Elements 2i, 2i + 1 as floats, and back.
__device__ __forceinline__ uint64_t pair_of(const Eight<float>& e, int i) {
  return two(__uint_as_float(e.w[2 * i]), __uint_as_float(e.w[2 * i + 1]));
}
__device__ __forceinline__ uint64_t pair_of(const Eight<bf16>& e, int i) {
  return two(__uint_as_float(e.w[i] << 16), __uint_as_float(e.w[i] & 0xffff0000u));
}
__device__ __forceinline__ uint64_t pair_of(const Eight<f16>& e, int i) {
  return two(to_f32(f16{static_cast<uint16_t>(e.w[i])}), to_f32(f16{static_cast<uint16_t>(e.w[i] >> 16)}));
}
template <typename T> __device__ __forceinline__ void set_pair(Eight<T>& e, int i, uint64_t v) {
  if constexpr (sizeof(T) == 4) {
    e.w[2 * i] = static_cast<uint32_t>(v);
    e.w[2 * i + 1] = static_cast<uint32_t>(v >> 32);
  } else {
    e.w[i] = pack<T>(lo_of(v), hi_of(v));
  }
}

// Smallest and largest of the eight, NaN if one of them is.  The 16-bit types keep (min, -max) as one
// packed pair, so a step across lanes is one shuffle and one packed minimum.
template <typename T> struct Range {
  uint32_t p;
  static __device__ __forceinline__ uint32_t min_of(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (std::is_same<T, bf16>::value)
      asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else
      asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
  __device__ __forceinline__ void of(const Eight<T>& e) {
    constexpr uint32_t neg = 0x80008000u;
    const uint32_t lo = min_of(min_of(e.w[0], e.w[1]), min_of(e.w[2], e.w[3]));
    const uint32_t hi = min_of(min_of(e.w[0] ^ neg, e.w[1] ^ neg), min_of(e.w[2] ^ neg, e.w[3] ^ neg));
    p = min_of(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));
  }
  __device__ __forceinline__ void with(const Range& o) { p = min_of(p, o.p); }
  __device__ __forceinline__ void across(int lanes) {
#pragma unroll
    for (int o = lanes / 2; o > 0; o >>= 1) p = min_of(p, __shfl_xor_sync(0xffffffffu, p, o));
  }
  __device__ __forceinline__ float lo() const { return to_f32(T{static_cast<uint16_t>(p)}); }
  __device__ __forceinline__ float hi() const { return -to_f32(T{static_cast<uint16_t>(p >> 16)}); }
};
template <> struct Range<float> {
  float a, b;
  static __device__ __forceinline__ float min_of(float x, float y) {
    float d;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(x), "f"(y));
    return d;
  }
  static __device__ __forceinline__ float max_of(float x, float y) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(x), "f"(y));
    return d;
  }
  __device__ __forceinline__ void of(const Eight<float>& e) {
    a = b = __uint_as_float(e.w[0]);
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      a = min_of(a, __uint_as_float(e.w[i]));
      b = max_of(b, __uint_as_float(e.w[i]));
    }
  }
  __device__ __forceinline__ void with(const Range& o) {
    a = min_of(a, o.a);
    b = max_of(b, o.b);
  }
  __device__ __forceinline__ void across(int lanes) {
#pragma unroll
    for (int o = lanes / 2; o > 0; o >>= 1) {
      a = min_of(a, __shfl_xor_sync(0xffffffffu, a, o));
      b = max_of(b, __shfl_xor_sync(0xffffffffu, b, o));
    }
  }
  __device__ __forceinline__ float lo() const { return a; }
  __device__ __forceinline__ float hi() const { return b; }
};

// A row number in [0, 2^31) of a [batch][kv_heads][n] array, taken apart.
struct RowSplit {
  FastDiv by_n, by_heads;
};
struct Row {
  int b, h, i;
};
__device__ __forceinline__ Row split_row(const RowSplit& s, int row) {
  Row r;
  const int bh = static_cast<int>(div_by(s.by_n, static_cast<uint32_t>(row)));
  r.i = row - bh * static_cast<int>(s.by_n.d);
  r.b = static_cast<int>(div_by(s.by_heads, static_cast<uint32_t>(bh)));
  r.h = bh - r.b * static_cast<int>(s.by_heads.d);
  return r;
}
// Row `first` + l of a block of at most `most` rows whose first is known: no division where a block spans two
// heads at most.
__device__ __forceinline__ Row row_after(const RowSplit& s, const Row& first, int first_row, int l, uint32_t most) {
  if (s.by_n.d < most) return split_row(s, first_row + l);
  Row r = first;
  r.i += l;
  if (r.i >= static_cast<int>(s.by_n.d)) {
    r.i -= static_cast<int>(s.by_n.d);
    if (++r.h == static_cast<int>(s.by_heads.d)) {
      r.h = 0;
      ++r.b;
    }
  }
  return r;
}

// Token rows a thread works on at once: their loads are in flight together (1, 2, 4 of them: 227, 225, 275 us for
// the writes that update_kernel's comment names, 102, 99, 107 for fetch_kernel's reads; blocks of 256 threads 238, 101).
constexpr int kRows = 2;

// 1.5 2^23: a float in [0, 2^22) added to it leaves the nearest whole number (ties to even) in the low bits.
constexpr float kRound = 12582912.f;
constexpr uint32_t kRoundBits = 0x4B400000u;

struct UpdateParams {
  Cache c;
  const void* x[2];      // k, v
  int64_t st[2][3];      // their token, head and batch strides (elements)
  void* dense[2];        // values written back, [batch][kv_heads][tokens][D]; null: none
  const int32_t* offsets;
  const int32_t* counts;  // null: all `tokens`
  RowSplit split;
  int rows;
  int* error_flag;
};

// The group's scale and bias, and the reciprocal that codes are taken with.
struct Affine {
  float sc, bi, inv;
  bool plain;  // quotients lie in [0, top + 1/2), or with `over` in [0, top + 3/2), and the reciprocal's steps give them
  bool over;   // the largest codes are to be held at top: bf16 rounds a scale by 2^-8 of it, one code in 255 (7 % of
               // groups of 64 normals; the other types' roundings stay below half a code)
};
template <typename T, int BITS> __device__ __forceinline__ Affine affine_of(const Range<T>& r) {
  constexpr float top = (1 << BITS) - 1, part = 1.f / top;
  Affine a;
  const float lo = r.lo(), hi = r.hi(), d = hi - lo;
  // d / top by the rounded reciprocal of top and the remainder: the IEEE quotient (Markstein, "Computation of
  // elementary functions on the IBM RISC System/6000 processor", 1990; checked for every mantissa of d) unless
  // something over- or underflows; below 1e-8 it does not count
  float q = d * part;
  q = fmaf(fmaf(-top, q, d), part, q);
  if (!(d < 1e38f)) q = __fdiv_rn(d, top);
  a.sc = lo == lo ? round_to<T>(fmaxf(q, 1e-8f)) : lo;
  a.bi = lo;  // a value of type T
  if (sizeof(T) == 2) {
    // one Newton step from one unit in the last place: the rounded reciprocal of a mantissa of 8 or 11 bits
    // (whose reciprocals keep 2^-36 away from the middle between two floats)
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(a.sc));
    a.inv = fmaf(fmaf(-a.sc, y, 1.f), y, y);
  } else {
    a.inv = __frcp_rn(a.sc);
  }
  constexpr bool holds = std::is_same<T, bf16>::value && BITS == 8;
  const float most = d * a.inv;
  a.plain = most < top + (holds ? 1.4999f : 0.4999f);
  a.over = holds && most >= top + 0.4999f;
  if (sizeof(T) == 4) a.plain = a.plain && (__float_as_uint(a.sc) & 0x7fffffu) != 0x7fffffu;
  return a;
}

// Codes of eight values: words for the cache, and as floats.  (x - bias) /
// scale is the product with the rounded reciprocal corrected by its remainder
// (Markstein's steps: one gives the IEEE quotient of a 16-bit type's short
// scale, two that of any scale but the one of all-ones mantissa), two values to
// an instruction.  Ties between codes are frequent in 16-bit data (one value
// in 450 of bf16 normals), so a quotient that is only nearly right would need
// a second look in every third warp.
template <typename T, int BITS>
__device__ __forceinline__ void codes8(const Eight<T>& x, const Affine& a, uint32_t* words, uint64_t* q) {
  constexpr float top = (1 << BITS) - 1;
  const uint64_t nb = two(-a.bi, -a.bi), inv = two(a.inv, a.inv), ns = two(-a.sc, -a.sc);
  const uint64_t up = two(kRound, kRound), down = two(-kRound, -kRound);
  uint64_t t[4], any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t d = add2(pair_of(x, i), nb);
    any = add2(any, d);
    uint64_t v = mul2(d, inv);
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(T)) / 2; ++k) v = fma2(fma2(ns, v, d), inv, v);
    t[i] = add2(v, up);
    q[i] = add2(t[i], down);
  }
  if (a.over) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = two(fminf(lo_of(t[i]), kRound + top), fminf(hi_of(t[i]), kRound + top));
      q[i] = add2(t[i], down);
    }
  }
  if (!a.plain || !(lo_of(any) + hi_of(any) < INFINITY)) {  // odd scales, or a value that is no number (code 0)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t xs = pair_of(x, i);
      float f[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        f[k] = fminf(fmaxf(rintf(__fdiv_rn((k ? hi_of(xs) : lo_of(xs)) - a.bi, a.sc)), 0.f), top);
      q[i] = two(f[0], f[1]);
      t[i] = add2(q[i], up);
    }
  }
#pragma unroll
  for (int w = 0; w < BITS / 4; ++w) {
    uint32_t sum = 0u - kRoundBits * (BITS == 4 ? 0x11111111u : 0x01010101u);
#pragma unroll
    for (int e = 0; e < 32 / BITS; ++e) {
      const uint64_t p = t[(w * (32 / BITS) + e) / 2];
      sum += static_cast<uint32_t>(e & 1 ? p >> 32 : p) << (e * BITS);
    }
    words[w] = sum;
  }
}

// Bound by HBM (update of 4 x 32 heads x 8192 tokens of 128 bf16 values with
// the values written back: 1.22 GB in 225 us, 5.4 TB/s, 0.83 of the copy rate)
// and by issue slots (0.69 of them).  A thread takes sixteen neighbouring
// values of a row, so that its address and the group's scale are worked out once
// for them; a group is G / 16 neighbouring lanes.  (Eight of either half of the
// row make every access of a warp contiguous: 4 % faster for f32 with its values
// written back, 4 to 10 % slower for the 16-bit types and without values.)
template <typename T, int BITS, int D, int G>
__global__ void __launch_bounds__(kThreads) update_kernel(const UpdateParams p) {
  constexpr int LANES = D / 16;                 // threads to a row
  constexpr int PER_PASS = kThreads / LANES;    // rows to a pass of the block
  constexpr int LG = G / 16;                    // lanes of a group
  constexpr int NG = D / G;
  const int side = blockIdx.y;
  const int c = threadIdx.x % LANES;
  const int first_row = blockIdx.x * (PER_PASS * kRows), row0 = first_row + static_cast<int>(threadIdx.x) / LANES;
  const Row first = split_row(p.split, first_row);
  const T* xs = static_cast<const T*>(p.x[side]);
  Eight<T> in[kRows][2];
  bool have[kRows];     // a row of x
  bool live[kRows];     // ... that goes into the cache
  uint32_t at[kRows];   // ... there
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int row = row0 + u * PER_PASS;
    have[u] = row < p.rows;
    live[u] = false;
    at[u] = kNoRow;
    in[u][0] = in[u][1] = Eight<T>{};
    if (have[u]) {
      const Row r = row_after(p.split, first, first_row, row - first_row, PER_PASS * kRows);
      const T* x = xs + r.b * p.st[side][2] + r.h * p.st[side][1] + r.i * p.st[side][0] + c * 16;
      in[u][0] = load8(x);
      in[u][1] = load8(x + 8);
      live[u] = !p.counts || r.i < __ldg(p.counts + r.b);
      if (live[u]) {
        at[u] = row_of(p.c.map, r.b, r.h, static_cast<int64_t>(__ldg(p.offsets + r.b)) + r.i);
        if (at[u] == kNoRow) atomicExch(p.error_flag, PHEW_ERR_INVALID);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    Range<T> r, r1;
    r.of(in[u][0]);
    r1.of(in[u][1]);
    r.with(r1);
    r.across(LG);
    if (!have[u]) continue;
    T* dense = nullptr;
    if (p.dense[side]) dense = static_cast<T*>(p.dense[side]) + static_cast<int64_t>(row0 + u * PER_PASS) * D + c * 16;
    if (!live[u]) {
      if (dense) {
        store8(dense, Eight<T>{});
        store8(dense + 8, Eight<T>{});
      }
      continue;
    }
    const Affine a = affine_of<T, BITS>(r);
    uint32_t words[2][BITS / 4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint64_t q[4];
      codes8<T, BITS>(in[u][half], a, words[half], q);
      if (dense) {
        Eight<T> out;
#pragma unroll
        for (int i = 0; i < 4; ++i) set_pair(out, i, fma2(two(a.sc, a.sc), q[i], two(a.bi, a.bi)));
        store8(dense + half * 8, out);
      }
    }
    if (at[u] != kNoRow) {
      uint32_t* dst = p.c.codes[side] + static_cast<int64_t>(at[u]) * (D * BITS / 32) + c * (BITS / 2);
      if (BITS == 4)
        *reinterpret_cast<uint2*>(dst) = make_uint2(words[0][0], words[1][0]);
      else
        *reinterpret_cast<uint4*>(dst) = make_uint4(words[0][0], words[0][BITS / 4 - 1], words[1][0], words[1][BITS / 4 - 1]);
      if (c % LG == 0) {
        const int64_t s_at = static_cast<int64_t>(at[u]) * NG + c / LG;
        static_cast<T*>(p.c.scales[side])[s_at] = from_f32<T>(a.sc);
        static_cast<T*>(p.c.biases[side])[s_at] = from_f32<T>(a.bi);
      }
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

// Bound by HBM, mostly by the values written (16 ragged sequences of up to
// 8192 tokens, 8 heads of 128 in bf16: 99 us, 0.96 of the copy rate).  Eight
// codes of either half of a row to a thread, so that every access of a warp is
// contiguous.  A code becomes a float by a byte permutation into 2^23 + code
// (conversions run at an eighth of the rate), two values to an instruction from
// there.
template <typename T, int BITS, int D>
__global__ void __launch_bounds__(kThreads) fetch_kernel(const FetchParams p) {
  constexpr int LANES = D / 16;
  constexpr int PER_PASS = kThreads / LANES;
  constexpr int W = BITS / 4;  // words of eight codes
  const int side = blockIdx.y;
  const int c = threadIdx.x % LANES;
  const int first_row = blockIdx.x * (PER_PASS * kRows), row0 = first_row + static_cast<int>(threadIdx.x) / LANES;
  const Row first = split_row(p.split, first_row);
  const int ng = D / p.c.group, shift = p.c.group == 32 ? 5 : p.c.group == 64 ? 6 : 7;
  uint32_t at[kRows];
  bool skip[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int row = row0 + u * PER_PASS;
    at[u] = kNoRow;
    skip[u] = row >= p.rows;
    if (row < p.rows) {
      const Row r = row_after(p.split, first, first_row, row - first_row, PER_PASS * kRows);
      const int length = __ldg(p.lengths + r.b);
      if (r.i < length) {
        at[u] = row_of(p.c.map, r.b, r.h, r.i);
        if (at[u] == kNoRow) atomicExch(p.error_flag, PHEW_ERR_INVALID);
      }
    }
  }
  uint32_t w[kRows][2][W];
  T sc[kRows][2], bi[kRows][2];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    if (at[u] == kNoRow) continue;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint32_t* src = p.c.codes[side] + static_cast<int64_t>(at[u]) * (D * BITS / 32) + (half * (D / 16) + c) * W;
      if (BITS == 4) {
        w[u][half][0] = __ldg(src);
      } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
        w[u][half][0] = v.x;
        w[u][half][W - 1] = v.y;
      }
      const int64_t s_at = static_cast<int64_t>(at[u]) * ng + ((half * (D / 2) + c * 8) >> shift);
      sc[u][half] = static_cast<const T*>(p.c.scales[side])[s_at];
      bi[u][half] = static_cast<const T*>(p.c.biases[side])[s_at];
    }
  }
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const int row = row0 + u * PER_PASS;
    if (skip[u]) continue;
    T* dst = static_cast<T*>(p.dense[side]) + static_cast<int64_t>(row) * D + c * 8;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      Eight<T> out{};
      if (at[u] != kNoRow) {
        const float s = to_f32(sc[u][half]), z = to_f32(bi[u][half]);
        constexpr uint32_t base = 0x4B000000u;  // 2^23
        // even and odd codes of 4 bits, or all of 8, a byte each
        const uint32_t even = BITS == 4 ? w[u][half][0] & 0x0f0f0f0fu : w[u][half][0];
        const uint32_t odd = BITS == 4 ? (w[u][half][0] >> 4) & 0x0f0f0f0fu : w[u][half][W - 1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t lo, hi;
          if (BITS == 4) {
            lo = __byte_perm(even, base, 0x7540 + i);
            hi = __byte_perm(odd, base, 0x7540 + i);
          } else {
            lo = __byte_perm(i < 2 ? even : odd, base, 0x7540 + 2 * (i & 1));
            hi = __byte_perm(i < 2 ? even : odd, base, 0x7541 + 2 * (i & 1));
          }
          const uint64_t n = add2(two(__uint_as_float(lo), __uint_as_float(hi)), two(-8388608.f, -8388608.f));
          set_pair(out, i, fma2(two(s, s), n, two(z, z)));
        }
      }
      store8(dst + half * (D / 2), out);
    }
  }
}

// Blocks along x for `rows` token rows of a side.
dim3 grid_for(int64_t rows, int head_dim) {
  const int64_t per_block = static_cast<int64_t>(kThreads / (head_dim / 16)) * kRows;
  return dim3(static_cast<unsigned>((rows + per_block - 1) / per_block), 2);
}

template <typename T, int BITS> void launch_update(const UpdateParams& p, cudaStream_t st) {
  const dim3 grid = grid_for(p.rows, p.c.head_dim);
#define PHEW_KV_UPDATE(D, G) \
  if (p.c.head_dim == D && p.c.group == G) return update_kernel<T, BITS, D, G><<<grid, kThreads, 0, st>>>(p)
  PHEW_KV_UPDATE(64, 32);
  PHEW_KV_UPDATE(64, 64);
  PHEW_KV_UPDATE(128, 32);
  PHEW_KV_UPDATE(128, 64);
  PHEW_KV_UPDATE(128, 128);
  PHEW_KV_UPDATE(256, 32);
  PHEW_KV_UPDATE(256, 64);
  PHEW_KV_UPDATE(256, 128);
#undef PHEW_KV_UPDATE
}

template <typename T> int update_typed(const UpdateParams& p, cudaStream_t st) {
  if (p.c.bits == 4)
    launch_update<T, 4>(p, st);
  else
    launch_update<T, 8>(p, st);
  return launch_status("kv update_kernel");
}

template <typename T, int BITS> void launch_fetch(const FetchParams& p, cudaStream_t st) {
  const dim3 grid = grid_for(p.rows, p.c.head_dim);
  switch (p.c.head_dim) {
    case 64: fetch_kernel<T, BITS, 64><<<grid, kThreads, 0, st>>>(p); break;
    case 128: fetch_kernel<T, BITS, 128><<<grid, kThreads, 0, st>>>(p); break;
    default: fetch_kernel<T, BITS, 256><<<grid, kThreads, 0, st>>>(p); break;
  }
}

template <typename T> int fetch_typed(const FetchParams& p, cudaStream_t st) {
  if (p.c.bits == 4)
    launch_fetch<T, 4>(p, st);
  else
    launch_fetch<T, 8>(p, st);
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
