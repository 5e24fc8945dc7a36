// Softmax pieces of the tcgen05 attention kernels: one thread per query row,
// its 128 scores of a key tile in registers, weights written back to TMEM.
#pragma once

#include "tc_common.cuh"

namespace phew {
namespace attn {

using namespace tc;

// ---- scalar and packed (f32x2) arithmetic helpers ----
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t f2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float lo_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float hi_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// max(a, b, c); like fmaxf a NaN operand is ignored.  (A NaN score still
// poisons its row: exp2 of it is NaN and so is the row sum.)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t d;
  if (BF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// P = exp2(raw * c - m) over one row of 128 scores, packed into 64 16-bit
// pairs and stored to TMEM at s_addr (columns 0..63 of the S buffer).
// Returns the row sum of this tile's (unrounded) P.
template <bool BF16>
__device__ __forceinline__ float compute_p(const uint32_t* raw, float c, float m, uint32_t s_addr) {
  const uint64_t c2 = f2(c, c), nm2 = f2(-m, -m);
  uint64_t l2[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int pi = 16 * h + i;
      const uint64_t x = fma2(f2(__uint_as_float(raw[2 * pi]), __uint_as_float(raw[2 * pi + 1])), c2, nm2);
      const uint64_t e = f2(ex2(lo_of(x)), ex2(hi_of(x)));
      l2[i & 1] = add2(l2[i & 1], e);
      pk[i] = pack2<BF16>(lo_of(e), hi_of(e));
    }
    tmem_st16(s_addr + 16 * h, pk);
  }
  const uint64_t l = add2(l2[0], l2[1]);
  return lo_of(l) + hi_of(l);
}

// max over 128 scores: eight independent chains of three-input max.
__device__ __forceinline__ float row_max(const uint32_t* raw) {
  float m8[8];
#pragma unroll
  for (int a = 0; a < 8; ++a)
    m8[a] = max3(__uint_as_float(raw[3 * a]), __uint_as_float(raw[3 * a + 1]), __uint_as_float(raw[3 * a + 2]));
#pragma unroll
  for (int i = 24; i + 16 <= 128; i += 16)
#pragma unroll
    for (int a = 0; a < 8; ++a)
      m8[a] = max3(m8[a], __uint_as_float(raw[i + 2 * a]), __uint_as_float(raw[i + 2 * a + 1]));
#pragma unroll
  for (int a = 0; a < 8; ++a) m8[a] = fmaxf(m8[a], __uint_as_float(raw[120 + a]));
  return max3(max3(m8[0], m8[1], m8[2]), max3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7]));
}

}  // namespace attn
}  // namespace phew
