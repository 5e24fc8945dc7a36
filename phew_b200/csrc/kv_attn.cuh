// Attention of few query rows over a 4-bit cache (decode, drafted tokens).
//
//   s_rj = scale * sum_g sk[j,g] (q_r . c_j)_g + (zk[j,g] + 8 sk[j,g]) sum(q_r)_g
//   o_r  = sum_j p_rj (sum_g sv[j,g] c_j + (zv[j,g] + 8 sv[j,g])) / sum_j p_rj
//
// with c = code - 8, a whole number that bf16 and f16 hold exactly: scales and
// biases never touch a code, they act on the small score tile (keys) and on
// the softmax weights (values).  A cache head's `per` query heads and the
// query tokens are the rows r = token * per + head, eight or sixteen to a
// block, so keys and values are read once for all of them.
//
// Bound by HBM (a packed row of 128 with groups of 64 is 72 bytes): at 6.5
// TB/s an SM gets 41 codes a clock, which leaves about three instruction
// lanes for each.  So
//  * both products run on mma.sync m16n8k16 with keys (scores) and head
//    dimension (output) along m and the few query rows along n: no padding
//    of eight rows to sixteen, and codes go from packed words to fragments in
//    registers with one shift and one logic operation per pair.  (tcgen05
//    would need the codes as 16-bit tiles in shared memory: four times the
//    bytes, written and read once more than the 128 bytes a clock an SM has.)
//  * a word's eight codes stay with the thread that loads it: the order of
//    the head dimension inside a product is free, so queries are arranged to
//    match (pairs i, i + 4 of a word) and nothing is shuffled;
//  * weights move from the score fragment (key-major) to the operand of the
//    second product by movmatrix, in registers;
//  * every warp walks its own 32 of each 128 keys with its own running
//    maximum and sum and its own ring of cp.async stages: no block barrier in
//    the loop; warps join in shared memory once per segment.
//
// Work split: the (sequence, row block, cache head) segments of all
// sequences, cut into tiles of 128 keys, are one line of W tiles; block c of n
// takes tiles [cW/n, (c+1)W/n), so any mix of lengths loads the SMs evenly and
// no host ever needs the lengths.  A segment that lies in one block is
// finished there; a cut one leaves partial sums (maximum, sum, output) that
// the combine kernel joins in a fixed order.
#pragma once

#include <atomic>
#include <type_traits>

#include "kv_cache.cuh"

namespace phew {
namespace kv {

constexpr int kWarps = 4;
constexpr int kStageKeys = 32;                  // keys of one warp's stage
constexpr int kTile = kWarps * kStageKeys;      // keys of one block step
constexpr float kGrow = 8.0f;                   // log2 units a score may pass the running maximum by
constexpr float kFloor = -1.0e38f;              // running maximum before the first key

struct AttnParams {
  Cache c;
  const void* q;
  int64_t st[3];  // q's token, head and batch strides (elements)
  void* o;        // [batch][heads][tokens][D]
  const int32_t* lengths;
  const int32_t* counts;  // null: all `tokens`
  int batch, heads, tokens, per;  // per: query heads to a cache head
  int blocks;                     // row blocks of a sequence's tokens * per rows
  FastDiv by_per, by_blocks;
  float scale_log2;
  bool causal;
  float* part;   // [n][2][rows][D] partial outputs, then [n][2][rows][2] (maximum, sum)
  float* part_ml;
  int64_t* meta;  // [n][2]: segment of partial 0 (begun by an earlier block) and 1 (left to later ones); -1: none
  int* error_flag;
};

// One sequence's row block.
struct Entry {
  int b, block;
  int length, count;
  int end;    // keys [0, end) that any of its rows sees
  int tiles;  // at least one, so that some block writes the rows of an empty one
};

__device__ __forceinline__ Entry entry_at(const AttnParams& p, int e, int rows) {
  Entry t;
  t.b = static_cast<int>(div_by(p.by_blocks, static_cast<uint32_t>(e)));
  t.block = e - t.b * p.blocks;
  t.count = p.counts ? clamp_count(__ldg(p.counts + t.b), p.tokens) : p.tokens;
  t.length = clamp_count(__ldg(p.lengths + t.b), capacity(p.c.map));
  const int first = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(t.block * rows)));
  const int last = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(t.block * rows + rows - 1)));
  t.end = first >= t.count ? 0 : seen_end(t.length, t.count, last < t.count ? last : t.count - 1, p.causal);
  t.tiles = t.end > kTile ? (t.end + kTile - 1) / kTile : 1;
  return t;
}

template <typename T, int D_, int G_, int NT_> struct Shape {
  static constexpr int D = D_, G = G_, NT = NT_;
  static constexpr int ROWS = 8 * NT;
  static constexpr int NG = D / G;
  static constexpr bool F32 = sizeof(T) == 4;
  // terms of a value split into bf16: queries (f32: 24 bits in three; f16 and bf16 as they are) and weights
  // (bf16 results: one, 2^-9 of a weight; f16: two, 2^-17; f32: three)
  static constexpr int TQ = F32 ? 3 : 1;
  static constexpr int TP = F32 ? 3 : std::is_same<T, f16>::value ? 2 : 1;
  static constexpr int SB = NG * static_cast<int>(sizeof(T));   // bytes of a key's scales
  static constexpr int SROW = SB < 4 ? 4 : SB;
  static constexpr int CODE_BYTES = kStageKeys * D / 2;         // one side's codes of a stage
  static constexpr int STAGE = 2 * CODE_BYTES + 4 * kStageKeys * SROW;
  static constexpr int STAGES = D == 64 ? 4 : D == 128 ? 3 : 2;
  static constexpr int RING = STAGE * STAGES;                   // per warp
  static constexpr int OROW = D + 4;                            // floats of a row when warps join
  static constexpr int JOIN = kWarps * ROWS * (OROW + 2) * 4;
  static constexpr int SMEM = RING * kWarps > JOIN ? RING * kWarps : JOIN;
  static constexpr int CTAS = D == 256 ? (F32 || G == 32 ? 2 : 3) : D == 128 ? (F32 ? 2 : NT == 2 ? 3 : 4) : (F32 || NT == 2 ? 3 : 4);
};

// ---- small pieces ---------------------------------------------------------

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
template <int N> __device__ __forceinline__ void copy_async(uint32_t dst, const void* src, int valid) {
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(valid) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int N> __device__ __forceinline__ void load_words(uint32_t addr, uint32_t* w) {
  if constexpr (N == 1)
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
  else if constexpr (N == 2)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  else
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

template <typename T> __device__ __forceinline__ uint32_t pack_out(float lo, float hi) {
  return static_cast<uint32_t>(from_f32<T>(lo).bits) | static_cast<uint32_t>(from_f32<T>(hi).bits) << 16;
}

// (a & b) | c
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

// Codes u and u + 4 of w's two 16-bit halves' (bits 4u and 16 + 4u) as a pair of bf16 code - 8:
// 0x4300 | n is 128 + n, and 128 + n - 136 is exact.
template <int U> __device__ __forceinline__ uint32_t pair_bf16(uint32_t w) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(and_or(w >> (4 * U), 0x000f000fu, 0x43004300u)), "r"(0x43084308u));
  return d;
}
// The same as f16: with the code one digit further left 0x5400 | n << 4 is 64 + n.
template <int U> __device__ __forceinline__ uint32_t pair_f16(uint32_t w) {
  uint32_t d;
  const uint32_t x = U == 0 ? w << 4 : w >> (U == 0 ? 0 : 4 * U - 4);
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(and_or(x, 0x00f000f0u, 0x54005400u)), "r"(0x54805480u));
  return d;
}

template <bool HALF>
__device__ __forceinline__ void mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 8 x 8 transpose of 16-bit elements across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
  return d;
}

// 16-byte chunk of stage row r that chunk c is kept in: rows that one warp-wide
// load touches together then lie in different banks (bit-reversed row number
// above the rows that share a 128-byte line).
template <int D> __device__ __forceinline__ int swizzle(int r, int c) {
  if constexpr (D == 64)
    return c ^ ((r >> 2) & 1);
  else if constexpr (D == 128)
    return c ^ ((((r >> 1) & 1) << 1) | ((r >> 2) & 1));
  else
    return c ^ (((r & 1) << 2) | (r & 2) | ((r >> 2) & 1));
}

// Key that slot i of eight holds, in score rows and in the second product's
// k order alike: the pair of slots 2t, 2t + 1 is the keys t, t + 4, so that a
// warp's loads of value words take four neighbouring rows.
__device__ __forceinline__ int key_of_slot(int i) { return (i & ~7) | ((i >> 1) & 3) | ((i & 1) << 2); }

// ---- one warp's stage ring --------------------------------------------------

template <typename S, typename T> struct Ring {
  const Cache& c;
  uint32_t base;     // shared address of this warp's stages
  uint32_t* parity;  // per stage: odd rows (scales of two bytes: which half of the loaded word)
  int lane;

  // Starts the copy of the 32 rows that the lanes hold into stage `s`.
  __device__ __forceinline__ void issue(int s, uint32_t row) const {
    const uint32_t at = base + s * S::STAGE;
    constexpr int CH = S::D / 32;  // 16-byte chunks of a row
#pragma unroll
    for (int side = 0; side < 2; ++side) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int id = i * 32 + lane, r = id / CH, ch = id % CH;
        const uint32_t src = __shfl_sync(0xffffffffu, row, side == 0 ? key_of_slot(r) : r);
        const bool have = src != kNoRow;
        copy_async<16>(at + side * S::CODE_BYTES + r * (S::D / 2) + swizzle<S::D>(r, ch) * 16,
                       c.codes[side] + (have ? static_cast<int64_t>(src) * (S::D / 8) + ch * 4 : 0), have ? 16 : 0);
      }
    }
    const bool have = row != kNoRow;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const char* arr = static_cast<const char*>((a & 1) ? c.biases[a >> 1] : c.scales[a >> 1]);
      const uint32_t dst = at + 2 * S::CODE_BYTES + (a * kStageKeys + lane) * S::SROW;
      if constexpr (S::SB == 2) {
        // the aligned word around the two bytes; the array's last row alone has no partner behind it
        const int64_t off = (static_cast<int64_t>(have ? row : 0) * 2) & ~3ll;
        const uint32_t rows = static_cast<uint32_t>(c.map.pages) * static_cast<uint32_t>(c.map.kv_heads) *
                              static_cast<uint32_t>(c.map.page_size);
        copy_async<4>(dst, arr + off, !have ? 0 : (row | 1u) < rows ? 4 : 2);
      } else {
        constexpr int N = S::SB < 16 ? S::SB : 16;
#pragma unroll
        for (int i = 0; i < S::SB; i += N)
          copy_async<N>(dst + i, arr + (have ? static_cast<int64_t>(row) * S::SB + i : 0), have ? N : 0);
      }
    }
    if constexpr (S::SB == 2) {
      const uint32_t odd = __ballot_sync(0xffffffffu, row & 1);
      if (lane == 0) parity[s] = odd;
    }
    copy_commit();
  }

  // Scales (which = 0) or biases (1) of key `key` of stage `s` on one side, as floats.
  __device__ __forceinline__ void scales(int s, int side, int which, int key, float* out) const {
    const uint32_t at = base + s * S::STAGE + 2 * S::CODE_BYTES + ((side * 2 + which) * kStageKeys + key) * S::SROW;
    if constexpr (S::SB == 2) {
      uint32_t w;
      load_words<1>(at, &w);
      if ((parity[s] >> key) & 1) w >>= 16;
      T t;
      t.bits = static_cast<uint16_t>(w);
      out[0] = to_f32(t);
    } else {
      uint32_t w[S::SB / 4];
      constexpr int N = S::SB < 16 ? S::SB / 4 : 4;
#pragma unroll
      for (int i = 0; i < S::SB / 4; i += N) load_words<N>(at + i * 4, w + i);
#pragma unroll
      for (int g = 0; g < S::NG; ++g) {
        if constexpr (S::F32) {
          out[g] = __uint_as_float(w[g]);
        } else {
          T t;
          t.bits = static_cast<uint16_t>(g & 1 ? w[g / 2] >> 16 : w[g / 2] & 0xffff);
          out[g] = to_f32(t);
        }
      }
    }
  }
};

// ---- the kernel -----------------------------------------------------------------

template <typename S, typename T>
__global__ void __launch_bounds__(kWarps * 32, S::CTAS) attn_kernel(const AttnParams p) {
  constexpr int D = S::D, G = S::G, NT = S::NT, NG = S::NG, ROWS = S::ROWS, TQ = S::TQ, TP = S::TP;
  constexpr int WPT = G / 32;   // words of a group that one thread multiplies with the queries
  constexpr int WT = D / 32;    // of a row
  constexpr bool HALF = std::is_same<T, f16>::value;  // f16 queries: the score product runs in f16
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_red[kWarps];
  __shared__ int64_t s_prefix;
  __shared__ int s_entry;
  __shared__ uint32_t s_parity[kWarps][S::STAGES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r8 = lane >> 2, t4 = lane & 3;
  const int kv_heads = p.c.map.kv_heads;

  // ---- this block's share of the line of tiles ----
  const int entries = p.batch * p.blocks;
  int64_t mine = 0;
  for (int e = threadIdx.x; e < entries; e += kWarps * 32) {
    const Entry t = entry_at(p, e, ROWS);
    mine += t.tiles;
    if (blockIdx.x == 0 && t.block == 0 && __ldg(p.lengths + t.b) != t.length) atomicExch(p.error_flag, PHEW_ERR_INVALID);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) s_red[warp] = mine;
  __syncthreads();
  const int64_t total = (s_red[0] + s_red[1] + s_red[2] + s_red[3]) * kv_heads;
  const int64_t n = total < gridDim.x ? total : gridDim.x;
  if (blockIdx.x >= n) {
    if (threadIdx.x < 2) p.meta[2 * blockIdx.x + threadIdx.x] = -1;
    return;
  }
  asm volatile("griddepcontrol.launch_dependents;");  // the combine kernel may be set up from here on; it waits for this one
  int64_t x = total * blockIdx.x / n;
  const int64_t x_end = total * (blockIdx.x + 1) / n;
  // the entry that tile x belongs to: the first whose tiles, with those before it, pass x / kv_heads
  {
    const int64_t target = x / kv_heads;
    int64_t run = 0;
    for (int e0 = 0; e0 < entries; e0 += kWarps * 32) {
      const int e = e0 + static_cast<int>(threadIdx.x);
      const int64_t own = e < entries ? entry_at(p, e, ROWS).tiles : 0;
      int64_t inc = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
      }
      __syncthreads();
      if (lane == 31) s_red[warp] = inc;
      __syncthreads();
      for (int w = 0; w < warp; ++w) inc += s_red[w];
      inc += run;
      if (inc > target && inc - own <= target) {
        s_entry = e;
        s_prefix = inc - own;
      }
      run += s_red[0] + s_red[1] + s_red[2] + s_red[3];
      if (run > target) break;
    }
    __syncthreads();
  }
  int e = s_entry;
  int64_t base = s_prefix * kv_heads;
  int64_t left0 = -1, left1 = -1;  // segments of this block's two partials

  const Ring<S, T> ring{p.c, smem_addr(smem) + warp * S::RING, s_parity[warp], lane};

  while (x < x_end) {
    const Entry ent = entry_at(p, e, ROWS);
    for (; x < x_end && x < base + static_cast<int64_t>(kv_heads) * ent.tiles;) {
      const int h = static_cast<int>((x - base) / ent.tiles);
      const int64_t seg0 = base + static_cast<int64_t>(h) * ent.tiles;
      const int t0 = static_cast<int>(x - seg0);
      const int t1 = static_cast<int>((x_end < seg0 + ent.tiles ? x_end : seg0 + ent.tiles) - seg0);
      x = seg0 + t1;

      // ---- queries as the n operand, their group sums, and how far each row sees ----
      uint32_t qf[NT][TQ][WT][4];
      float qs[NT][2][NG];
      int lim[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = ent.block * ROWS + nt * 8 + r8;
        const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(r)));
        const bool have = tok < ent.count;
        const T* q = static_cast<const T*>(p.q) + ent.b * p.st[2] + (h * p.per + (r - tok * p.per)) * p.st[1] + tok * p.st[0];
        float sum[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          sum[g] = 0.f;
#pragma unroll
          for (int i = 0; i < WPT; ++i) {
            float v[8];
            const T* at = q + g * G + (t4 * WPT + i) * 8;
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = 0.f;
            if (have) {
              T raw[8];
#pragma unroll
              for (int k = 0; k < static_cast<int>(sizeof(T)) / 2; ++k)
                *reinterpret_cast<uint4*>(raw + k * (16 / sizeof(T))) = __ldg(reinterpret_cast<const uint4*>(at) + k);
#pragma unroll
              for (int k = 0; k < 8; ++k) v[k] = to_f32(raw[k]);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) sum[g] += v[k];
#pragma unroll
            for (int tq = 0; tq < TQ; ++tq)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                uint32_t w;
                if constexpr (HALF) {
                  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(v[k + 4]), "f"(v[k]));
                } else {
                  w = pack_bf16(v[k], v[k + 4]);
                  if (tq + 1 < TQ) {  // what the next term still has to carry
                    v[k] -= __uint_as_float(w << 16);
                    v[k + 4] -= __uint_as_float(w & 0xffff0000u);
                  }
                }
                qf[nt][tq][g * WPT + i][k] = w;
              }
          }
          sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
          sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
        }
        // rows of the score fragment's columns: 2 t4 and 2 t4 + 1
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
#pragma unroll
          for (int g = 0; g < NG; ++g) qs[nt][cc][g] = __shfl_sync(0xffffffffu, sum[g], (2 * t4 + cc) * 4);
          const int rr = ent.block * ROWS + nt * 8 + 2 * t4 + cc;
          const int tok_cc = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(rr)));
          // rows without a query run along unmasked (their weights are finite and never stored)
          lim[nt][cc] = tok_cc < ent.count ? seen_end(ent.length, ent.count, tok_cc, p.causal) : 0x7fffffff;
        }
      }
      int lim_min = lim[0][0];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) lim_min = min(lim_min, min(lim[nt][0], lim[nt][1]));
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, o));

      float acc[NT][D / 16][4];
      float m[NT][2], l[NT][2], bsum[NT][2][NG];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[nt][i][k] = 0.f;
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          m[nt][cc] = kFloor;
          l[nt][cc] = 0.f;
#pragma unroll
          for (int g = 0; g < NG; ++g) bsum[nt][cc][g] = 0.f;
        }
      }

      // ---- the ring: page numbers one stage ahead of the copies, copies STAGES - 1 ahead of the products ----
      const int steps = t1 - t0;
      int want_page = -1, want_r = 0;  // -1: no key
      bool want = false;
      auto look_up = [&](int i) {
        const int key = (t0 + i) * kTile + warp * kStageKeys + lane;
        want = i < steps && key < ent.end;
        if (want) {
          const int col = static_cast<int>(div_by(p.c.map.by_page, static_cast<uint32_t>(key)));
          want_r = key - col * p.c.map.page_size;
          want_page = page_at(p.c.map, ent.b, col);
        }
      };
      auto start_copy = [&](int i) {
        uint32_t row = kNoRow;
        if (want) {
          if (page_ok(p.c.map, want_page))
            row = row_at(p.c.map, want_page, h, want_r);
          else
            atomicExch(p.error_flag, PHEW_ERR_INVALID);
        }
        if (i < steps)
          ring.issue(i % S::STAGES, row);
        else
          copy_commit();
      };
      look_up(0);
#pragma unroll
      for (int i = 0; i < S::STAGES - 1; ++i) {
        start_copy(i);
        look_up(i + 1);
      }
      for (int i = 0; i < steps; ++i) {
        copy_wait<S::STAGES - 2>();
        __syncwarp();
        start_copy(i + S::STAGES - 1);
        look_up(i + S::STAGES);
        const int key0 = (t0 + i) * kTile + warp * kStageKeys;
        if (key0 >= ent.end) continue;
        const int st = i % S::STAGES;
        const uint32_t k_at = ring.base + st * S::STAGE, v_at = k_at + S::CODE_BYTES;

        // ---- scores of 2 x 16 keys: rows r8, r8 + 8 of the fragment hold keys key_of_slot(r8), + 8 ----
        float s[2][NT][4];
        const int my_key = key_of_slot(r8);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          float sk[2][NG], bk[2][NG];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            ring.scales(st, 0, 0, kb * 16 + half * 8 + my_key, sk[half]);
            ring.scales(st, 0, 1, kb * 16 + half * 8 + my_key, bk[half]);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) s[kb][nt][k] = 0.f;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            uint32_t wa[WPT], wb[WPT];
            const int r0 = kb * 16 + r8, word = g * (G / 8) + t4 * WPT;
            load_words<WPT>(k_at + r0 * (D / 2) + swizzle<D>(r0, word >> 2) * 16 + (word & 3) * 4, wa);
            load_words<WPT>(k_at + (r0 + 8) * (D / 2) + swizzle<D>(r0 + 8, word >> 2) * 16 + (word & 3) * 4, wb);
            float d[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int k = 0; k < 4; ++k) d[nt][k] = 0.f;
#pragma unroll
            for (int w = 0; w < WPT; ++w) {
              uint32_t a[4], b[4];
              if constexpr (HALF) {
                a[0] = pair_f16<0>(wa[w]); a[1] = pair_f16<1>(wa[w]); a[2] = pair_f16<2>(wa[w]); a[3] = pair_f16<3>(wa[w]);
                b[0] = pair_f16<0>(wb[w]); b[1] = pair_f16<1>(wb[w]); b[2] = pair_f16<2>(wb[w]); b[3] = pair_f16<3>(wb[w]);
              } else {
                a[0] = pair_bf16<0>(wa[w]); a[1] = pair_bf16<1>(wa[w]); a[2] = pair_bf16<2>(wa[w]); a[3] = pair_bf16<3>(wa[w]);
                b[0] = pair_bf16<0>(wb[w]); b[1] = pair_bf16<1>(wb[w]); b[2] = pair_bf16<2>(wb[w]); b[3] = pair_bf16<3>(wb[w]);
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int tq = TQ - 1; tq >= 0; --tq) {
                  const uint32_t* q = qf[nt][tq][g * WPT + w];
                  mma<HALF>(d[nt], a[0], b[0], a[1], b[1], q[0], q[1]);
                  mma<HALF>(d[nt], a[2], b[2], a[3], b[3], q[2], q[3]);
                }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const float z = fmaf(8.f, sk[half][g], bk[half][g]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                  float& y = s[kb][nt][2 * half + cc];
                  y = fmaf(sk[half][g], d[nt][2 * half + cc], fmaf(z, qs[nt][cc][g], y));
                }
            }
          }
        }
        // ---- running maximum: moved only when a score passes it by kGrow, so weights stay below 2^kGrow ----
        const bool edge = key0 + kStageKeys > lim_min;
        bool grow = false;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float& y = s[kb][nt][k];
              y *= p.scale_log2;
              if (edge && key0 + kb * 16 + (k >> 1) * 8 + my_key >= lim[nt][k & 1]) y = -INFINITY;
              grow = grow || y > m[nt][k & 1] + kGrow;
            }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              float top = fmaxf(fmaxf(s[0][nt][cc], s[0][nt][2 + cc]), fmaxf(s[1][nt][cc], s[1][nt][2 + cc]));
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
              const float m_new = fmaxf(m[nt][cc], top);
              const float alpha = exp2_fast(m[nt][cc] - m_new);
              m[nt][cc] = m_new;
              l[nt][cc] *= alpha;
#pragma unroll
              for (int g = 0; g < NG; ++g) bsum[nt][cc][g] *= alpha;
#pragma unroll
              for (int j = 0; j < D / 16; ++j) {
                acc[nt][j][cc] *= alpha;
                acc[nt][j][2 + cc] *= alpha;
              }
            }
        }
        // ---- weights, their sums, and the second product ----
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          uint32_t pb[NT][NG][TP][2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float sv[NG], bv[NG];
            ring.scales(st, 1, 0, kb * 16 + half * 8 + my_key, sv);
            ring.scales(st, 1, 1, kb * 16 + half * 8 + my_key, bv);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float w[2];
#pragma unroll
              for (int cc = 0; cc < 2; ++cc) {
                w[cc] = exp2_fast(s[kb][nt][2 * half + cc] - m[nt][cc]);
                l[nt][cc] += w[cc];
              }
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                float f[2];
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                  f[cc] = w[cc] * sv[g];
                  float z = w[cc] * fmaf(8.f, sv[g], bv[g]);
                  if (edge && w[cc] == 0.f) f[cc] = z = 0.f;  // a key this row does not see may hold anything
                  bsum[nt][cc][g] += z;
                }
#pragma unroll
                for (int tp = 0; tp < TP; ++tp) {
                  const uint32_t pk = pack_bf16(f[0], f[1]);
                  if (tp + 1 < TP) {
                    f[0] -= __uint_as_float(pk << 16);
                    f[1] -= __uint_as_float(pk & 0xffff0000u);
                  }
                  pb[nt][g][tp][half] = transpose8(pk);
                }
              }
            }
          }
          const int key = kb * 16 + t4;  // keys key, + 4, + 8, + 12
          if constexpr (G >= 64) {
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
              const int g = j * 64 / G, word = j * 8 + r8;
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                load_words<1>(v_at + (key + 4 * k) * (D / 2) + swizzle<D>(key + 4 * k, word >> 2) * 16 + (word & 3) * 4, &w[k]);
              const uint32_t x0 = __byte_perm(w[0], w[1], 0x5410), x1 = __byte_perm(w[0], w[1], 0x7632);
              const uint32_t y0 = __byte_perm(w[2], w[3], 0x5410), y1 = __byte_perm(w[2], w[3], 0x7632);
              auto tile = [&](int u, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int tp = TP - 1; tp >= 0; --tp)
                    mma<false>(acc[nt][j * 4 + u], a0, a1, a2, a3, pb[nt][g][tp][0], pb[nt][g][tp][1]);
              };
              tile(0, pair_bf16<0>(x0), pair_bf16<0>(x1), pair_bf16<0>(y0), pair_bf16<0>(y1));
              tile(1, pair_bf16<1>(x0), pair_bf16<1>(x1), pair_bf16<1>(y0), pair_bf16<1>(y1));
              tile(2, pair_bf16<2>(x0), pair_bf16<2>(x1), pair_bf16<2>(y0), pair_bf16<2>(y1));
              tile(3, pair_bf16<3>(x0), pair_bf16<3>(x1), pair_bf16<3>(y0), pair_bf16<3>(y1));
            }
          } else {
            // groups of four words: a fragment's eight rows are the two halves of each
            const uint32_t pick = r8 & 4 ? 0x7632 : 0x5410;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const int word = g * 4 + (r8 & 3);
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                load_words<1>(v_at + (key + 4 * k) * (D / 2) + swizzle<D>(key + 4 * k, word >> 2) * 16 + (word & 3) * 4, &w[k]);
              const uint32_t x0 = __byte_perm(w[0], w[1], pick), y0 = __byte_perm(w[2], w[3], pick);
              auto tile = [&](int u, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int tp = TP - 1; tp >= 0; --tp)
                    mma<false>(acc[nt][g * 2 + u], a0, a1, a2, a3, pb[nt][g][tp][0], pb[nt][g][tp][1]);
              };
              tile(0, pair_bf16<0>(x0), pair_bf16<2>(x0), pair_bf16<0>(y0), pair_bf16<2>(y0));
              tile(1, pair_bf16<1>(x0), pair_bf16<3>(x0), pair_bf16<1>(y0), pair_bf16<3>(y0));
            }
          }
        }
      }

      // ---- join the warps: each writes its rows, the block adds them up ----
      copy_wait<0>();
      __syncthreads();
      float* join = reinterpret_cast<float*>(smem);                    // [warp][ROWS][OROW]
      float* join_ml = join + kWarps * ROWS * S::OROW;                 // [warp][ROWS][2]
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          const int row = nt * 8 + 2 * t4 + cc;
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            l[nt][cc] += __shfl_xor_sync(0xffffffffu, l[nt][cc], o);
#pragma unroll
            for (int g = 0; g < NG; ++g) bsum[nt][cc][g] += __shfl_xor_sync(0xffffffffu, bsum[nt][cc][g], o);
          }
          float* dst = join + (warp * ROWS + row) * S::OROW;
          if constexpr (G >= 64) {
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
              const float z = bsum[nt][cc][j * 64 / G];
              float4* at = reinterpret_cast<float4*>(dst + (j * 8 + r8) * 8);
              at[0] = make_float4(acc[nt][j * 4][cc] + z, acc[nt][j * 4 + 1][cc] + z, acc[nt][j * 4 + 2][cc] + z, acc[nt][j * 4 + 3][cc] + z);
              at[1] = make_float4(acc[nt][j * 4][2 + cc] + z, acc[nt][j * 4 + 1][2 + cc] + z, acc[nt][j * 4 + 2][2 + cc] + z, acc[nt][j * 4 + 3][2 + cc] + z);
            }
          } else {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const float z = bsum[nt][cc][g];
              *reinterpret_cast<float4*>(dst + (g * 4 + (r8 & 3)) * 8 + (r8 & 4)) =
                  make_float4(acc[nt][g * 2][cc] + z, acc[nt][g * 2 + 1][cc] + z, acc[nt][g * 2][2 + cc] + z, acc[nt][g * 2 + 1][2 + cc] + z);
            }
          }
          if (r8 == 0) {
            join_ml[(warp * ROWS + row) * 2] = m[nt][cc];
            join_ml[(warp * ROWS + row) * 2 + 1] = l[nt][cc];
          }
        }
      __syncthreads();
      const bool whole = t0 == 0 && t1 == ent.tiles;
      const int slot = t0 > 0 ? 0 : 1;
      if (!whole) (slot == 0 ? left0 : left1) = static_cast<int64_t>(e) * kv_heads + h;
      for (int i = threadIdx.x; i < ROWS * (D / 4); i += kWarps * 32) {
        const int row = i / (D / 4), d4 = i % (D / 4);
        float mm = kFloor;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, join_ml[(w * ROWS + row) * 2]);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float ll = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float f = exp2_fast(join_ml[(w * ROWS + row) * 2] - mm);
          const float4 v = *reinterpret_cast<const float4*>(join + (w * ROWS + row) * S::OROW + d4 * 4);
          ll = fmaf(f, join_ml[(w * ROWS + row) * 2 + 1], ll);
          o.x = fmaf(f, v.x, o.x);
          o.y = fmaf(f, v.y, o.y);
          o.z = fmaf(f, v.z, o.z);
          o.w = fmaf(f, v.w, o.w);
        }
        if (whole) {
          const int r = ent.block * ROWS + row;
          const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(r)));
          if (tok < p.tokens) {
            const float inv = ll == 0.f || tok >= ent.count ? 0.f : 1.f / ll;
            T* dst = static_cast<T*>(p.o) +
                     ((static_cast<int64_t>(ent.b) * p.heads + h * p.per + (r - tok * p.per)) * p.tokens + tok) * D + d4 * 4;
            if (inv == 0.f) o = make_float4(0.f, 0.f, 0.f, 0.f);
            if constexpr (S::F32)
              *reinterpret_cast<float4*>(dst) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
            else
              *reinterpret_cast<uint2*>(dst) = make_uint2(pack_out<T>(o.x * inv, o.y * inv), pack_out<T>(o.z * inv, o.w * inv));
          }
        } else {
          const int64_t at = (2 * static_cast<int64_t>(blockIdx.x) + slot) * ROWS + row;
          *reinterpret_cast<float4*>(p.part + at * D + d4 * 4) = o;
          if (d4 == 0) {
            p.part_ml[at * 2] = mm;
            p.part_ml[at * 2 + 1] = ll;
          }
        }
      }
      __syncthreads();  // before the next segment's copies reuse the shared memory
    }
    base += static_cast<int64_t>(kv_heads) * ent.tiles;
    ++e;
  }
  if (threadIdx.x == 0) {
    p.meta[2 * blockIdx.x] = left0;
    p.meta[2 * blockIdx.x + 1] = left1;
  }
}

// Joins the partials of the segment that block blockIdx.x began and left:
// its partial 1, then the partials 0 of the blocks after it, in that order.
// One block of the grid per row.
template <typename S, typename T>
__global__ void __launch_bounds__(S::D) combine_kernel(const AttnParams p, int n) {
  constexpr int D = S::D, ROWS = S::ROWS;
  const int c = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // attn_kernel is done and its partials are visible
  const int64_t seg = p.meta[2 * c + 1];
  if (seg < 0) return;
  const int kv_heads = p.c.map.kv_heads;
  const int e = static_cast<int>(seg / kv_heads), h = static_cast<int>(seg - static_cast<int64_t>(e) * kv_heads);
  const int b = static_cast<int>(div_by(p.by_blocks, static_cast<uint32_t>(e)));
  const int r = (e - b * p.blocks) * ROWS + row;
  const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(r)));
  if (tok >= p.tokens) return;
  const bool live = !p.counts || tok < p.counts[b];
  __shared__ int s_last;
  // how many blocks after c go on with the segment
  int last = c;
  for (int c0 = c + 1;; c0 += D) {
    if (tid == 0) s_last = c0 + D;
    __syncthreads();
    if (c0 + tid >= n || p.meta[2 * (c0 + tid)] != seg) atomicMin(&s_last, c0 + tid);
    __syncthreads();
    last = s_last - 1;
    __syncthreads();
    if (last < c0 + D - 1) break;
  }
  auto at = [&](int k) { return (2 * static_cast<int64_t>(k) + (k == c ? 1 : 0)) * ROWS + row; };
  __shared__ float s_max[D / 32];
  float mm = kFloor;
  for (int k = c + tid; k <= last; k += D) mm = fmaxf(mm, p.part_ml[at(k) * 2]);
  mm = warp_max(mm);
  if ((tid & 31) == 0) s_max[tid >> 5] = mm;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < D / 32; ++w) mm = fmaxf(mm, s_max[w]);
  float o = 0.f, l = 0.f;
#pragma unroll 4
  for (int k = c; k <= last; ++k) {
    const float f = exp2_fast(p.part_ml[at(k) * 2] - mm);
    l = fmaf(f, p.part_ml[at(k) * 2 + 1], l);
    o = fmaf(f, p.part[at(k) * D + tid], o);
  }
  static_cast<T*>(p.o)[((static_cast<int64_t>(b) * p.heads + h * p.per + (r - tok * p.per)) * p.tokens + tok) * D + tid] =
      from_f32<T>(l == 0.f || !live ? 0.f : o / l);
}

// What a launch of attn_kernel needs from the host.
struct AttnPlan {
  int rows, grid;
  size_t bytes;
};

template <typename S> AttnPlan plan_of() {
  AttnPlan a;
  a.rows = S::ROWS;
  a.grid = sm_count_current() * S::CTAS;
  a.bytes = static_cast<size_t>(a.grid) * 2 * (static_cast<size_t>(S::ROWS) * (S::D + 2) * 4 + 8);
  return a;
}

// Dynamic shared memory of a kernel above 48 KB, allowed once per device (bit d: done on device d).
using SmemAllowed = std::atomic<uint64_t>;
template <typename K> int allow_smem(SmemAllowed& done, K* kernel, int bytes) {
  int dev = 0;
  PHEW_CHECK_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (bit && (done.load(std::memory_order_relaxed) & bit)) return PHEW_OK;
  PHEW_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  done.fetch_or(bit, std::memory_order_relaxed);
  return PHEW_OK;
}

template <typename S, typename T> int launch_attn(AttnParams p, void* workspace, cudaStream_t st) {
  const AttnPlan a = plan_of<S>();
  const int64_t rows = static_cast<int64_t>(p.tokens) * p.per;
  p.blocks = static_cast<int>((rows + S::ROWS - 1) / S::ROWS);
  p.by_blocks = fast_div(static_cast<uint32_t>(p.blocks));
  PHEW_REQUIRE(static_cast<int64_t>(p.batch) * p.blocks < (1ll << 31), "phew_kv_attention: too many query rows");
  p.meta = static_cast<int64_t*>(workspace);
  p.part = reinterpret_cast<float*>(p.meta + 2 * a.grid);
  p.part_ml = p.part + static_cast<size_t>(a.grid) * 2 * S::ROWS * S::D;
  static SmemAllowed allowed;
  if (int s = allow_smem(allowed, attn_kernel<S, T>, S::SMEM)) return s;
  attn_kernel<S, T><<<a.grid, kWarps * 32, S::SMEM, st>>>(p);
  if (int s = launch_status("kv attn_kernel")) return s;
  // a programmatic dependent: set up while attn_kernel runs
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.grid, S::ROWS);
  cfg.blockDim = dim3(S::D);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PHEW_CHECK_CUDA(cudaLaunchKernelEx(&cfg, combine_kernel<S, T>, p, static_cast<int>(a.grid)));
  return launch_status("kv combine_kernel");
}

// Row tiles of eight to a block: two for more than eight query rows, where registers allow it (16-bit
// types with heads up to 128; wider heads and the three terms of f32 would spill the second tile).
template <typename T> int row_tiles(int head_dim, int64_t rows) {
  return sizeof(T) == 2 && head_dim <= 128 && rows > 8 ? 2 : 1;
}

// Calls f with the Shape for a head dimension, a group size and a number of query rows.
template <typename T, typename F> auto with_shape(int head_dim, int group, int64_t rows, F f) {
  const int nt = row_tiles<T>(head_dim, rows);
#define PHEW_KV_SHAPE(D, G)                                                            \
  if (head_dim == D && group == G) {                                                   \
    if constexpr (D <= 128 && sizeof(T) == 2)                                          \
      if (nt == 2) return f(Shape<T, D, G, 2>());                                      \
    return f(Shape<T, D, G, 1>());                                                     \
  }
  PHEW_KV_SHAPE(64, 32)
  PHEW_KV_SHAPE(64, 64)
  PHEW_KV_SHAPE(128, 32)
  PHEW_KV_SHAPE(128, 64)
  PHEW_KV_SHAPE(128, 128)
  PHEW_KV_SHAPE(256, 32)
  PHEW_KV_SHAPE(256, 64)
#undef PHEW_KV_SHAPE
  return f(Shape<T, 256, 128, 1>());
}

// Scratch bytes and launch per type; instantiated in a translation unit each, which compile side by side.
template <typename T> size_t attn_bytes(int head_dim, int group, int64_t rows) {
  return with_shape<T>(head_dim, group, rows, [](auto s) { return plan_of<decltype(s)>().bytes; });
}
template <typename T> int run_attn(const AttnParams& p, void* workspace, cudaStream_t st) {
  return with_shape<T>(p.c.head_dim, p.c.group, static_cast<int64_t>(p.tokens) * p.per,
                       [&](auto s) { return launch_attn<decltype(s), T>(p, workspace, st); });
}
#ifndef PHEW_KV_ATTN_TYPE
extern template size_t attn_bytes<float>(int, int, int64_t);
extern template size_t attn_bytes<f16>(int, int, int64_t);
extern template size_t attn_bytes<bf16>(int, int, int64_t);
extern template int run_attn<float>(const AttnParams&, void*, cudaStream_t);
extern template int run_attn<f16>(const AttnParams&, void*, cudaStream_t);
extern template int run_attn<bf16>(const AttnParams&, void*, cudaStream_t);
#endif

}  // namespace kv
}  // namespace phew
