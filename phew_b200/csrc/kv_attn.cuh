// Attention of few query rows over a 4-bit cache (decode, drafted tokens).
//
//   s_rj = scale * sum_g sk[j,g] (q_r . n_j)_g + zk[j,g] sum(q_r)_g
//   o_r  = sum_j p_rj (sum_g sv[j,g] n_j + zv[j,g]) / sum_j p_rj
//
// with n the codes as they lie in the cache: scales and biases never touch a
// code, they act on the small score tile (keys) and on the softmax weights
// (values).  A cache head's `per` query heads and the query tokens are the
// rows r = token * per + head, eight or sixteen to a block, so keys and values
// are read once for all of them.
//
// Bound by HBM (a packed row of 128 with groups of 64 is 72 bytes): at 6.5
// TB/s an SM gets 41 codes a clock, which leaves 1.6 integer instructions (two
// warp instructions a clock, measured) and 3 of any kind for each 32.  So
//  * both products run on mma.sync m16n8k16 with keys (scores) and head
//    dimension (output) along m and the few query rows along n: no padding of
//    eight rows to sixteen.  (tcgen05 would need the codes as 16-bit tiles in
//    shared memory: four times the bytes, written and read once more than the
//    128 bytes a clock an SM has.)
//  * codes need no conversion: sixteen bits that hold n in 0 .. 15 are the f16
//    subnormal n 2^-24, and n one digit up is 16 n 2^-24, so one logic operation
//    makes a pair of operands, `w & 0x000f000f` or `w & 0x00f000f0`, and one
//    shift by eight brings the word's other half under the same masks: 5
//    instructions for eight codes.  The 16 goes into the query (keys) or out of
//    the sum (values), exactly.  (f16 values, and f32's keys and values, take
//    n - 8 as normal numbers, one more instruction a pair: Shape says why.
//    e4m3, which holds a nibble in a byte as it
//    is, was tried: mma.sync on that type is expanded into conversions here,
//    11 instructions each.)
//  * queries and weights times value scales are f16 after a power of two.  A
//    row's largest query element goes to [2^14, 2^15): what falls below f16's
//    range is under 2^-38 of it.  Weights times scales have a factor for each
//    row and group, set by the largest of them that the row has met, so that
//    neither another group's values nor a key that the row does not attend
//    to cost it bits: f16's smallest step is at most 2^-22 of that largest
//    one.  The factors lie in shared memory and are looked at again only when a
//    row's maximum moves, or a scale itself would pass f16's range under one of
//    them (one comparison a tile; a segment's first tile always: 0.5 us of a
//    short call, 1.5 with two row tiles).  f32 queries and weights are two f16
//    terms (22 bits), and its sums leave the tensor core, which cuts what it
//    adds off, every 16 keys;
//  * a word's eight codes stay with the thread that loads it: the order of
//    the head dimension inside a product is free, so queries are arranged to
//    match and nothing is shuffled; weights move from the score fragment
//    (key-major) to the operand of the second product by movmatrix;
//  * every warp walks keys of its own with its own running maximum and sum
//    and its own ring of cp.async stages: no block barrier anywhere, so the
//    latencies at a segment's begin and end are hidden by the SM's other warps.
//
// Work split: the (sequence, row block, cache head) segments of all
// sequences, cut into tiles of 32 keys, are one line of W units (a segment's
// begin counts as kBegin tiles); warp c of n takes units [cW/n, (c+1)W/n), so
// any mix of lengths loads the SMs evenly and no host ever needs the lengths.
// A segment that lies in one warp is finished there; a cut one leaves partial
// sums (maximum, sum, output) that the combine kernel joins in a fixed order.
//
// Measured: 64 sequences of up to 8192 keys, 32 heads of 128 over 8, bf16:
// 82 us, 3.8 TB/s of the bytes that must be read (0.57 of a copy).  Three warps
// to a scheduler (168 registers) issue every other cycle: 663 instructions to
// a tile, waits on one another's results between them.  Four (128 registers)
// spill, or read the queries from shared memory, for the same time.
#pragma once

#include <atomic>
#include <type_traits>

#include "kv_cache.cuh"

namespace phew {
namespace kv {

constexpr int kWarps = 4;       // of a block; they share nothing
constexpr int kTile = 32;       // keys of a tile: one warp's stage
// Tiles that the latencies of a segment's begin are worth (1, 2, 4: 41.6, 37.5, 39.9 us for 256 x 8 segments of 300
// keys; no difference for 128 of 8192)
constexpr int kBegin = 2;
constexpr uint32_t kEven = 0x000f000fu, kOdd = 0x00f000f0u;  // codes of a word as pairs of f16
constexpr float kGrow = 8.0f;                   // log2 units that a row's scores may grow by before its sums are scaled
constexpr int kCentreTiles = 16;                // tiles of bare codes in one sum
constexpr float kFloor = -1.0e38f;              // running maximum before the first key
constexpr float kF16Most = 32768.f;             // what weights times scales are held below
constexpr float kNoFactor = 0x1p68f;            // a row's and group's factor before its first weight

struct AttnParams {
  Cache c;
  const void* q;
  int64_t st[3];  // q's token, head and batch strides (elements)
  void* o;        // [batch][heads][tokens][D]
  const int32_t* lengths;
  const int32_t* counts;  // null: all `tokens`
  int batch, heads, tokens, per;  // per: query heads to a cache head
  int blocks;                     // row blocks of a sequence's tokens * per rows
  int step_col, step_row;         // kTile tokens in pages and rows
  uint32_t page_rows;             // kv_heads * page_size
  bool eights;                    // pages hold whole eights of rows
  FastDiv by_per, by_blocks;
  float scale_log2;
  bool causal;
  // scratch: of every warp two partials, 0 of a segment that an earlier warp began and 1 of one that it leaves
  float* part;     // [warp][2][rows][D] outputs
  float* part_ml;  // [warp][2][rows][2] maximum and sum
  int2* span;      // [segment] first and last warp; equal where one warp finished it
  int* error_flag;
};

// One sequence's row block.
struct Entry {
  int b, block;
  int length, count;
  int end;    // keys [0, end) that any of its rows sees
  int tiles;  // at least one, so that some warp writes the rows of an empty one
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
  // f16 terms of a query and of a weight: one is exact for 16-bit queries and rounds a weight by 2^-12 of it
  static constexpr int TERMS = F32 ? 2 : 1;
  // n - 8 instead of n in the second product: exact, and the rounded weights are then multiplied by half as
  // much.  f16 results see that (3.0e-4 of their norm instead of 3.8e-4, attend_long 45 -> 48 us), bf16's do
  // not.  f32 takes keys that way too: the tensor core lines a subnormal up as 2^-14 when it adds, so products
  // of the bare digits lose their last bits (5e-6 of an output's norm instead of 4e-7).
  static constexpr bool V_CENTRED = !std::is_same<T, bf16>::value;
  static constexpr int SB = NG * static_cast<int>(sizeof(T));   // bytes of a key's scales
  static constexpr int SROW = SB < 4 ? 4 : SB;
  static constexpr int CODE_BYTES = kTile * D / 2;         // one side's codes of a stage
  static constexpr int STAGE = 2 * CODE_BYTES + 4 * kTile * SROW;
  static constexpr int AFFINE = kTile * NG * 8;            // scales and biases of a stage's side as float pairs
  static constexpr int FACTORS = ((ROWS + 1) * NG * 4 + 127) / 128 * 128;  // of rows and groups; their largest to a group
  // blocks to an SM (their registers: 65536 / (128 CTAS) to a thread), and as many stages as their share of
  // the SM's 228 KB holds beside the 1 KB that each block costs
  static constexpr int CTAS = D == 256 ? 2 : D == 128 ? (F32 || NT == 2 ? 2 : 3) : (F32 || NT == 2 ? 3 : 4);
  static constexpr int SHARE = (228 / CTAS - 1) * 1024 / kWarps;
  static constexpr int STAGES = (SHARE - AFFINE - FACTORS) / STAGE < 4 ? (SHARE - AFFINE - FACTORS) / STAGE : 4;
  static_assert(STAGES >= 2, "a ring needs two stages");
  static constexpr int RING = STAGE * STAGES + AFFINE + FACTORS;  // per warp
  static constexpr int SMEM = RING * kWarps;
};

// ---- small pieces ---------------------------------------------------------

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// N bytes of which `valid` are read, the rest zero
template <int N> __device__ __forceinline__ void copy_async_upto(uint32_t dst, const void* src, int valid) {
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

// 1 / x of a power of two between 2^-126 and 2^126.
__device__ __forceinline__ float inverse_pow2(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T> __device__ __forceinline__ uint32_t pack_out(float lo, float hi) {
  return static_cast<uint32_t>(from_f32<T>(lo).bits) | static_cast<uint32_t>(from_f32<T>(hi).bits) << 16;
}

// c += a b and c = a b, f16 with fp32 sums.
__device__ __forceinline__ void mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// A word's codes under a mask as pairs of f16, digits of a subnormal: n 2^-24 (odd codes 16 n 2^-24).  CENTRED:
// n - 8 (16 (n - 8)), by way of 1024 + n.
template <bool CENTRED> __device__ __forceinline__ uint32_t even_codes(uint32_t w) {
  if constexpr (!CENTRED) return w & kEven;
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"((w & kEven) | 0x64006400u), "r"(0x64086408u));
  return d;
}
template <bool CENTRED> __device__ __forceinline__ uint32_t odd_codes(uint32_t w) {
  if constexpr (!CENTRED) return w & kOdd;
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"((w & kOdd) | 0x64006400u), "r"(0x64806480u));
  return d;
}

// Two values rounded to f16 (lo in the low half); `rest`: what is left of them.
template <bool REST> __device__ __forceinline__ uint32_t take_f16(float& lo, float& hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  if constexpr (REST) {
    lo -= to_f32(f16{static_cast<uint16_t>(d)});
    hi -= to_f32(f16{static_cast<uint16_t>(d >> 16)});
  }
  return d;
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
  static constexpr int CH = S::D / 32;  // 16-byte chunks of a row
  static constexpr int RP = 32 / CH;    // rows that one copy of the warp covers
  const Cache& c;
  uint32_t base;    // shared address of this warp's stages, then of its float pairs
  int lane;
  uint32_t odd;     // bit s: this lane's row of stage s is odd (two-byte scales: which half of the loaded word)

  __device__ __forceinline__ uint32_t pairs() const { return base + S::STAGE * S::STAGES; }

  // Starts the copy of the 32 rows that the lanes hold into stage `s`, zeros for the scales and biases of a lane
  // that has no `page`; EIGHTS: rows of eight keys lie side by side.
  template <bool EIGHTS> __device__ __forceinline__ void issue(int s, uint32_t row, bool page) {
    const uint32_t at = base + s * S::STAGE;
    const int ch = lane % CH, sub = lane / CH;
    constexpr uint32_t ROW = S::D / 2;
    if constexpr (EIGHTS && RP % 8 == 0) {
      // one row number to RP / 8 eights: the rest of a lane's row is its place among the eight
      const uint32_t k_off = key_of_slot(sub & 7) * ROW + ch * 16, v_off = (sub & 7) * ROW + ch * 16;
      const char* k = reinterpret_cast<const char*>(c.codes[0]) + k_off;
      const char* v = reinterpret_cast<const char*>(c.codes[1]) + v_off;
      const uint32_t dst = at + sub * ROW + swizzle<S::D>(sub, ch) * 16;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const uint32_t src = __shfl_sync(0xffffffffu, row, i * RP + (RP == 8 ? 0 : sub & ~7));
        copy_async16(dst + i * RP * ROW, k + static_cast<uint64_t>(src) * ROW);
        copy_async16(dst + S::CODE_BYTES + i * RP * ROW, v + static_cast<uint64_t>(src) * ROW);
      }
    } else {
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const char* codes = reinterpret_cast<const char*>(c.codes[side]) + ch * 16;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int r = i * RP + sub;
          const uint32_t src = __shfl_sync(0xffffffffu, row, side == 0 ? key_of_slot(r) : r);
          copy_async16(at + side * S::CODE_BYTES + r * ROW + swizzle<S::D>(r, ch) * 16,
                       codes + static_cast<uint64_t>(src) * ROW);
        }
      }
    }
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      const char* arr = static_cast<const char*>((a & 1) ? c.biases[a >> 1] : c.scales[a >> 1]);
      const uint32_t dst = at + 2 * S::CODE_BYTES + (a * kTile + lane) * S::SROW;
      if constexpr (S::SB == 2) {
        // the aligned word around the two bytes; the array's last row alone has no partner behind it
        const uint32_t rows = static_cast<uint32_t>(c.map.pages) * static_cast<uint32_t>(c.map.kv_heads) *
                              static_cast<uint32_t>(c.map.page_size);
        copy_async_upto<4>(dst, arr + static_cast<uint64_t>(row & ~1u) * 2, !page ? 0 : (row | 1u) < rows ? 4 : 2);
      } else {
        constexpr int N = S::SB < 16 ? S::SB : 16;
#pragma unroll
        for (int i = 0; i < S::SB; i += N)
          copy_async_upto<N>(dst + i, arr + static_cast<uint64_t>(row) * S::SB + i, page ? N : 0);
      }
    }
    if constexpr (S::SB == 2) odd = (odd & ~(1u << s)) | ((row & 1u) << s);
    copy_commit();
  }

  // Scales and biases of a side of stage `s`, a key to a lane; nothing for a lane without a key.
  __device__ __forceinline__ void load(int s, int side, bool have, float* sc, float* bi) const {
    const uint32_t at = base + s * S::STAGE + 2 * S::CODE_BYTES + (side * 2 * kTile + lane) * S::SROW;
    read(at, s, sc);
    read(at + kTile * S::SROW, s, bi);
#pragma unroll
    for (int g = 0; g < S::NG; ++g)
      if (!have) sc[g] = bi[g] = 0.f;
  }
  // ... for the whole warp to read, as pairs of floats.
  __device__ __forceinline__ void share(const float* sc, const float* bi) const {
    const uint32_t dst = pairs() + lane * S::NG * 8;
    if constexpr (S::NG == 1) {
      asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(dst), "f"(sc[0]), "f"(bi[0]) : "memory");
    } else {
#pragma unroll
      for (int g = 0; g < S::NG; g += 2)
        asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst + g * 8), "f"(sc[g]), "f"(bi[g]),
                     "f"(sc[g + 1]), "f"(bi[g + 1])
                     : "memory");
    }
  }
  __device__ __forceinline__ void read(uint32_t at, int s, float* out) const {
    if constexpr (S::SB == 2) {
      uint32_t w;
      load_words<1>(at, &w);
      out[0] = to_f32(T{static_cast<uint16_t>((odd >> s) & 1 ? w >> 16 : w)});
    } else {
      uint32_t w[S::SB / 4];
      constexpr int N = S::SB < 16 ? S::SB / 4 : 4;
#pragma unroll
      for (int i = 0; i < S::SB / 4; i += N) load_words<N>(at + i * 4, w + i);
#pragma unroll
      for (int g = 0; g < S::NG; ++g) {
        if constexpr (S::F32)
          out[g] = __uint_as_float(w[g]);
        else
          out[g] = to_f32(T{static_cast<uint16_t>(g & 1 ? w[g / 2] >> 16 : w[g / 2])});
      }
    }
  }
  // Factors of rows 2 t4 and 2 t4 + 1 of row tile nt, [group][row].
  __device__ __forceinline__ uint32_t factors(int nt) const {
    return pairs() + S::AFFINE + (nt * 4 + (lane & 3)) * S::NG * 8;
  }
  __device__ __forceinline__ void load_factors(int nt, float (*up)[2]) const {
    const uint32_t at = factors(nt);
    if constexpr (S::NG == 1) {
      asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(up[0][0]), "=f"(up[0][1]) : "r"(at));
    } else {
#pragma unroll
      for (int g = 0; g < S::NG; g += 2)
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(up[g][0]), "=f"(up[g][1]), "=f"(up[g + 1][0]), "=f"(up[g + 1][1])
                     : "r"(at + g * 8));
    }
  }
  // ... called by every lane, which hold the same for the same rows.
  __device__ __forceinline__ void store_factors(int nt, const float (*up)[2]) const {
    if (lane < 4) {
#pragma unroll
      for (int g = 0; g < S::NG; ++g)
        asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(factors(nt) + g * 8), "f"(up[g][0]), "f"(up[g][1]) : "memory");
    }
  }
  // The largest of all rows' factors, to a group.
  __device__ __forceinline__ uint32_t most() const { return pairs() + S::AFFINE + S::ROWS * S::NG * 4; }
  __device__ __forceinline__ void load_most(float* v) const {
    uint32_t w[S::NG];
    constexpr int N = S::NG < 4 ? S::NG : 4;
#pragma unroll
    for (int g = 0; g < S::NG; g += N) load_words<N>(most() + g * 4, w + g);
#pragma unroll
    for (int g = 0; g < S::NG; ++g) v[g] = __uint_as_float(w[g]);
  }
  __device__ __forceinline__ void store_most(const float* v) const {
    if (lane == 0) {
#pragma unroll
      for (int g = 0; g < S::NG; ++g) asm volatile("st.shared.f32 [%0], %1;" ::"r"(most() + g * 4), "f"(v[g]) : "memory");
    }
  }
  // Scales and biases of key `key` on the side shared last.
  __device__ __forceinline__ void affine(int key, float* sc, float* bi) const {
    const uint32_t at = pairs() + key * S::NG * 8;
    if constexpr (S::NG == 1) {
      asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(sc[0]), "=f"(bi[0]) : "r"(at));
    } else {
#pragma unroll
      for (int g = 0; g < S::NG; g += 2)
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(sc[g]), "=f"(bi[g]), "=f"(sc[g + 1]), "=f"(bi[g + 1])
                     : "r"(at + g * 8));
    }
  }
};

// ---- the kernel -----------------------------------------------------------------

template <typename S, typename T>
__global__ void __launch_bounds__(kWarps * 32, S::CTAS) attn_kernel(const AttnParams p) {
  constexpr int D = S::D, G = S::G, NT = S::NT, NG = S::NG, ROWS = S::ROWS, TERMS = S::TERMS;
  constexpr bool KC = S::F32, VC = S::V_CENTRED;  // key and value codes less 8 in the products
  constexpr int WPT = G / 32;   // words of a group that one thread multiplies with the queries
  constexpr int WT = D / 32;    // of a row
  extern __shared__ __align__(128) uint8_t smem[];
  // (shared memory of its own would cost a block its place on the SM: these come before the ring's use of it)
  uint64_t* s_red = reinterpret_cast<uint64_t*>(smem);
  uint64_t* s_prefix = s_red + kWarps;
  uint64_t* s_target = s_prefix + kWarps;
  int* s_entry = reinterpret_cast<int*>(s_target + kWarps);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r8 = lane >> 2, t4 = lane & 3;
  const int kv_heads = p.c.map.kv_heads;

  // ---- this warp's share of the line: of W units the first W mod n warps take one more ----
  asm volatile("griddepcontrol.launch_dependents;");  // the combine kernel may be set up from here on; it waits for this one
  const int entries = p.batch * p.blocks;
  uint32_t own = 0;  // units of this thread's first entry for one head
  uint64_t sum = 0;
  for (int e = threadIdx.x; e < entries; e += kWarps * 32) {
    const Entry t = entry_at(p, e, ROWS);
    const uint32_t units = t.tiles + kBegin;
    if (e == static_cast<int>(threadIdx.x)) own = units;
    sum += units;
    if (blockIdx.x == 0 && t.block == 0 && __ldg(p.lengths + t.b) != t.length) atomicExch(p.error_flag, PHEW_ERR_INVALID);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_red[warp] = sum;
  __syncthreads();
  sum = s_red[0] + s_red[1] + s_red[2] + s_red[3];
  const uint64_t total = sum * kv_heads;
  const uint32_t all_warps = gridDim.x * kWarps;
  const uint32_t n = total < all_warps ? static_cast<uint32_t>(total) : all_warps;
  if (blockIdx.x >= n) return;  // no warp of the block has work
  // neighbours on the line run on different SMs, and a short line on as many as it can
  const uint32_t self = warp * gridDim.x + blockIdx.x;
  const bool narrow = total >> 32 == 0;
  const uint64_t each = narrow ? static_cast<uint32_t>(total) / n : total / n;
  const uint32_t more = static_cast<uint32_t>(total - each * n);
  uint64_t x = self * each + min(self, more);
  const uint64_t x_end = x + each + (self < more);
  // the entry that the first unit lies in: the first whose units, with those before it, pass x / kv_heads
  if (lane == 0)
    s_target[warp] = self < n ? (narrow ? static_cast<uint32_t>(x) / static_cast<uint32_t>(kv_heads) : x / kv_heads) : ~0ull;
  uint64_t run = 0;
  for (int e0 = 0; e0 < entries; e0 += kWarps * 32) {
    const int i = e0 + static_cast<int>(threadIdx.x);
    if (e0 > 0) own = i < entries ? entry_at(p, i, ROWS).tiles + kBegin : 0;
    uint64_t inc = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    __syncthreads();
    if (lane == 31) s_red[warp] = inc;
    __syncthreads();
    for (int w = 0; w < warp; ++w) inc += s_red[w];
    inc += run;
    uint64_t most = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const uint64_t want = s_target[w];
      if (inc > want && inc - own <= want) {
        s_entry[w] = i;
        s_prefix[w] = inc - own;
      }
      if (want != ~0ull) most = want;  // (targets grow with the warp)
    }
    run += s_red[0] + s_red[1] + s_red[2] + s_red[3];
    if (run > most) break;
  }
  __syncthreads();
  int e = s_entry[warp];
  uint64_t base = s_prefix[warp];
  __syncthreads();  // (the ring takes the shared memory over; the last barrier)
  if (self >= n) return;
  base *= kv_heads;

  Ring<S, T> ring{p.c, smem_addr(smem) + warp * S::RING, lane, 0u};

  while (x < x_end) {
    const Entry ent = entry_at(p, e, ROWS);
    const uint32_t units = ent.tiles + kBegin;  // (units of a sequence's heads together fit 32 bits)
    for (; x < x_end && x < base + static_cast<uint64_t>(kv_heads) * units;) {
      const int h = static_cast<int>(static_cast<uint32_t>(x - base) / units);
      const uint64_t seg0 = base + static_cast<uint64_t>(h) * units;
      const int t0 = max(static_cast<int>(x - seg0) - kBegin, 0);
      x = min(x_end, seg0 + units);
      const int t1 = static_cast<int>(x - seg0) - kBegin;
      if (t1 <= t0) continue;  // units of the begin alone

      // ---- the ring: page numbers one stage ahead of the copies, copies STAGES - 1 ahead of the products.
      // A lane without a key copies row 0 of the cache: whatever it holds is masked.  So does one whose page is none
      // of the cache's, with zeros for scales and biases: its key and value count as zeros, as in the tcgen05
      // kernel. ----
      struct Look {
        int page;  // -1: no key
        uint32_t row;
      };
      int key = t0 * kTile + lane;  // of the next look-up
      int col = static_cast<int>(div_by(p.c.map.by_page, static_cast<uint32_t>(key)));
      int in_page = key - col * p.c.map.page_size;
      const int32_t* pages = p.c.map.table ? p.c.map.table + ent.b * p.c.map.table_stride : nullptr;
      const uint32_t head_row = static_cast<uint32_t>(h) * static_cast<uint32_t>(p.c.map.page_size);
      const int key_end = min(ent.end, t1 * kTile);
      auto look_up = [&]() {
        Look k{0, 0};
        const bool have = key < key_end;
        if (have) k.page = pages ? __ldg(pages + col) : ent.b;
        k.row = have ? head_row + static_cast<uint32_t>(in_page) : kNoRow;
        key += kTile;
        in_page += p.step_row;
        col += p.step_col;
        if (in_page >= p.c.map.page_size) {
          in_page -= p.c.map.page_size;
          ++col;
        }
        return k;
      };
      int left = t1 - t0, st_in = 0, st_out = 0;  // copies still to start, and the stages that come next
      auto start_copy = [&](const Look& k) {
        if (left > 0) {
          uint32_t row = 0;
          bool page = true;
          if (k.row != kNoRow) {
            page = page_ok(p.c.map, k.page);
            if (page)
              row = static_cast<uint32_t>(k.page) * p.page_rows + k.row;
            else
              atomicExch(p.error_flag, PHEW_ERR_INVALID);
          }
          if (p.eights)
            ring.template issue<true>(st_in, row, page);
          else
            ring.template issue<false>(st_in, row, page);
          st_in = st_in + 1 == S::STAGES ? 0 : st_in + 1;
          --left;
        } else {
          copy_commit();
        }
      };
      Look first[S::STAGES - 1];
#pragma unroll
      for (int i = 0; i < S::STAGES - 1; ++i) first[i] = look_up();
      Look next = look_up();

      // ---- queries: their loads travel beside the look-ups' ----
      constexpr int QV = static_cast<int>(sizeof(T)) / 2;  // 16-byte loads of eight values
      uint4 raw[NT][WT][QV];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int r = ent.block * ROWS + nt * 8 + r8;
        const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(r)));
        const T* q = static_cast<const T*>(p.q) + ent.b * p.st[2] + (h * p.per + (r - tok * p.per)) * p.st[1] + tok * p.st[0];
#pragma unroll
        for (int w = 0; w < WT; ++w)
#pragma unroll
          for (int k = 0; k < QV; ++k)
            raw[nt][w][k] = tok < ent.count
                                ? __ldg(reinterpret_cast<const uint4*>(q + (w / WPT) * G + (t4 * WPT + w % WPT) * 8) + k)
                                : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < S::STAGES - 1; ++i) start_copy(first[i]);

      // ---- queries as the n operand, their group sums, and how far each row sees ----
      uint32_t qf[NT][TERMS][WT][4];
      float qs[NT][2][NG], unit[NT][2];  // a score is unit times what the product gives
      int lim[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float v[WT][8], top = 0.f;
#pragma unroll
        for (int w = 0; w < WT; ++w)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            v[w][k] = to_f32(reinterpret_cast<const T*>(raw[nt][w])[k]);
            top = fmaxf(top, fabsf(v[w][k]));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the row's largest magnitude to [2^14, 2^15)
        const uint32_t e = max(__float_as_uint(top) >> 23, 20u);
        const float up = __uint_as_float((268u - e) << 23);
        const float row_unit = p.scale_log2 * 0x1p24f * __uint_as_float((e - 14u) << 23);  // 2^24 scale / up
        float sum[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          sum[g] = 0.f;
#pragma unroll
          for (int i = 0; i < WPT; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k) sum[g] += v[g * WPT + i][k] *= up;  // (unscaled, a sum may pass fp32's range)
          sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
          sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
        }
#pragma unroll
        for (int w = 0; w < WT; ++w) {
#pragma unroll
          for (int k = 1; k < 8; k += 2) v[w][k] *= 0.0625f;  // odd codes count sixteenfold
#pragma unroll
          for (int t = 0; t < TERMS; ++t)
#pragma unroll
            for (int k = 0; k < 4; ++k) qf[nt][t][w][k] = take_f16<TERMS == 2>(v[w][k], v[w][k + 4]);
        }
        // rows of the score fragment's columns: 2 t4 and 2 t4 + 1
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          const int from = (2 * t4 + cc) * 4;
#pragma unroll
          for (int g = 0; g < NG; ++g) qs[nt][cc][g] = __shfl_sync(0xffffffffu, sum[g], from);
          unit[nt][cc] = __shfl_sync(0xffffffffu, row_unit, from);
          const int rr = ent.block * ROWS + nt * 8 + 2 * t4 + cc;
          const int tok_cc = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(rr)));
          // rows without a query run along unmasked (never stored)
          lim[nt][cc] = tok_cc < ent.count ? seen_end(ent.length, ent.count, tok_cc, p.causal) : 0x7fffffff;
        }
      }
      int lim_min = lim[0][0];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) lim_min = min(lim_min, min(lim[nt][0], lim[nt][1]));
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, o));

      float acc[NT][D / 16][4];
      // a row's weights are 2^(score - m), m kGrow above its largest score when it last moved; it moves when a
      // score passes it by `pass`, which is 0 once the row has seen a key and below any score before
      float m[NT][2], pass[NT][2], l[NT][2], bsum[NT][2][NG];
      float wsum[NT][2][NG];  // of bf16: the weights times scales behind `acc`
      __syncwarp();           // (the last segment's factors have been read)
      {
        float most[NG];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          // a row that sees none of these keys has no weights to fit
          float up[NG][2];
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) up[g][cc] = lim[nt][cc] > t0 * kTile ? kNoFactor : 1.f;
          ring.store_factors(nt, up);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) most[g] = kNoFactor;
        ring.store_most(most);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[nt][i][k] = 0.f;
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          m[nt][cc] = 0.f;
          pass[nt][cc] = kFloor;
          l[nt][cc] = 0.f;
#pragma unroll
          for (int g = 0; g < NG; ++g) bsum[nt][cc][g] = wsum[nt][cc][g] = 0.f;
        }
      }

      const int my_key = key_of_slot(r8);

      // Factors of the rows and groups whose weights times scales pass f16's range in this tile, are their first, or
      // are taken against a new m (a row's moved by `moved`, 0 where it stayed): what was large before may be nothing
      // now, and a factor may grow again, by 2^60 more than the sums have shrunk at most (of 2^31 keys they are below
      // 2^58 before).  The tile's largest scale goes to [2^12, 2^13), unless that left less than 2^-2 of the row's
      // largest weight times scale: then the scales that pass the range have next to no weight.
      auto fit = [&](float (*s)[NT][4], const float* sv, const float (*moved)[2]) {
        uint32_t top[NG];
        float most[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const uint32_t bits = __float_as_uint(fabsf(sv[g]));  // (magnitudes order as their bits)
          top[g] = __reduce_max_sync(0xffffffffu, bits < 0x7f800000u ? bits : 0u);
          most[g] = 0.f;
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float part[NG][2], up[NG][2];  // the row's largest weight times scale
#pragma unroll
          for (int g = 0; g < NG; ++g) part[g][0] = part[g][1] = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float a[NG], z[NG];
            ring.affine(k * 8 + my_key, a, z);
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              const float w = exp2_fast(s[k >> 1][nt][2 * (k & 1) + cc]);
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                const float f = w * fabsf(a[g]);
                if (f < INFINITY) part[g][cc] = fmaxf(part[g][cc], f);
              }
            }
          }
          ring.load_factors(nt, up);
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              float f = part[g][cc];
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) f = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, o));
              float by = 1.f, rest = 1.f;  // two halves of the step: it may be 2^183
              const bool again = up[g][cc] == kNoFactor || moved[nt][cc] != 0.f;
              if (f * up[g][cc] > kF16Most || (again && f > 0.f)) {
                const int e = max(266 - static_cast<int>(top[g] >> 23),
                                  252 - static_cast<int>(__float_as_uint(f) >> 23));
                const int from = static_cast<int>(__float_as_uint(up[g][cc]) >> 23);
                const int most_step = 60 + static_cast<int>(fminf(fmaxf(moved[nt][cc], 0.f), 200.f));
                const int step = min(min(e, 195) - from, most_step);  // (195: kNoFactor)
                by = __int_as_float(((step >> 1) + 127) << 23);
                rest = __int_as_float((step - (step >> 1) + 127) << 23);
                up[g][cc] = __int_as_float((from + step) << 23);
              }
              most[g] = fmaxf(most[g], up[g][cc]);
              wsum[nt][cc][g] = wsum[nt][cc][g] * by * rest;
#pragma unroll
              for (int i = g * G / 16; i < (g + 1) * G / 16; ++i) {
                acc[nt][i][cc] = acc[nt][i][cc] * by * rest;
                acc[nt][i][2 + cc] = acc[nt][i][2 + cc] * by * rest;
              }
            }
          __syncwarp();
          ring.store_factors(nt, up);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          most[g] = fmaxf(most[g], __shfl_xor_sync(0xffffffffu, most[g], 1));
          most[g] = fmaxf(most[g], __shfl_xor_sync(0xffffffffu, most[g], 2));
        }
        ring.store_most(most);
        __syncwarp();
      };

      // One stage of 32 keys; EDGE: some row does not see all of them.
      auto stage = [&](int st, int key0, auto edge_c) {
        constexpr bool EDGE = decltype(edge_c)::value;
        const uint32_t k_at = ring.base + st * S::STAGE, v_at = k_at + S::CODE_BYTES;
        // ---- scores of 2 x 16 keys: rows r8, r8 + 8 of the fragment hold keys key_of_slot(r8), + 8 ----
        float s[2][NT][4];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          float sk[2][NG], zk[2][NG];
          ring.affine(kb * 16 + my_key, sk[0], zk[0]);
          ring.affine(kb * 16 + 8 + my_key, sk[1], zk[1]);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            uint32_t wa[WPT], wb[WPT];
            const int r0 = kb * 16 + r8, word = g * (G / 8) + t4 * WPT;
            load_words<WPT>(k_at + r0 * (D / 2) + swizzle<D>(r0, word >> 2) * 16 + (word & 3) * 4, wa);
            load_words<WPT>(k_at + (r0 + 8) * (D / 2) + swizzle<D>(r0 + 8, word >> 2) * 16 + (word & 3) * 4, wb);
            float d[NT][4];
#pragma unroll
            for (int w = 0; w < WPT; ++w) {
              const uint32_t ya = wa[w] >> 8, yb = wb[w] >> 8;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int t = TERMS - 1; t >= 0; --t) {
                  const uint32_t* q = qf[nt][t][g * WPT + w];
                  if (w == 0 && t == TERMS - 1)
                    mma_first(d[nt], even_codes<KC>(wa[w]), even_codes<KC>(wb[w]), odd_codes<KC>(wa[w]), odd_codes<KC>(wb[w]),
                              q[0], q[1]);
                  else
                    mma(d[nt], even_codes<KC>(wa[w]), even_codes<KC>(wb[w]), odd_codes<KC>(wa[w]), odd_codes<KC>(wb[w]), q[0],
                        q[1]);
                  mma(d[nt], even_codes<KC>(ya), even_codes<KC>(yb), odd_codes<KC>(ya), odd_codes<KC>(yb), q[2], q[3]);
                }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                  float& y = s[kb][nt][2 * half + cc];
                  y = g == 0 ? zk[half][g] * qs[nt][cc][g] : fmaf(zk[half][g], qs[nt][cc][g], y);
                  y = fmaf(sk[half][g], d[nt][2 * half + cc], y);
                }
          }
        }
        // ---- m: moved only when a score passes it; weights stay below 1 ----
        bool grow = false;
        float moved[NT][2] = {};
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              float& y = s[kb][nt][k];
              y = fmaf(unit[nt][k & 1], y, -m[nt][k & 1]);
              if (EDGE && key0 + kb * 16 + (k >> 1) * 8 + my_key >= lim[nt][k & 1]) y = -INFINITY;
              grow = grow || y > pass[nt][k & 1];
            }
        grow = __any_sync(0xffffffffu, grow);
        if (grow) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              float top = fmaxf(fmaxf(s[0][nt][cc], s[0][nt][2 + cc]), fmaxf(s[1][nt][cc], s[1][nt][2 + cc]));
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
              const bool move = top > pass[nt][cc];
              const float by = move ? top + kGrow : 0.f;
              const float alpha = exp2_fast(fminf(-by, 0.f));  // (a row's first keys find nothing to scale)
              if (move) pass[nt][cc] = 0.f;
              moved[nt][cc] = by;
              m[nt][cc] += by;
              l[nt][cc] *= alpha;
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                bsum[nt][cc][g] *= alpha;
                wsum[nt][cc][g] *= alpha;
              }
#pragma unroll
              for (int j = 0; j < D / 16; ++j) {
                acc[nt][j][cc] *= alpha;
                acc[nt][j][2 + cc] *= alpha;
              }
#pragma unroll
              for (int kb = 0; kb < 2; ++kb) {
                s[kb][nt][cc] -= by;
                s[kb][nt][2 + cc] -= by;
              }
            }
        }
        // ---- value scales and biases for the whole warp ----
        {
          float sv[NG], zv[NG], most[NG];
          ring.load(st, 1, !EDGE || key0 + lane < ent.end, sv, zv);
          ring.load_most(most);
          bool over = false;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            over = over || (fabsf(sv[g]) * most[g] > kF16Most && fabsf(sv[g]) < INFINITY);
            if (VC) zv[g] = fmaf(8.f, sv[g], zv[g]);
          }
          __syncwarp();
          ring.share(sv, zv);
          __syncwarp();
          if (__any_sync(0xffffffffu, over) || grow) fit(s, sv, moved);
        }
        // ---- weights, their sums, and the second product ----
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          uint32_t pb[NT][NG][TERMS][2];
          float up[NT][NG][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) ring.load_factors(nt, up[nt]);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float sv[NG], zv[NG];
            ring.affine(kb * 16 + half * 8 + my_key, sv, zv);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float w[2];
#pragma unroll
              for (int cc = 0; cc < 2; ++cc) {
                w[cc] = exp2_fast(s[kb][nt][2 * half + cc]);
                l[nt][cc] += w[cc];
              }
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                float f[2];
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                  // a key that this row does not see may hold anything
                  const bool none = EDGE && w[cc] == 0.f;
                  f[cc] = none ? 0.f : w[cc] * sv[g] * up[nt][g][cc];
                  if (!VC) wsum[nt][cc][g] += f[cc];
                  bsum[nt][cc][g] = none ? bsum[nt][cc][g] : fmaf(w[cc], zv[g], bsum[nt][cc][g]);
                }
#pragma unroll
                for (int t = 0; t < TERMS; ++t) pb[nt][g][t][half] = transpose8(take_f16<TERMS == 2>(f[0], f[1]));
              }
            }
          }
          // outputs of fragment i, in group g: these 16 keys' weights times their codes
          auto tile = [&](int i, int g, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              if constexpr (TERMS == 2) {
                float d[4];
                mma_first(d, a0, a1, a2, a3, pb[nt][g][1][0], pb[nt][g][1][1]);
                mma(d, a0, a1, a2, a3, pb[nt][g][0][0], pb[nt][g][0][1]);
#pragma unroll
                for (int k = 0; k < 4; ++k) acc[nt][i][k] += d[k];
              } else {
                mma(acc[nt][i], a0, a1, a2, a3, pb[nt][g][0][0], pb[nt][g][0][1]);
              }
          };
          const int vk = kb * 16 + t4;  // keys vk, + 4, + 8, + 12
          if constexpr (G >= 64) {
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
              const int g = j * 64 / G, word = j * 8 + r8;
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k)
                load_words<1>(v_at + (vk + 4 * k) * (D / 2) + swizzle<D>(vk + 4 * k, word >> 2) * 16 + (word & 3) * 4, &w[k]);
              const uint32_t x0 = __byte_perm(w[0], w[1], 0x5410), x1 = __byte_perm(w[0], w[1], 0x7632);
              const uint32_t y0 = __byte_perm(w[2], w[3], 0x5410), y1 = __byte_perm(w[2], w[3], 0x7632);
              tile(j * 4 + 0, g, even_codes<VC>(x0), even_codes<VC>(x1), even_codes<VC>(y0), even_codes<VC>(y1));
              tile(j * 4 + 1, g, odd_codes<VC>(x0), odd_codes<VC>(x1), odd_codes<VC>(y0), odd_codes<VC>(y1));
              tile(j * 4 + 2, g, even_codes<VC>(x0 >> 8), even_codes<VC>(x1 >> 8), even_codes<VC>(y0 >> 8), even_codes<VC>(y1 >> 8));
              tile(j * 4 + 3, g, odd_codes<VC>(x0 >> 8), odd_codes<VC>(x1 >> 8), odd_codes<VC>(y0 >> 8), odd_codes<VC>(y1 >> 8));
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
                load_words<1>(v_at + (vk + 4 * k) * (D / 2) + swizzle<D>(vk + 4 * k, word >> 2) * 16 + (word & 3) * 4, &w[k]);
              const uint32_t x0 = __byte_perm(w[0], w[1], pick), y0 = __byte_perm(w[2], w[3], pick);
              // (codes 0 and 2, then 1 and 3 of a half: both even or both odd)
              tile(g * 2 + 0, g, even_codes<VC>(x0), even_codes<VC>(x0 >> 8), even_codes<VC>(y0), even_codes<VC>(y0 >> 8));
              tile(g * 2 + 1, g, odd_codes<VC>(x0), odd_codes<VC>(x0 >> 8), odd_codes<VC>(y0), odd_codes<VC>(y0 >> 8));
            }
          }
        }
      };

      // Bare digits' sums grow with the keys, and the tensor core cuts off what it adds to them: 2^-24 of the
      // sum a step, always towards zero, hundreds of times that of what a flat softmax leaves of it.  So 8 times
      // the weights go over to the biases' side before a sum is kCentreTiles long.
      auto centre = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float up[NG][2];
          ring.load_factors(nt, up);
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              float& w = wsum[nt][cc][g];
              bsum[nt][cc][g] = fmaf(8.f * inverse_pow2(up[g][cc]), w, bsum[nt][cc][g]);
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
#pragma unroll
              for (int i = g * G / 16; i < (g + 1) * G / 16; ++i) {
                const float f = i & 1 ? -0x1p-17f : -0x1p-21f;
                acc[nt][i][cc] = fmaf(f, w, acc[nt][i][cc]);
                acc[nt][i][2 + cc] = fmaf(f, w, acc[nt][i][2 + cc]);
              }
              w = 0.f;
            }
        }
      };

      for (int key0 = t0 * kTile; key0 < t1 * kTile; key0 += kTile) {
        copy_wait<S::STAGES - 2>();
        __syncwarp();
        start_copy(next);
        next = look_up();
        if (key0 >= ent.end) break;  // (a tile without keys: the only one of its segment)
        {
          float sk[NG], zk[NG];
          ring.load(st_out, 0, key0 + lane < ent.end, sk, zk);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            if (KC) zk[g] = fmaf(8.f, sk[g], zk[g]);
            // (2^-24 of a score, so that a large key's bias times a query's sum of 2^21 stays in range; an infinite
            // key would give scores of either infinity: no number, as its products are)
            sk[g] = fmaf(sk[g], KC ? 0x1p-24f : 1.f, fmaf(0.f, sk[g], 0.f * zk[g]));
            zk[g] *= 0x1p-24f;
          }
          ring.share(sk, zk);
        }
        __syncwarp();
        if (key0 + kTile > lim_min)
          stage(st_out, key0, std::true_type());
        else
          stage(st_out, key0, std::false_type());
        st_out = st_out + 1 == S::STAGES ? 0 : st_out + 1;
        if (!VC && (key0 / kTile - t0) % kCentreTiles == kCentreTiles - 1) centre();
      }

      // ---- the segment's result, or this warp's part of it ----
      copy_wait<0>();
      __syncwarp();
      const int64_t segment = static_cast<int64_t>(e) * kv_heads + h;
      const bool whole = t0 == 0 && t1 == ent.tiles;
      if (lane == 0) {
        if (t0 == 0) p.span[segment].x = static_cast<int>(self);
        if (t1 == ent.tiles) p.span[segment].y = static_cast<int>(self);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float up[NG][2];
        ring.load_factors(nt, up);
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
          const int row = nt * 8 + 2 * t4 + cc;
          float sum = l[nt][cc];
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
            for (int g = 0; g < NG; ++g) bsum[nt][cc][g] += __shfl_xor_sync(0xffffffffu, bsum[nt][cc][g], o);
          }
          const int r = ent.block * ROWS + row;
          const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(r)));
          const float inv = sum == 0.f || tok >= ent.count ? 0.f : 1.f / sum;
          T* out = static_cast<T*>(p.o) +
                   ((static_cast<int64_t>(ent.b) * p.heads + h * p.per + (r - tok * p.per)) * p.tokens + tok) * D;
          const int64_t slot = (2 * static_cast<int64_t>(self) + (t0 > 0 ? 0 : 1)) * ROWS + row;
          // `n` (4 or 8) neighbouring head dimensions from d on
          auto put = [&](int d, const float* v, auto n_c) {
            constexpr int N = decltype(n_c)::value;
            if (!whole) {
#pragma unroll
              for (int i = 0; i < N; i += 4)
                *reinterpret_cast<float4*>(p.part + slot * D + d + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
            } else if (tok < p.tokens) {
              float f[N];
#pragma unroll
              for (int i = 0; i < N; ++i) f[i] = inv == 0.f ? 0.f : v[i] * inv;
              if constexpr (S::F32) {
#pragma unroll
                for (int i = 0; i < N; i += 4)
                  *reinterpret_cast<float4*>(out + d + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
              } else if constexpr (N == 8) {
                *reinterpret_cast<uint4*>(out + d) = make_uint4(pack_out<T>(f[0], f[1]), pack_out<T>(f[2], f[3]),
                                                                pack_out<T>(f[4], f[5]), pack_out<T>(f[6], f[7]));
              } else {
                *reinterpret_cast<uint2*>(out + d) = make_uint2(pack_out<T>(f[0], f[1]), pack_out<T>(f[2], f[3]));
              }
            }
          };
          // what a sum counts: codes 2^-24 in it, odd ones sixteenfold, weights times scales with their factor
          const float even = VC ? 1.f : 0x1p24f, odd = even * 0x1p-4f;
          if constexpr (G >= 64) {
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
              const float z = bsum[nt][cc][j * 64 / G], down = inverse_pow2(up[j * 64 / G][cc]);
              float v[8];
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                v[u] = fmaf(acc[nt][j * 4 + u][cc] * (u & 1 ? odd : even), down, z);
                v[u + 4] = fmaf(acc[nt][j * 4 + u][2 + cc] * (u & 1 ? odd : even), down, z);
              }
              put((j * 8 + r8) * 8, v, std::integral_constant<int, 8>());
            }
          } else {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const float z = bsum[nt][cc][g], down = inverse_pow2(up[g][cc]);
              const float v[4] = {fmaf(acc[nt][g * 2][cc] * even, down, z), fmaf(acc[nt][g * 2 + 1][cc] * odd, down, z),
                                  fmaf(acc[nt][g * 2][2 + cc] * even, down, z), fmaf(acc[nt][g * 2 + 1][2 + cc] * odd, down, z)};
              put((g * 4 + (r8 & 3)) * 8 + (r8 & 4), v, std::integral_constant<int, 4>());
            }
          }
          if (!whole && r8 == 0) {
            p.part_ml[slot * 2] = pass[nt][cc] == kFloor ? kFloor : m[nt][cc];  // (kFloor: no key seen)
            p.part_ml[slot * 2 + 1] = sum;
          }
        }
      }
    }
    base += static_cast<uint64_t>(kv_heads) * units;
    ++e;
  }
}

// Joins the partials of a segment: partial 1 of its first warp, then the
// partials 0 of the warps after it, in that order.  WARPS 1: a warp to a row, a
// block to eight rows of a segment.  Else a block to a row, its warps taking
// every WARPS-th partial each, joined in shared memory.
template <typename S, typename T, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 256 : 32 * WARPS) combine_kernel(const AttnParams p) {
  constexpr int D = S::D, ROWS = S::ROWS, E = D / 32;
  constexpr bool WIDE = WARPS > 1;
  const int segment = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // attn_kernel is done and its partials are visible
  const int2 span = p.span[segment];
  if (span.x == span.y) return;
  const int kv_heads = p.c.map.kv_heads;
  const int e = segment / kv_heads, h = segment - e * kv_heads;
  const int b = static_cast<int>(div_by(p.by_blocks, static_cast<uint32_t>(e)));
  const int row = WIDE ? blockIdx.y : blockIdx.y * 8 + warp;
  const int r = (e - b * p.blocks) * ROWS + row;
  const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(r)));
  if (tok >= p.tokens) return;
  const bool live = !p.counts || tok < p.counts[b];
  auto at = [&](int k) { return (2 * static_cast<int64_t>(k) + (k == span.x ? 1 : 0)) * ROWS + row; };
  // (a running maximum, so that no load waits for another)
  float m = kFloor, l = 0.f, o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.f;
#pragma unroll 4
  for (int k = span.x + (WIDE ? warp : 0); k <= span.y; k += WARPS) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + at(k) * 2);
    const float2* v = reinterpret_cast<const float2*>(p.part + at(k) * D) + lane;
    const float m_new = fmaxf(m, ml.x), was = exp2_fast(m - m_new), f = exp2_fast(ml.x - m_new);
    m = m_new;
    l = fmaf(l, was, f * ml.y);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 x = v[i * 16];
      o[i] = fmaf(f, x.x, o[i] * was);
      o[i + 1] = fmaf(f, x.y, o[i + 1] * was);
    }
  }
  if constexpr (WIDE) {
    __shared__ float s_o[WARPS][D], s_l[WARPS], s_m[WARPS];
#pragma unroll
    for (int i = 0; i < E; i += 2) *reinterpret_cast<float2*>(&s_o[warp][i * 32 + lane * 2]) = make_float2(o[i], o[i + 1]);
    if (lane == 0) {
      s_l[warp] = l;
      s_m[warp] = m;
    }
    __syncthreads();
    if (warp) return;
#pragma unroll
    for (int w = 1; w < WARPS; ++w) m = fmaxf(m, s_m[w]);
    l = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = exp2_fast(s_m[w] - m);
      l = fmaf(f, s_l[w], l);
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        o[i] = fmaf(f, s_o[w][i * 32 + lane * 2], o[i]);
        o[i + 1] = fmaf(f, s_o[w][i * 32 + lane * 2 + 1], o[i + 1]);
      }
    }
  }
  const float inv = l == 0.f || !live ? 0.f : 1.f / l;
  T* out = static_cast<T*>(p.o) + ((static_cast<int64_t>(b) * p.heads + h * p.per + (r - tok * p.per)) * p.tokens + tok) * D + lane * 2;
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    const float x = inv == 0.f ? 0.f : o[i] * inv, y = inv == 0.f ? 0.f : o[i + 1] * inv;
    if constexpr (S::F32)
      *reinterpret_cast<float2*>(out + i * 32) = make_float2(x, y);
    else
      *reinterpret_cast<uint32_t*>(out + i * 32) = pack_out<T>(x, y);
  }
}

// Blocks of a launch and its scratch bytes: partials of every warp, a span per segment.
template <typename S> int grid_of() { return sm_count_current() * S::CTAS; }
template <typename S> size_t part_floats() { return static_cast<size_t>(grid_of<S>()) * kWarps * 2 * S::ROWS; }
template <typename S> int64_t blocks_of(int64_t rows) { return (rows + S::ROWS - 1) / S::ROWS; }
template <typename S> size_t bytes_of(int64_t batch, int kv_heads, int64_t rows) {
  return part_floats<S>() * (S::D + 2) * 4 + static_cast<size_t>(batch * kv_heads * blocks_of<S>(rows)) * sizeof(int2);
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
  const int64_t blocks = blocks_of<S>(static_cast<int64_t>(p.tokens) * p.per);
  const int64_t segments = p.batch * blocks * p.c.map.kv_heads;
  PHEW_REQUIRE(segments < (1ll << 31), "phew_kv_attention: too many query rows");
  p.blocks = static_cast<int>(blocks);
  p.by_blocks = fast_div(static_cast<uint32_t>(blocks));
  const int page = p.c.map.page_size;
  p.step_col = kTile / page;
  p.step_row = kTile % page;
  p.page_rows = static_cast<uint32_t>(p.c.map.kv_heads) * static_cast<uint32_t>(page);
  p.eights = page % 8 == 0;
  p.part = static_cast<float*>(workspace);
  p.part_ml = p.part + part_floats<S>() * S::D;
  p.span = reinterpret_cast<int2*>(p.part_ml + part_floats<S>() * 2);
  static SmemAllowed allowed;
  if (int s = allow_smem(allowed, attn_kernel<S, T>, S::SMEM)) return s;
  attn_kernel<S, T><<<grid_of<S>(), kWarps * 32, S::SMEM, st>>>(p);
  if (int s = launch_status("kv attn_kernel")) return s;
  // a programmatic dependent: set up while attn_kernel runs
  cudaLaunchConfig_t cfg = {};
  // partials to a segment: about the warps that it could be spread over.  Up to four, one warp reads them in one
  // go; eight warps (18 to a segment: 15 us for a call, 24 with one warp); sixteen (222: 45 us, 49 with eight)
  const int64_t spread = static_cast<int64_t>(grid_of<S>()) * kWarps / segments;
  const int warps = spread <= 4 ? 1 : spread <= 64 ? 8 : 16;
  cfg.gridDim = dim3(static_cast<unsigned>(segments), warps > 1 ? S::ROWS : S::NT);
  cfg.blockDim = dim3(warps > 1 ? 32 * warps : 256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PHEW_CHECK_CUDA(warps == 1   ? cudaLaunchKernelEx(&cfg, combine_kernel<S, T, 1>, p)
                  : warps == 8 ? cudaLaunchKernelEx(&cfg, combine_kernel<S, T, 8>, p)
                               : cudaLaunchKernelEx(&cfg, combine_kernel<S, T, 16>, p));
  return launch_status("kv combine_kernel");
}

// Row tiles of eight to a block: two for more than eight query rows, where registers allow it (16-bit
// types with heads up to 128; wider heads and the two terms of f32 would spill the second tile).  Two against one,
// 8 cache heads of 8192 keys / 16 x 8 of 2048 / 8 of 65536: 12 rows 16 : 16, 26 : 29, 36 : 44 us, 32 rows 17 : 20,
// 37 : 44, 57 : 75.
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
template <typename T> size_t attn_bytes(int64_t batch, int kv_heads, int head_dim, int group, int64_t rows) {
  return with_shape<T>(head_dim, group, rows, [&](auto s) { return bytes_of<decltype(s)>(batch, kv_heads, rows); });
}
template <typename T> int run_attn(const AttnParams& p, void* workspace, cudaStream_t st) {
  return with_shape<T>(p.c.head_dim, p.c.group, static_cast<int64_t>(p.tokens) * p.per,
                       [&](auto s) { return launch_attn<decltype(s), T>(p, workspace, st); });
}
#ifndef PHEW_KV_ATTN_TYPE
extern template size_t attn_bytes<float>(int64_t, int, int, int, int64_t);
extern template size_t attn_bytes<f16>(int64_t, int, int, int, int64_t);
extern template size_t attn_bytes<bf16>(int64_t, int, int, int, int64_t);
extern template int run_attn<float>(const AttnParams&, void*, cudaStream_t);
extern template int run_attn<f16>(const AttnParams&, void*, cudaStream_t);
extern template int run_attn<bf16>(const AttnParams&, void*, cudaStream_t);
#endif

}  // namespace kv
}  // namespace phew
