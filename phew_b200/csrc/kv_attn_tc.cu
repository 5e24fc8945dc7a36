// Attention of many query rows over a 4-bit cache (chunks of a prompt), on the
// tcgen05 tensor cores.
//
// The rows of a cache head are r = token * per + head over its `per` query
// heads; a CTA takes 256 of them (two 128-row tiles a and b) and walks the
// keys in tiles of 128.  Bound by the chain score product - softmax - output
// product of each tile, at about the rate of the exponentials.
//
// Operands are f16 whatever the type: a tile's keys and its values (dense; those
// of a quarter of it, 32 keys, where tiles are packed) in units of a power of
// two, the largest magnitude at [2^14, 2^15); a query in units of its own,
// exactly.  With ke, ve the units' exponents
//   t_ij = c_i 2^ke (q'_i . k'_j) + ve,  p_ij = 2^(t_ij - m_i),  o_i = sum_j p_ij v'_j,
//   l_i = sum_j p_ij 2^-ve
// so units cost an element nothing: they enter with the constants of a tile.
// m_i is 7 below a row's largest t when it moves, which leaves f16's smallest
// weight 2^-31 of the largest.  Keys, values and weights are rounded to 11 bits
// this way, for bf16 too (whose own 8 bits cost 3.2e-3 of an output's norm, 1.7e-3
// of them its rounding).  Scores, maxima and sums are 32-bit.  Where magnitudes in
// a tile lie further apart than f16 holds (Reach::odd) its rows are computed again
// by plain_rows_kernel, in fp32: 27 ms for the chunk below, for caches that no
// model writes.  (A launch of its own, 2 us; at the end of this kernel its code
// cost 10 to 20.)
//
// Two forms:
//
// Dense (kExpandBlocks row blocks or more, whose every CTA would expand the
// same keys again): the cache is expanded once to scratch, and tiles arrive by
// TMA.  One pass of HBM over the keys against 0.5 us for each CTA and tile
// (measured: 256 CTAs x 56 tiles).
//
// Packed (few row blocks): producer warps load packed rows (two units of 32
// keys ahead, in registers), expand them as f16(scale * code + bias) - two
// instructions a value: a shift and a logic operation per pair of codes, an
// exact subtraction, a packed multiply-add - and store them in the 128-byte
// swizzle that the tensor core reads.  Those instructions take issue slots
// from the softmax, which is why the dense form exists; more producer warps
// (7 for 3) did not help.
//
// A pair of tiles takes 3600 clocks: each query tile's chain of 1750 in the
// softmax (1024 of them the exponentials), 360 until its warps are heard, 1560
// in its two products; the tensor core, which serves both tiles, is busy for
// 2100.  Measured without gain (247 us for the chunk below): two threads to a
// row (244), the output product begun on the first half of the weights (258),
// a quarter of the exponentials as polynomials (274), spinning on barriers
// (273).
//
//   warp 0        TMEM owner and MMA issuer: per key tile j and query tile t,
//                 O_t += P_t V_j, then S_t = Q_t K_{j+1}^T
//   next warps    dense: one, TMA.  Packed: three producers; the line of units
//                 K_0, V_0, K_1, ... in quarters of 32 keys, every third one to
//                 a warp.  Both fill two-deep rings of K and V
//   last 8 warps  softmax of tile a and b, one query row per thread; they also
//                 convert Q and write O
//
// TMEM: S_a, S_b, O_a, O_b of 128 columns each.  Heads of 256 have one query
// tile to a CTA (O takes 256 columns), rings one deep and always the dense form.
//
// Within eight neighbouring head dimensions packed tiles hold them in the
// order 0 4 1 5 2 6 3 7, which is how pairs fall out of a word of codes; queries
// are stored to match and outputs read back through the same order.
//
// Long caches with few rows are split: a CTA takes a share of the key tiles
// and leaves partial sums, joined in a fixed order by the combine kernel.
//
// Measured, causal, heads of 128 in bf16: two prompts of 4096 tokens on 32
// heads, 334 us (823 TFLOP/s); the last 2048 of 8192 tokens on 32 heads over 8,
// 247 us (974 TFLOP/s).  Errors of an output's norm: 1.7e-3 in bf16, 4.6e-4 in
// f16 (2.1e-4 its own rounding; 2.9e-4 with keys and values as two terms each,
// at 462 us instead of 257 for that chunk in f16).
//
// Every wait is bounded; one that runs out sets error_flag[1] and the CTA
// winds down with its TMEM freed.
#include "attn_softmax.cuh"
#include "kv_attn_tc.cuh"

namespace phew {
namespace kv {
namespace {

using namespace tc;
using attn::add2;
using attn::ex2;
using attn::f2;
using attn::fma2;
using attn::hi_of;
using attn::lo_of;
using attn::max3;
using attn::pack2;

constexpr int kTileRows = 128;
constexpr int kTcTile = 128;       // keys of a tile
constexpr int kProducers = 3;      // warps 1 .. 3 of the packed form
constexpr int kTmemCols = 512;
constexpr float kTcFloor = -1.0e38f;
constexpr float kTcUnder = 7.0f;   // log2 units that m lies below a row's largest t when it moves
constexpr float kTcMost = 15.0f;   // ... that t may pass it by (weights up to 2^15 are f16)
constexpr int kUnitMin = -60;      // their smallest exponent: l, in units of values, stays in fp32's range
constexpr int kUnits = 4;          // tiles whose units are kept: a softmax warp is at most two behind the loads

template <int D_, int G_> struct TcShape {
  static constexpr int D = D_, G = G_, NG = D / G;
  static constexpr int HALVES = D / 64;
  static constexpr int HALF_BYTES = kTcTile * 128;           // 64 columns of 16 bits, 128-byte rows
  static constexpr int TILE_BYTES = HALF_BYTES * HALVES;
  static constexpr int QT = D <= 128 ? 2 : 1;                // query tiles of a CTA
  static constexpr int ROWS = QT * kTileRows;
  static constexpr int RING = D <= 128 ? 2 : 1;              // tiles of K, and of V, in flight
  static constexpr int SMEM = (QT + 2 * RING) * TILE_BYTES + 1024 + 512;
  // slot and phase of key tile j in the rings
  static __device__ __forceinline__ int slot(int j) { return RING == 2 ? j & 1 : 0; }
  static __device__ __forceinline__ uint32_t phase(int j) { return (RING == 2 ? j >> 1 : j) & 1; }
};

constexpr int tc_threads(bool dense, int tiles) { return 32 * ((dense ? 2 : 1 + kProducers) + 4 * tiles); }

// A tile's units, as softmax threads take them: of its quarters, or in the dense form of the whole tile ([0]).
struct alignas(16) Units {
  float k[4];       // 2^ke
  float v[4], l[4]; // ve, 2^-ve
  uint8_t odd[8];   // of keys, of values
  uint32_t pad[2];
};
static_assert(sizeof(Units) == 64, "copied in 16-byte pieces");

struct TcParams {
  Cache c;
  const void* q;
  int64_t st[3];
  void* o;
  const int32_t* lengths;
  const int32_t* counts;
  int batch, heads, tokens, per;
  int blocks;  // 256-row blocks of a cache head
  int splits;
  int rows;    // dense: token rows of a cache head in the expanded keys and values
  const Units* units;  // dense: [batch * kv_heads][rows / 128]
  int* odd;            // of every CTA, a bit to a query tile: keys were met that f16 does not hold
  FastDiv by_per;
  float scale_log2;  // > 0
  bool causal;
  float* part;     // [segment][split][256][D] when splits > 1
  float* part_ml;  // [segment][split][256][2]
  int* error_flag;
  unsigned long long wait_ns;
  int withhold;  // test hook: the V tile of this key tile is never announced (-1: none)
};

// code pairs (U, U + 4) of a word as f16, exactly
template <int U> __device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  uint32_t d, x;
  const uint32_t y = U == 0 ? w << 4 : w >> (U == 0 ? 0 : 4 * U - 4);
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(x) : "r"(y), "r"(0x00f000f0u), "r"(0x54005400u));
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0x54005400u));  // 64 + n - 64
  return d;
}
__device__ __forceinline__ uint32_t fma_pair(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + e) << 23); }  // -126 .. 127
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// Magnitudes that a part of a tile's codes reach, as bits (which order as the magnitudes do), 0 where there is none.
struct Reach {
  uint32_t far = 0;                                       // the largest
  uint32_t key = 0x7f7fffffu, group = 0x7f7fffffu;        // the smallest key's largest, the smallest group's

  // A key's groups, one after the other, then `done`.  Parts that are no finite numbers count as nothing; a group of
  // zeros (bias 0, the smallest scale there is) has no magnitude to lose.
  uint32_t now = 0;
  __device__ __forceinline__ void add(float s, float z) {
    if (!(finite(s) && finite(z))) return;
    const uint32_t r = min(max(__float_as_uint(fabsf(z)), __float_as_uint(fabsf(fmaf(15.f, s, z)))), 0x7f7fffffu);
    far = max(far, r);
    if (z == 0.f && fabsf(s) < 1.1e-8f) return;
    now = max(now, r);
    if (r) group = min(group, r);
  }
  __device__ __forceinline__ void done() {
    if (now) key = min(key, now);
  }
  __device__ __forceinline__ void across_warp() {
    far = __reduce_max_sync(0xffffffffu, far);
    key = __reduce_min_sync(0xffffffffu, key);
    group = __reduce_min_sync(0xffffffffu, group);
  }
  __device__ __forceinline__ int unit() const { return max(static_cast<int>(far >> 23) - 127 - 14, kUnitMin); }
  // Whether f16 does not hold the part.  In its units a group's values keep 11 bits down to 2^-14; `finest`: what its
  // magnitude has to be for that (packed tiles round the scale too, a fifteenth of it or less).  A row that gives the
  // largest value no weight has its m from the other keys of the part, as far too high for the rest of the sequence as
  // the largest lies above them; down to 2^-2 that leaves weights steps of 2^-16 of the largest.
  __device__ __forceinline__ bool odd(int side, int finest) const {
    const auto below = [&](uint32_t bits, int e) { return static_cast<int>(bits >> 23) - 127 - unit() < e; };
    return far && (below(group, finest) || (side && below(key, -2)));
  }
};

// Units of a side: of `part` of NU parts of a tile.
template <int NU> __device__ __forceinline__ void set_units(Units* u, int side, int part, int e, bool odd) {
  if (side == 0) {
    u->k[part] = pow2(e);
  } else {
    u->v[part] = static_cast<float>(e);
    u->l[part] = pow2(-e);
  }
  if (NU == 1)
    *reinterpret_cast<uint32_t*>(u->odd + side * 4) = odd;
  else
    u->odd[side * 4 + part] = odd;
}

// Exponent of a row of queries: in units of it the row's largest magnitude, `top`, lies at [2^14, 2^15).
__device__ __forceinline__ int query_unit(float top) { return static_cast<int>(max(__float_as_uint(top) >> 23, 20u)) - 127 - 14; }

template <bool BF16> __device__ __forceinline__ float half_of(uint32_t w, int i) {
  const uint32_t x = i ? w >> 16 : w & 0xffffu;
  return BF16 ? __uint_as_float(x << 16) : to_f32(f16{static_cast<uint16_t>(x)});
}

// What a row's scores are worth, and the exponents of its values, in each of a tile's NU parts.
template <int NU> struct Row {
  float c[NU], v[NU];
};
// `query`: 2^qe.  A worth is more than nothing, so that a masked score stays -infinity.
template <int NU> __device__ __forceinline__ Row<NU> row_units(float scale_log2, float query, uint32_t units) {
  Row<NU> r;
  uint32_t k[NU], v[NU];
  load_words<NU>(units, k);
  load_words<NU>(units + 16, v);
#pragma unroll
  for (int h = 0; h < NU; ++h) {
    r.c[h] = fmaxf(scale_log2 * (query * __uint_as_float(k[h])), 0x1p-126f);
    r.v[h] = __uint_as_float(v[h]);
  }
  return r;
}

// Weights of a row's 128 scores, packed into 64 pairs of f16 and stored to TMEM at s_addr (columns 0..63 of the S
// buffer).  Returns the row sum of this tile's (unrounded) weights.
template <int NU>
__device__ __forceinline__ float weights(const uint32_t* raw, const Row<NU>& r, float m, uint32_t units, uint32_t s_addr) {
  float sum = 0.f;
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    uint32_t down;
    load_words<1>(units + 32 + (NU == 1 ? 0 : 4 * h), &down);
    const float c = r.c[NU == 1 ? 0 : h], off = r.v[NU == 1 ? 0 : h] - m;
    const uint64_t c2 = f2(c, c), o2 = f2(off, off);
    uint64_t l2[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int pi = 16 * h + i;
      const uint64_t x = fma2(f2(__uint_as_float(raw[2 * pi]), __uint_as_float(raw[2 * pi + 1])), c2, o2);
      const uint64_t e = f2(ex2(lo_of(x)), ex2(hi_of(x)));
      l2[i & 1] = add2(l2[i & 1], e);
      pk[i] = pack2<false>(lo_of(e), hi_of(e));
    }
    tmem_st16(s_addr + 16 * h, pk);
    const uint64_t l = add2(l2[0], l2[1]);
    sum = fmaf(lo_of(l) + hi_of(l), __uint_as_float(down), sum);
  }
  return sum;
}

// Largest t of a row's 128 scores (NaN ones aside).
template <int NU> __device__ __forceinline__ float largest(const uint32_t* raw, const Row<NU>& r) {
  float top[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    float m4[4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
      m4[a] = max3(__uint_as_float(raw[32 * h + 2 * a]), __uint_as_float(raw[32 * h + 2 * a + 1]),
                   __uint_as_float(raw[32 * h + 8 + a]));
#pragma unroll
    for (int i = 12; i + 8 <= 32; i += 8)
#pragma unroll
      for (int a = 0; a < 4; ++a)
        m4[a] = max3(m4[a], __uint_as_float(raw[32 * h + i + 2 * a]), __uint_as_float(raw[32 * h + i + 2 * a + 1]));
    const float m = max3(max3(m4[0], m4[1], __uint_as_float(raw[32 * h + 28])), max3(m4[2], m4[3], __uint_as_float(raw[32 * h + 29])),
                         fmaxf(__uint_as_float(raw[32 * h + 30]), __uint_as_float(raw[32 * h + 31])));
    top[h] = NU == 1 ? m : fmaf(m, r.c[NU == 1 ? 0 : h], r.v[NU == 1 ? 0 : h]);
  }
  const float m = max3(top[0], top[1], fmaxf(top[2], top[3]));
  return NU == 1 ? fmaf(m, r.c[0], r.v[0]) : m;
}

__device__ __forceinline__ void store_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, int bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// shared-memory writes of this thread become visible to the tensor core
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A CTA's rows of queries and key tiles, by its number.
struct Share {
  int bh, b, h, rb, split, count, length, row0;
  int j0, n_max, n_t[2];  // first key tile, how many from it on, for both query tiles and each
};
template <typename S> __device__ __forceinline__ Share share_of(const TcParams& p) {
  Share s;
  // Cache heads in groups of 16, so that the CTAs running at one time share few heads' keys in the L2; within a
  // group row blocks from the last (the longest under a causal mask) down, a block's heads and splits together.
  const int kv_heads = p.c.map.kv_heads;
  const int all_heads = p.batch * kv_heads, in_group = 16 * p.blocks * p.splits;
  const int group = static_cast<int>(blockIdx.x) / in_group, rem = static_cast<int>(blockIdx.x) % in_group;
  const int wide = min(16, all_heads - 16 * group) * p.splits;
  s.rb = p.blocks - 1 - rem / wide;
  s.split = rem % wide % p.splits;
  s.bh = 16 * group + rem % wide / p.splits;
  s.b = s.bh / kv_heads;
  s.h = s.bh % kv_heads;
  s.count = p.counts ? clamp_count(__ldg(p.counts + s.b), p.tokens) : p.tokens;
  s.length = clamp_count(__ldg(p.lengths + s.b), capacity(p.c.map));
  s.row0 = s.rb * S::ROWS;
  int need[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int first = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(s.row0 + t * kTileRows)));
    const int last = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(s.row0 + t * kTileRows + kTileRows - 1)));
    const int end = first >= s.count ? 0 : seen_end(s.length, s.count, last < s.count ? last : s.count - 1, p.causal);
    need[t] = t < S::QT ? (end + kTcTile - 1) / kTcTile : 0;
  }
  const int all = max(need[0], need[1]);
  s.j0 = static_cast<int>(static_cast<int64_t>(all) * s.split / p.splits);
  s.n_max = static_cast<int>(static_cast<int64_t>(all) * (s.split + 1) / p.splits) - s.j0;
  for (int t = 0; t < 2; ++t) s.n_t[t] = min(max(need[t] - s.j0, 0), s.n_max);
  return s;
}

template <typename S, bool BF16, bool DENSE>
__global__ void __launch_bounds__(tc_threads(DENSE, S::QT), 1)
    attn_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const TcParams p) {
  constexpr int D = S::D, NG = S::NG;
  constexpr int FIRST = DENSE ? 2 : 1 + kProducers;  // softmax warp
  constexpr int NU = DENSE ? 1 : 4;                  // units to a tile
  using T = typename std::conditional<BF16, bf16, f16>::type;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                                       // [QT] tiles
  uint8_t* sK = smem + S::QT * S::TILE_BYTES;               // [RING]
  uint8_t* sV = smem + (S::QT + S::RING) * S::TILE_BYTES;   // [RING]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (S::QT + 2 * S::RING) * S::TILE_BYTES);
  uint64_t* q_full = bars;        // [2]
  uint64_t* k_full = bars + 2;    // [2]
  uint64_t* k_empty = bars + 4;   // [2]
  uint64_t* v_full = bars + 6;    // [2]
  uint64_t* v_empty = bars + 8;   // [2]
  uint64_t* s_full = bars + 10;   // [2]
  uint64_t* p_full = bars + 12;   // [2]
  uint64_t* o_done = bars + 14;   // [2]
  uint64_t* drain = bars + 16;
  uint64_t* u_full = bars + 17;   // [kUnits]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 21);
  int* s_poison = reinterpret_cast<int*>(tmem_slot + 1);  // first key whose values are not finite
  int* s_odd = reinterpret_cast<int*>(bars + 22);         // [2] a tile of keys that f16 does not hold was met
  Units* s_units = reinterpret_cast<Units*>(bars + 24);   // [kUnits]
  int* wait_flag = p.error_flag + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- which rows and which keys ----
  const Share sh = share_of<S>(p);
  const int b = sh.b, h = sh.h, bh = sh.bh, rb = sh.rb, split = sh.split, count = sh.count, length = sh.length;
  const int row0 = sh.row0, j0 = sh.j0, n_max = sh.n_max;
  const int n_t[2] = {sh.n_t[0], sh.n_t[1]};
  if (threadIdx.x == 0 && length != __ldg(p.lengths + b)) atomicExch(p.error_flag, PHEW_ERR_INVALID);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&k_full[i], DENSE ? 1 : 4);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], DENSE ? 1 : 4);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(drain, 1);
    for (int i = 0; i < kUnits; ++i) mbar_init(&u_full[i], DENSE ? 1 : 8);
    *s_poison = 0x7fffffff;
    s_odd[0] = s_odd[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) tmem_alloc(tmem_slot, kTmemCols);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  int k_last[2] = {-1, -1}, v_last[2] = {-1, -1};  // dense: the key tile whose load each ring slot received last
  int u_last = -1;                                 // ... whose units were loaded last

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t id_qk = instr_desc_f16(0, 0, kTileRows, kTcTile);
      constexpr uint32_t id_pv = instr_desc_f16(0, 1, kTileRows, D);
      auto issue_s = [&](int t, uint32_t k_addr) {
        const uint32_t q_addr = smem_u32(sQ + t * S::TILE_BYTES);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * S::HALF_BYTES + (kk & 3) * 32;
          mma_ss(tmem + t * 128, smem_desc(q_addr + off, 16, 1024), smem_desc(k_addr + off, 16, 1024), id_qk,
                 kk > 0 ? 1u : 0u);
        }
        commit(&s_full[t]);
      };
      if (n_max > 0) {
        if (!mbar_wait(&k_full[0], 0, wait_flag, p.wait_ns)) ok = false;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!ok || n_t[t] == 0) continue;
          if (!mbar_wait(&q_full[t], 0, wait_flag, p.wait_ns)) { ok = false; continue; }
          fence_after_sync();
          issue_s(t, smem_u32(sK));
        }
        if (ok) commit(&k_empty[0]);
      }
      for (int j = 0; j < n_max && ok; ++j) {
        const int s = S::slot(j), s1 = S::slot(j + 1);
        const bool more = j + 1 < n_max;
        if (!mbar_wait(&v_full[s], S::phase(j), wait_flag, p.wait_ns)) { ok = false; break; }
        if (more && !mbar_wait(&k_full[s1], S::phase(j + 1), wait_flag, p.wait_ns)) { ok = false; break; }
        const uint32_t v_addr = smem_u32(sV + s * S::TILE_BYTES);
        const uint32_t k_addr = smem_u32(sK + s1 * S::TILE_BYTES);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (!ok || j >= n_t[t]) continue;
          if (!mbar_wait(&p_full[t], j & 1, wait_flag, p.wait_ns)) { ok = false; continue; }
          fence_after_sync();
#pragma unroll
          for (int kk = 0; kk < kTcTile / 16; ++kk)
            mma_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, smem_desc(v_addr + kk * (16 * 128), S::HALF_BYTES, 1024),
                   id_pv, (j > 0 || kk > 0) ? 1u : 0u);
          commit(&o_done[t]);
          if (j + 1 < n_t[t]) {
            // S_t holds P_t until this product has read it
            if (!mbar_wait(&o_done[t], j & 1, wait_flag, p.wait_ns)) { ok = false; continue; }
            fence_after_sync();
            issue_s(t, k_addr);
          }
        }
        if (!ok) break;
        commit(&v_empty[s]);
        if (more) commit(&k_empty[s1]);
      }
    }
  } else if (DENSE && warp == 1) {
    // ---------------- TMA ----------------
    if (lane == 0) {
      // the expanded keys and values are there.  Every CTA waits, one without keys too: a grid of which none did
      // could end before the expansion, and what follows it on the stream would find that still writing.
      asm volatile("griddepcontrol.wait;" ::: "memory");
      const int first = bh * p.rows + j0 * kTcTile;
      auto load = [&](const CUtensorMap* tm, uint64_t* bar, uint8_t* dst, int row) {
        mbar_expect_tx(bar, S::TILE_BYTES);
#pragma unroll
        for (int i = 0; i < S::HALVES; ++i) tma_load_2d(dst + i * S::HALF_BYTES, tm, bar, i * 64, row);
      };
      for (int j = 0; j < n_max && ok; ++j) {
        const int s = S::slot(j);
        const uint32_t ph = S::phase(j) ^ 1;
        if (!mbar_wait(&k_empty[s], ph, wait_flag, p.wait_ns)) { ok = false; break; }
        load(&tm_k, &k_full[s], sK + s * S::TILE_BYTES, first + j * kTcTile);
        // (the softmax has read the units of tile j - 4: scores of j - 2 were made after its weights of j - 3)
        u_last = j;
        uint64_t* bar = &u_full[j & (kUnits - 1)];
        mbar_expect_tx(bar, sizeof(Units));
        bulk_load(&s_units[j & (kUnits - 1)], p.units + static_cast<int64_t>(bh) * (p.rows / kTcTile) + j0 + j, sizeof(Units), bar);
        (s ? k_last[1] : k_last[0]) = j;
        if (!mbar_wait(&v_empty[s], ph, wait_flag, p.wait_ns)) { ok = false; break; }
        if (j == p.withhold) continue;  // test hook: this V tile never lands
        load(&tm_v, &v_full[s], sV + s * S::TILE_BYTES, first + j * kTcTile);
        (s ? v_last[1] : v_last[0]) = j;
      }
    }
  } else if (!DENSE && warp <= kProducers) {
    // ---------------- producers ----------------
    // unit u: quarter u % 4 of K (u / 4 even) or V (odd) of tile u / 8; this warp takes u = warp - 1, + 3, ...
    const int units = 8 * n_max;
    // a lane's key of a unit: its row (looked up a round ahead), then its codes and scales, which wait in
    // registers until the unit's turn comes.  (Copies to shared memory in their place would have to land
    // before every fence_async_shared.)
    struct Look {
      int page, row;  // row -1: no key
    };
    struct Packed {
      uint4 code[D / 32];
      uint32_t sb[2][(NG + 1) / 2];  // scales, biases
    };
    auto look_up = [&](int u) {
      Look k{0, -1};
      const int key = (j0 + (u >> 3)) * kTcTile + (u & 3) * 32 + lane;
      if (u < units && key < length) {
        const int col = static_cast<int>(div_by(p.c.map.by_page, static_cast<uint32_t>(key)));
        k.row = key - col * p.c.map.page_size;
        k.page = page_at(p.c.map, b, col);
      }
      return k;
    };
    auto fetch = [&](int u, const Look& k) {
      Packed x{};
      if (k.row >= 0) {
        if (page_ok(p.c.map, k.page)) {
          const int side = (u >> 2) & 1;
          const int64_t row = row_at(p.c.map, k.page, h, k.row);
          const uint4* codes = reinterpret_cast<const uint4*>(p.c.codes[side] + row * (D / 8));
#pragma unroll
          for (int i = 0; i < D / 32; ++i) x.code[i] = __ldg(codes + i);
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            const T* at = static_cast<const T*>(a ? p.c.biases[side] : p.c.scales[side]) + row * NG;
            if constexpr (NG == 1) {
              x.sb[a][0] = __ldg(reinterpret_cast<const uint16_t*>(at));
            } else {
#pragma unroll
              for (int i = 0; i < NG / 2; ++i) x.sb[a][i] = __ldg(reinterpret_cast<const uint32_t*>(at) + i);
            }
          }
        } else {
          atomicExch(p.error_flag, PHEW_ERR_INVALID);
        }
      }
      return x;
    };
    auto expand = [&](int u, Packed& x) {
      const int j = u >> 3, side = (u >> 2) & 1, row = (u & 3) * 32 + lane, slot = S::slot(j);
      // in units of the quarter's own power of two
      float s[NG], z[NG];
      Reach reach;
      bool fine = true;  // parts finite
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        s[g] = half_of<BF16>(x.sb[0][g / 2], g & 1);
        z[g] = half_of<BF16>(x.sb[1][g / 2], g & 1);
        reach.add(s[g], z[g]);
        fine = fine && finite(s[g]) && finite(z[g]);
      }
      reach.done();
      reach.across_warp();
      const int unit = reach.unit();
      const float down = pow2(-unit);
      if (lane == 0) {
        // (read by the softmax when the scores are there; it has read those of tile j - 4: this warp's unit before
        // this one found its slot empty of tile j - 3's)
        uint64_t* bar = &u_full[j & (kUnits - 1)];
        set_units<NU>(&s_units[j & (kUnits - 1)], side, u & 3, unit, reach.odd(side, -10));
        mbar_arrive(bar);
      }
      if (side == 1 && !fine) {
        // a weight of zero times infinity is no number, and a later query's keys may not touch an earlier
        // one: the values count as zero here and as "no number" for every row that sees the key
        atomicMin(s_poison, (j0 + j) * kTcTile + row);
#pragma unroll
        for (int g = 0; g < NG; ++g) s[g] = z[g] = 0.f;
      }
      uint32_t sc[NG], bi[NG];  // each twice in a register
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        sc[g] = pack2<false>(s[g] * down, s[g] * down);
        bi[g] = pack2<false>(z[g] * down, z[g] * down);
      }
      uint64_t* full = side == 0 ? &k_full[slot] : &v_full[slot];
      uint64_t* empty = side == 0 ? &k_empty[slot] : &v_empty[slot];
      if (lane == 0 && !mbar_wait(empty, S::phase(j) ^ 1, wait_flag, p.wait_ns)) ok = false;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) return;
      const uint32_t dst = smem_u32((side == 0 ? sK : sV) + slot * S::TILE_BYTES) + row * 128;
#pragma unroll
      for (int ch = 0; ch < D / 32; ++ch) {
        const uint32_t word[4] = {x.code[ch].x, x.code[ch].y, x.code[ch].z, x.code[ch].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int g = (ch * 32 + i * 8) / S::G, c16 = ch * 4 + i;
          const uint32_t v[4] = {fma_pair(sc[g], code_pair<0>(word[i]), bi[g]), fma_pair(sc[g], code_pair<1>(word[i]), bi[g]),
                                 fma_pair(sc[g], code_pair<2>(word[i]), bi[g]), fma_pair(sc[g], code_pair<3>(word[i]), bi[g])};
          store_shared16(dst + (c16 >> 3) * S::HALF_BYTES + (((c16 & 7) ^ (row & 7)) << 4), v[0], v[1], v[2], v[3]);
        }
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0 && !(side == 1 && j == p.withhold)) mbar_arrive(full);
    };
    constexpr int P = kProducers;
    const int u0 = warp - 1;
    Look la = look_up(u0), lb = look_up(u0 + P);
    Packed xa = fetch(u0, la), xb = fetch(u0 + P, lb);
    la = look_up(u0 + 2 * P);
    lb = look_up(u0 + 3 * P);
    for (int u = u0; u < units && ok; u += 2 * P) {
      expand(u, xa);
      xa = fetch(u + 2 * P, la);
      la = look_up(u + 4 * P);
      if (!ok || u + P >= units) break;
      expand(u + P, xb);
      xb = fetch(u + 3 * P, lb);
      lb = look_up(u + 5 * P);
    }
  } else {
    // ---------------- softmax and output ----------------
    const int t = (warp - FIRST) >> 2;
    const int quarter = warp & 3;             // TMEM lanes this warp may access
    const int row = quarter * 32 + lane;      // of the query tile
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lane_addr + t * 128;
    const uint32_t o_addr = tmem + lane_addr + 256 + t * 128;
    // (all lanes or none: one that gave up alone would leave the others in a vote)
    auto wait = [&](uint64_t* bar, uint32_t phase) {
      return __all_sync(0xffffffffu, mbar_wait(bar, phase, wait_flag, p.wait_ns));
    };
    const int nkv = t ? n_t[1] : n_t[0];
    int lim;
    float query = 1.f;  // 2^qe
    {
      const int r = row0 + t * kTileRows + row;
      const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(r)));
      lim = seen_end(length, count, tok, p.causal) - j0 * kTcTile;
      if (nkv > 0) {
        // sixteen lanes to a row, two rows at a time: their largest magnitudes (NaN ones aside), then the rows in units
        // of those (exactly, but for what lies 2^-29 below)
        const int half = lane >> 4, c16 = lane & 15;
        constexpr int CHUNKS = D / 8, STEPS = CHUNKS > 16 ? CHUNKS / 16 : 1;  // 16-byte pieces of a row, of a lane
        uint4 x[16][STEPS];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int rr = row0 + t * kTileRows + quarter * 32 + 2 * i + half;
          const int tt = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(rr)));
          const uint4* q = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + b * p.st[2] +
                                                          (h * p.per + (rr - tt * p.per)) * p.st[1] + tt * p.st[0]);
#pragma unroll
          for (int k = 0; k < STEPS; ++k)
            x[i][k] = tt < count && c16 + 16 * k < CHUNKS ? __ldg(q + c16 + 16 * k) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float top = 0.f;
#pragma unroll
          for (int k = 0; k < STEPS; ++k) {
            const uint32_t w[4] = {x[i][k].x, x[i][k].y, x[i][k].z, x[i][k].w};
#pragma unroll
            for (int y = 0; y < 4; ++y)
              top = fmaxf(top, fmaxf(fabsf(half_of<BF16>(w[y], 0)), fabsf(half_of<BF16>(w[y], 1))));
          }
#pragma unroll
          for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const int qe = query_unit(top);
          const float up = pow2(-qe);
          const int mine = __shfl_sync(0xffffffffu, qe, (lane & 1) * 16);
          if (lane >> 1 == i) query = pow2(mine);
          const int rw = quarter * 32 + 2 * i + half;
#pragma unroll
          for (int k = 0; k < STEPS; ++k) {
            uint32_t w[4] = {x[i][k].x, x[i][k].y, x[i][k].z, x[i][k].w};
#pragma unroll
            for (int y = 0; y < 4; ++y) w[y] = pack2<false>(half_of<BF16>(w[y], 0) * up, half_of<BF16>(w[y], 1) * up);
            const int ch = c16 + 16 * k;
            if (ch >= CHUNKS) continue;
            const uint32_t at = smem_u32(sQ + t * S::TILE_BYTES) + rw * 128 + (ch >> 3) * S::HALF_BYTES + (((ch & 7) ^ (rw & 7)) << 4);
            if constexpr (DENSE)
              store_shared16(at, w[0], w[1], w[2], w[3]);
            else
              store_shared16(at, __byte_perm(w[0], w[2], 0x5410), __byte_perm(w[0], w[2], 0x7632), __byte_perm(w[1], w[3], 0x5410),
                             __byte_perm(w[1], w[3], 0x7632));
          }
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[t]);
      }
    }
    float m_ref = kTcFloor, l = 0.f;
    for (int j = 0; j < nkv && ok; ++j) {
      // the tile's units: there long before its scores
      if (!wait(&u_full[j & (kUnits - 1)], (j / kUnits) & 1)) { ok = false; break; }
      const uint32_t units = smem_u32(&s_units[j & (kUnits - 1)]);
      {
        uint32_t bad[2];
        load_words<2>(units + 48, bad);
        if (bad[0] | bad[1]) s_odd[t] = 1;
      }
      const Row<NU> ru = row_units<NU>(p.scale_log2, query, units);
      if (!wait(&s_full[t], j & 1)) { ok = false; break; }
      fence_after_sync();
      uint32_t raw[128];
#pragma unroll
      for (int k = 0; k < 4; ++k) tmem_ld32(s_addr + k * 32, raw + k * 32);
      tmem_ld_wait();
      if (lim < kTcTile) {  // (lim: keys that the row sees, from this tile's first on)
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i >= lim) raw[i] = __float_as_uint(-INFINITY);
      }
      float tile_sum;
      bool rescale = false;
      float alpha = 1.f;
      if (j == 0) {
        m_ref = fmaxf(largest<NU>(raw, ru) - kTcUnder, kTcFloor);
        tile_sum = weights<NU>(raw, ru, m_ref, units, s_addr);
      } else {
        // weights against the running maximum while this tile's is reduced, redone if it grew too far
        tile_sum = weights<NU>(raw, ru, m_ref, units, s_addr);
        const float m_tile = largest<NU>(raw, ru) - kTcUnder;
        if (m_tile > m_ref + (kTcMost - kTcUnder)) {
          alpha = ex2(m_ref - m_tile);
          m_ref = m_tile;
          rescale = true;
        }
      }
      if (__any_sync(0xffffffffu, rescale)) {
        tmem_st_wait();
        tile_sum = weights<NU>(raw, ru, m_ref, units, s_addr);
        if (!wait(&o_done[t], (j - 1) & 1)) ok = false;
        fence_after_sync();
        if (ok) {
#pragma unroll
          for (int k = 0; k < D / 32; ++k) {
            uint32_t o[32];
            tmem_ld32(o_addr + k * 32, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(o_addr + k * 32, o);
          }
        }
      }
      l = fmaf(l, alpha, tile_sum);
      lim -= kTcTile;
      tmem_st_wait();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
    }
    if (ok && nkv > 0 && !wait(&o_done[t], (nkv - 1) & 1)) ok = false;
    fence_after_sync();
    if (ok) {
      // (where the row lies is worked out again: the loop has no registers to keep it in)
      int again = row;
      asm volatile("" : "+r"(again));
      const int r = row0 + t * kTileRows + again;
      const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(r)));
      const int head = h * p.per + (r - tok * p.per);
      const int end = seen_end(length, count, tok, p.causal);
      if (!DENSE && end > *reinterpret_cast<volatile int*>(s_poison)) l = __int_as_float(0x7fc00000);
      const bool live = nkv > 0 && end > 0;
      const bool split_up = p.splits > 1;
      const float inv = !live || l == 0.f ? 0.f : 1.f / l;
      const int64_t at = (static_cast<int64_t>(bh) * p.blocks + rb) * p.splits + split;
      float* part = split_up ? p.part + (at * S::ROWS + t * kTileRows + row) * D : nullptr;
      T* out = static_cast<T*>(p.o) + ((static_cast<int64_t>(b) * p.heads + head) * p.tokens + tok) * D;
      const bool mine = tok < p.tokens;
      if (split_up && mine) {
        float* ml = p.part_ml + (at * S::ROWS + t * kTileRows + row) * 2;
        ml[0] = live ? m_ref : kTcFloor;
        ml[1] = live ? l : 0.f;
      }
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        uint32_t o[32];
        if (nkv > 0) {  // (uniform in the warp)
          tmem_ld32(o_addr + k * 32, o);
          tmem_ld_wait();
        }
        if (!live) {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0;
        }
        if (!mine) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float f[8];
#pragma unroll
          for (int x = 0; x < 8; ++x)  // packed tiles: head dimensions 0 4 1 5 2 6 3 7 of eight
            f[x] = __uint_as_float(o[8 * i + (DENSE ? x : 2 * (x & 3) + (x >> 2))]);
          if (split_up) {
            float4* dst = reinterpret_cast<float4*>(part + k * 32 + i * 8);
            dst[0] = make_float4(f[0], f[1], f[2], f[3]);
            dst[1] = make_float4(f[4], f[5], f[6], f[7]);
          } else {
#pragma unroll
            for (int x = 0; x < 8; ++x) f[x] *= inv;
            *reinterpret_cast<uint4*>(out + k * 32 + i * 8) = make_uint4(pack2<BF16>(f[0], f[1]), pack2<BF16>(f[2], f[3]),
                                                                         pack2<BF16>(f[4], f[5]), pack2<BF16>(f[6], f[7]));
          }
        }
      }
    }
  }
  if (!ok) atomicExch(wait_flag, PHEW_ERR_TIMEOUT);
  fence_before_sync();
  if (__syncthreads_or(!ok)) {
    // a wait ran out somewhere: let the issued products and loads finish before the TMEM and shared memory go
    if (warp == 0 && lane == 0) {
      commit(drain);
      mbar_wait(drain, 0, nullptr, p.wait_ns);
    } else if (DENSE && warp == 1 && lane == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (k_last[i] >= 0) mbar_wait(&k_full[i], S::phase(k_last[i]), nullptr, p.wait_ns);
        if (v_last[i] >= 0) mbar_wait(&v_full[i], S::phase(v_last[i]), nullptr, p.wait_ns);
      }
      for (int j = max(u_last - kUnits + 1, 0); j <= u_last; ++j)
        mbar_wait(&u_full[j & (kUnits - 1)], (j / kUnits) & 1, nullptr, p.wait_ns);
    }
    fence_before_sync();
    __syncthreads();
  }
  if (warp == 0) {
    fence_after_sync();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (threadIdx.x == 0) p.odd[blockIdx.x] = s_odd[0] | s_odd[1] << 1;
}

// Rows that met keys that f16 does not hold, again, in fp32 from the cache as it lies: a query tile of a CTA of
// attn_tc_kernel to a block, a thread to a row, sixteen keys at a time in shared memory.  Heads of 256 go through the
// keys twice, for half of their values each.
constexpr int kPlainKeys = 16;
template <typename S, bool BF16> __global__ void __launch_bounds__(kTileRows) plain_rows_kernel(const TcParams p) {
  using T = typename std::conditional<BF16, bf16, f16>::type;
  constexpr int D = S::D, DV = D < 128 ? D : 128;
  __shared__ __align__(16) float s_k[kPlainKeys][D], s_v[kPlainKeys][DV];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int t = blockIdx.y;
  if (!(p.odd[blockIdx.x] >> t & 1)) return;
  const Share sh = share_of<S>(p);
  const int r = sh.row0 + t * kTileRows + static_cast<int>(threadIdx.x);
  const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(r)));
  const int head = sh.h * p.per + (r - tok * p.per);
  const int first = sh.j0 * kTcTile, last = min(sh.length, first + (t ? sh.n_t[1] : sh.n_t[0]) * kTcTile);
  const int end = min(seen_end(sh.length, sh.count, tok, p.causal), last);  // 0 for a row without a query
  const T* q = static_cast<const T*>(p.q) + sh.b * p.st[2] + head * p.st[1] + tok * p.st[0];
  float top = 0.f;
  if (end > 0)
    for (int d = 0; d < D; ++d) top = fmaxf(top, fabsf(to_f32(q[d])));
  const int qe = query_unit(top);
  const float up = pow2(-qe);  // (qe is -121 .. 114)
  const int ng = D / p.c.group;
  for (int d0 = 0; d0 < D; d0 += DV) {
    float o[DV], m = kTcFloor, l = 0.f;
#pragma unroll
    for (int d = 0; d < DV; ++d) o[d] = 0.f;
    for (int key0 = first; key0 < last; key0 += kPlainKeys) {
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * kPlainKeys * (D / 8); i += kTileRows) {
        const int side = i / (kPlainKeys * (D / 8)), k = i / (D / 8) % kPlainKeys, w = i % (D / 8);
        if (side && (w * 8 < d0 || w * 8 >= d0 + DV)) continue;
        const uint32_t at = key0 + k < last ? row_of(p.c.map, sh.b, sh.h, key0 + k) : kNoRow;
        uint32_t word = 0;
        float sc = 0.f, bi = 0.f;  // (a bad page's: zeros; it is reported already)
        if (at != kNoRow) {
          const int64_t g = static_cast<int64_t>(at) * ng + w * 8 / p.c.group;
          word = p.c.codes[side][static_cast<int64_t>(at) * (D / 8) + w];
          sc = to_f32(static_cast<const T*>(p.c.scales[side])[g]);
          bi = to_f32(static_cast<const T*>(p.c.biases[side])[g]);
        }
        float* dst = side ? &s_v[k][w * 8 - d0] : &s_k[k][w * 8];
        // (keys times 2^-24: with a query of 2^15 the largest stay in range)
        const float by = side ? 1.f : 0x1p-24f;
        for (int x = 0; x < 8; ++x) dst[x] = fmaf(sc * by, static_cast<float>(word >> (4 * x) & 15), bi * by);
      }
      __syncthreads();
      if (key0 >= end) continue;
      float s[kPlainKeys];
#pragma unroll
      for (int k = 0; k < kPlainKeys; ++k) s[k] = 0.f;
      for (int d = 0; d < D; d += 4) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = to_f32(q[d + i]) * up;
#pragma unroll
        for (int k = 0; k < kPlainKeys; ++k) {
          const float4 y = *reinterpret_cast<const float4*>(&s_k[k][d]);
          s[k] = fmaf(x[0], y.x, fmaf(x[1], y.y, fmaf(x[2], y.z, fmaf(x[3], y.w, s[k]))));
        }
      }
#pragma unroll
      for (int k = 0; k < kPlainKeys; ++k) {
        if (key0 + k >= end) break;
        const float x = s[k] * (p.scale_log2 * 0x1p24f) * pow2(qe);
        const float m_new = fmaxf(m, x), was = ex2(m - m_new), w = ex2(x - m_new);
        m = m_new;
        l = fmaf(l, was, w);
#pragma unroll
        for (int d = 0; d < DV; d += 4) {
          const float4 y = *reinterpret_cast<const float4*>(&s_v[k][d]);
          o[d] = fmaf(w, y.x, o[d] * was);
          o[d + 1] = fmaf(w, y.y, o[d + 1] * was);
          o[d + 2] = fmaf(w, y.z, o[d + 2] * was);
          o[d + 3] = fmaf(w, y.w, o[d + 3] * was);
        }
      }
    }
    if (end <= first) continue;
    const int64_t slot = ((static_cast<int64_t>(sh.bh) * p.blocks + sh.rb) * p.splits + sh.split) * S::ROWS + t * kTileRows + threadIdx.x;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (p.splits > 1) {
      float* part = p.part + slot * D + d0;
#pragma unroll
      for (int d = 0; d < DV; ++d) part[d] = o[d];
      p.part_ml[slot * 2] = m;
      p.part_ml[slot * 2 + 1] = l;
    } else {
      T* out = static_cast<T*>(p.o) + ((static_cast<int64_t>(sh.b) * p.heads + head) * p.tokens + tok) * D + d0;
#pragma unroll
      for (int d = 0; d < DV; ++d) out[d] = from_f32<T>(o[d] * inv);
    }
  }
}

// Joins the splits of a row: one warp per row, splits in their order.
template <typename S, bool BF16>
__global__ void __launch_bounds__(256) combine_tc_kernel(const TcParams p) {
  constexpr int D = S::D, ROWS = S::ROWS;
  using T = typename std::conditional<BF16, bf16, f16>::type;
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t slot = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);  // (bh, block, row)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int row = static_cast<int>(slot % ROWS);
  const int64_t seg = slot / ROWS;
  const int rb = static_cast<int>(seg % p.blocks);
  const int bh = static_cast<int>(seg / p.blocks);
  const int r = rb * ROWS + row;
  const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(r)));
  if (tok >= p.tokens) return;
  const int b = bh / p.c.map.kv_heads, head = (bh % p.c.map.kv_heads) * p.per + (r - tok * p.per);
  float m = kTcFloor;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.part_ml[((seg * p.splits + s) * ROWS + row) * 2]);
  float o[E], l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const int64_t at = (seg * p.splits + s) * ROWS + row;
    const float f = ex2(p.part_ml[at * 2] - m);
    l = fmaf(f, p.part_ml[at * 2 + 1], l);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = fmaf(f, p.part[at * D + i * 32 + lane], o[i]);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* out = static_cast<T*>(p.o) + ((static_cast<int64_t>(b) * p.heads + head) * p.tokens + tok) * D;
#pragma unroll
  for (int i = 0; i < E; ++i) out[i * 32 + lane] = from_f32<T>(o[i] * inv);
}

struct ExpandParams {
  Cache c;
  void* dense[2];  // [batch * kv_heads][rows][D] f16
  Units* units;    // [batch * kv_heads][rows / 128]
  const int32_t* lengths;
  FastDiv by_tiles, by_heads;  // tiles of a head, heads
  int* error_flag;
};

// The dense form's keys and values, a tile and a side to a block: written up to a sequence's last tile, zero behind its
// last key.  A weight of zero would make a NaN of an infinity, so a key whose value's scale or bias is not finite gets
// zero for a value and NaN for a key: rows that see it get one through their score.
// Bound by HBM and latencies: two prompts of 4096 tokens on 32 heads of 128, 38 MB read and 134 MB written in 31 us.
// Launched so that a programmatic dependent may be set up meanwhile.
template <int D> constexpr int kExpandThreads = D <= 128 ? 128 : 256;
template <typename T, int D> __global__ void __launch_bounds__(kExpandThreads<D>) expand_kernel(const ExpandParams p) {
  asm volatile("griddepcontrol.launch_dependents;");
  constexpr int THREADS = kExpandThreads<D>, WORDS = D / 8;  // words of eight codes to a row
  constexpr int W = kTcTile * WORDS / THREADS;               // to a thread
  __shared__ uint32_t s_row[kTcTile];
  __shared__ Reach s_reach[kTcTile / 32];
  __shared__ float2 s_affine[kTcTile][D / 32];  // scale and bias of a key's groups
  const int side = blockIdx.y, tid = threadIdx.x;
  const uint32_t bh = div_by(p.by_tiles, blockIdx.x);
  const int tile = static_cast<int>(blockIdx.x - bh * p.by_tiles.d);
  const int b = static_cast<int>(div_by(p.by_heads, bh)), h = static_cast<int>(bh - b * p.by_heads.d);
  const int length = __ldg(p.lengths + b);
  if (tile * kTcTile >= length) return;
  const int ng = D / p.c.group, shift = p.c.group == 32 ? 2 : p.c.group == 64 ? 3 : 4;  // words to a group: 2^shift
  if (tid < kTcTile) {
    const int key = tile * kTcTile + tid;
    uint32_t at = kNoRow;
    if (key < length) {
      at = row_of(p.c.map, b, h, key);
      if (at == kNoRow) atomicExch(p.error_flag, PHEW_ERR_INVALID);
    }
    s_row[tid] = at;
    Reach reach;
#pragma unroll 4
    for (int g = 0; g < ng; ++g) {
      float2 a = make_float2(0.f, 0.f);
      if (at != kNoRow) {
        const int64_t i = static_cast<int64_t>(at) * ng + g;
        const float vs = to_f32(static_cast<const T*>(p.c.scales[1])[i]), vz = to_f32(static_cast<const T*>(p.c.biases[1])[i]);
        if (finite(vs) && finite(vz))
          a = side ? make_float2(vs, vz)
                   : make_float2(to_f32(static_cast<const T*>(p.c.scales[0])[i]), to_f32(static_cast<const T*>(p.c.biases[0])[i]));
        else
          a.y = side ? 0.f : __int_as_float(0x7fc00000);
      }
      s_affine[tid][g] = a;
      reach.add(a.x, a.y);
    }
    reach.done();
    reach.across_warp();
    if (tid % 32 == 0) s_reach[tid / 32] = reach;
  }
  __syncthreads();
  uint32_t word[W];
#pragma unroll
  for (int u = 0; u < W; ++u) {
    const int i = u * THREADS + tid;
    const uint32_t at = s_row[i / WORDS];
    word[u] = at == kNoRow ? 0 : __ldg(p.c.codes[side] + static_cast<int64_t>(at) * WORDS + i % WORDS);
  }
  Reach reach = s_reach[0];
#pragma unroll
  for (int i = 1; i < kTcTile / 32; ++i) {
    reach.far = max(reach.far, s_reach[i].far);
    reach.key = min(reach.key, s_reach[i].key);
    reach.group = min(reach.group, s_reach[i].group);
  }
  const int unit = reach.unit();
  if (tid == 0) set_units<1>(p.units + blockIdx.x, side, 0, unit, reach.odd(side, -14));
  const float down = pow2(-unit);
  uint4* dst = static_cast<uint4*>(p.dense[side]) + static_cast<int64_t>(blockIdx.x) * (kTcTile * WORDS) + tid;
#pragma unroll
  for (int u = 0; u < W; ++u) {
    const int w = u * THREADS + tid;
    const float2 a = s_affine[w / WORDS][w % WORDS >> shift];
    const uint64_t s2 = f2(a.x * down, a.x * down), z2 = f2(a.y * down, a.y * down);
    // a code as a float: a byte of it under 2^23
    constexpr uint32_t base = 0x4B000000u;
    const uint32_t even = word[u] & 0x0f0f0f0fu, other = (word[u] >> 4) & 0x0f0f0f0fu;
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t n = add2(f2(__uint_as_float(__byte_perm(even, base, 0x7540 + i)), __uint_as_float(__byte_perm(other, base, 0x7540 + i))),
                              f2(-8388608.f, -8388608.f));
      const uint64_t x = fma2(s2, n, z2);
      v[i] = pack2<false>(lo_of(x), hi_of(x));
    }
    dst[u * THREADS] = make_uint4(v[0], v[1], v[2], v[3]);
  }
}

template <typename T> int launch_expand(const ExpandParams& p, unsigned tiles, cudaStream_t st) {
  const dim3 grid(tiles, 2);
  switch (p.c.head_dim) {
    case 64: expand_kernel<T, 64><<<grid, kExpandThreads<64>, 0, st>>>(p); break;
    case 128: expand_kernel<T, 128><<<grid, kExpandThreads<128>, 0, st>>>(p); break;
    default: expand_kernel<T, 256><<<grid, kExpandThreads<256>, 0, st>>>(p); break;
  }
  return launch_status("kv expand_kernel");
}

// CTAs of a call, how many ways each row block's keys are split (enough to give
// every SM a CTA, two tiles of the longest possible sequence or more each), and
// whether the cache is expanded first.
// Query rows to a cache head above which the kernel is taken: up to there the mma.sync kernel's passes of 16 rows
// (8 of heads of 256) over the cache cost less than a tile of 128 that is mostly empty.  Measured, mma.sync against
// this kernel, 8 cache heads of 8192 keys / 16 x 8 of 2048 / 8 of 65536: at 48 rows 24 : 34, 54 : 60, 87 : 114 us,
// at 64 rows 26 : 34, 66 : 60, 110 : 114, at 96 rows 33 : 34, 91 : 61, 156 : 115.  Heads of 256, 8 of 8192 keys /
// 8 x 8 of 2048: at 64 rows 45 : 55, 78 : 78, at 96 rows 59 : 55, 109 : 79.
constexpr int64_t kTcAbove = 64;
// Row blocks from which one expansion beats one per CTA.  Expanded against packed, the same three caches: 1 block
// 37 : 38, 75 : 65, 138 : 133 us, 2 blocks 44 : 48, 117 : 127, 190 : 226, 3 blocks 50 : 61, 158 : 194, 248 : 322.
// Heads of 256 are always expanded.
constexpr int64_t kExpandBlocks = 2;
// Scratch that a call may take for it, a bound on memory and not on time.  Beyond, packed against expanded, 8 sequences of
// 8 heads of 128 behind tables for 65536 tokens (2 GiB), 2048 rows: 65536 keys each 6880 : 4643 us, 8192 869 : 641,
// 2048 243 : 252; heads of 256 behind 32768 tokens, on the mma.sync kernel: 32768 keys 32349 : 5345, 2048 2163 : 416.
constexpr int64_t kExpandBytes = int64_t(1) << 30;

int rows_of(int head_dim) { return head_dim <= 128 ? TcShape<128, 128>::ROWS : TcShape<256, 128>::ROWS; }

struct TcPlan {
  int64_t blocks, splits, ctas;
  int64_t rows;  // token rows of a cache head in the expanded cache; 0: packed
  size_t part_bytes, side_bytes, unit_bytes;
};
TcPlan tc_plan(int64_t batch, int kv_heads, int head_dim, int64_t q_rows, int64_t cap) {
  TcPlan t;
  const int rows = rows_of(head_dim);
  t.blocks = (q_rows + rows - 1) / rows;
  const int64_t base = batch * kv_heads * t.blocks, sms = sm_count_current();
  const int64_t tiles = (cap + kTcTile - 1) / kTcTile;
  t.splits = base >= sms ? 1 : sms / base;
  if (t.splits > tiles / 2) t.splits = tiles / 2;
  if (t.splits < 1) t.splits = 1;
  t.ctas = base * t.splits;
  t.part_bytes = t.splits == 1 ? 0 : static_cast<size_t>(t.ctas) * rows * (static_cast<size_t>(head_dim) + 2) * 4;
  t.rows = tiles * kTcTile;
  t.side_bytes = static_cast<size_t>(batch) * kv_heads * t.rows * head_dim * 2;
  if ((t.blocks < kExpandBlocks && head_dim <= 128) || static_cast<int64_t>(2 * t.side_bytes) > kExpandBytes ||
      batch * kv_heads * t.rows >= kMaxRows) {
    t.rows = 0;
    t.side_bytes = 0;
  }
  t.unit_bytes = static_cast<size_t>(batch) * kv_heads * (t.rows / kTcTile) * sizeof(Units);
  return t;
}

// [batch * kv_heads * rows][D] of f16; box of 64 columns x 128 rows, 128-byte swizzle.
int dense_map(CUtensorMap* tm, const void* base, int64_t rows, int D) {
  const uint64_t dims[2] = {static_cast<uint64_t>(D), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(D) * 2};
  const uint32_t box[2] = {64, static_cast<uint32_t>(kTcTile)};
  return make_map_16bit(tm, base, false, 2, dims, strides, box);
}

struct Maps {
  CUtensorMap k, v;  // dense
};

template <typename S, bool BF16, bool DENSE>
int launch_tc(const Maps& m, const TcParams& p, unsigned grid, cudaStream_t st) {
  static SmemAllowed allowed;
  if (int s = allow_smem(allowed, attn_tc_kernel<S, BF16, DENSE>, S::SMEM)) return s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(tc_threads(DENSE, S::QT));
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = DENSE ? 1 : 0;  // set up while the cache is expanded
  PHEW_CHECK_CUDA(cudaLaunchKernelEx(&cfg, attn_tc_kernel<S, BF16, DENSE>, m.k, m.v, p));
  if (int s = launch_status("kv attn_tc_kernel")) return s;
  cfg = {};
  cfg.gridDim = dim3(grid, S::QT);
  cfg.blockDim = dim3(kTileRows);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PHEW_CHECK_CUDA(cudaLaunchKernelEx(&cfg, plain_rows_kernel<S, BF16>, p));
  if (int s = launch_status("kv plain_rows_kernel")) return s;
  if (p.splits == 1) return PHEW_OK;
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(p.batch) * p.c.map.kv_heads * p.blocks * (S::ROWS / 8)));
  cfg.blockDim = dim3(256);
  PHEW_CHECK_CUDA(cudaLaunchKernelEx(&cfg, combine_tc_kernel<S, BF16>, p));
  return launch_status("kv combine_tc_kernel");
}

template <bool BF16>
int dispatch_tc(const Maps& m, const TcParams& p, unsigned grid, cudaStream_t st) {
  if (p.rows) {  // (the group no longer matters)
    if (p.c.head_dim == 64) return launch_tc<TcShape<64, 64>, BF16, true>(m, p, grid, st);
    if (p.c.head_dim == 128) return launch_tc<TcShape<128, 128>, BF16, true>(m, p, grid, st);
    return launch_tc<TcShape<256, 128>, BF16, true>(m, p, grid, st);
  }
  if (p.c.head_dim == 64)
    return p.c.group == 32 ? launch_tc<TcShape<64, 32>, BF16, false>(m, p, grid, st)
                           : launch_tc<TcShape<64, 64>, BF16, false>(m, p, grid, st);
  if (p.c.group == 32) return launch_tc<TcShape<128, 32>, BF16, false>(m, p, grid, st);
  if (p.c.group == 64) return launch_tc<TcShape<128, 64>, BF16, false>(m, p, grid, st);
  return launch_tc<TcShape<128, 128>, BF16, false>(m, p, grid, st);
}

}  // namespace

bool takes_tc(int64_t batch, int kv_heads, int head_dim, int dtype, int64_t rows, int64_t cap) {
  if (dtype == PHEW_F32) return false;
  return rows > kTcAbove && (head_dim <= 128 || tc_plan(batch, kv_heads, head_dim, rows, cap).rows > 0);
}

size_t tc_bytes(int64_t batch, int kv_heads, int head_dim, int64_t rows, int64_t cap) {
  const TcPlan t = tc_plan(batch, kv_heads, head_dim, rows, cap);
  return 2 * t.side_bytes + t.unit_bytes + t.part_bytes + (static_cast<size_t>(t.ctas) * 4 + 15) / 16 * 16;
}

int run_attn_tc(const AttnParams& a, bool bf16_type, void* workspace, cudaStream_t st) {
  const int D = a.c.head_dim;
  const TcPlan t = tc_plan(a.batch, a.c.map.kv_heads, D, static_cast<int64_t>(a.tokens) * a.per, capacity(a.c.map));
  PHEW_REQUIRE(t.ctas < (1ll << 31) / 32, "phew_kv_attention: too many query rows");
  TcParams p;
  p.c = a.c;
  p.q = a.q;
  for (int i = 0; i < 3; ++i) p.st[i] = a.st[i];
  p.o = a.o;
  p.lengths = a.lengths;
  p.counts = a.counts;
  p.batch = a.batch;
  p.heads = a.heads;
  p.tokens = a.tokens;
  p.per = a.per;
  p.blocks = static_cast<int>(t.blocks);
  p.splits = static_cast<int>(t.splits);
  p.rows = static_cast<int>(t.rows);
  p.by_per = a.by_per;
  p.scale_log2 = a.scale_log2;
  p.causal = a.causal;
  char* scratch = static_cast<char*>(workspace);
  Maps m = {};
  p.units = nullptr;
  if (t.rows) {
    const int64_t rows = static_cast<int64_t>(a.batch) * a.c.map.kv_heads * t.rows;
    if (int s = dense_map(&m.k, scratch, rows, D)) return s;
    if (int s = dense_map(&m.v, scratch + t.side_bytes, rows, D)) return s;
    ExpandParams e;
    e.c = a.c;
    e.dense[0] = scratch;
    e.dense[1] = scratch + t.side_bytes;
    p.units = e.units = reinterpret_cast<Units*>(scratch + 2 * t.side_bytes);
    e.lengths = a.lengths;
    e.by_tiles = fast_div(static_cast<uint32_t>(t.rows / kTcTile));
    e.by_heads = fast_div(static_cast<uint32_t>(a.c.map.kv_heads));
    e.error_flag = a.error_flag;
    const unsigned tiles = static_cast<unsigned>(rows / kTcTile);
    if (int s = bf16_type ? launch_expand<bf16>(e, tiles, st) : launch_expand<f16>(e, tiles, st)) return s;
  }
  p.part = reinterpret_cast<float*>(scratch + 2 * t.side_bytes + t.unit_bytes);
  p.part_ml = p.part + static_cast<size_t>(t.ctas) * rows_of(D) * D;
  p.odd = reinterpret_cast<int*>(scratch + 2 * t.side_bytes + t.unit_bytes + t.part_bytes);
  p.error_flag = a.error_flag;
  const tc::TestStall stall = tc::take_test_stall();
  p.wait_ns = stall.wait_ns;
  p.withhold = stall.withhold;
  const unsigned grid = static_cast<unsigned>(t.ctas);
  return bf16_type ? dispatch_tc<true>(m, p, grid, st) : dispatch_tc<false>(m, p, grid, st);
}

}  // namespace kv
}  // namespace phew
