// Attention of many query rows over a 4-bit cache (chunks of a prompt), on the
// tcgen05 tensor cores.
//
// The rows of a cache head are r = token * per + head over its `per` query
// heads; a CTA takes 256 of them (two 128-row tiles a and b) and walks the
// keys in tiles of 128.  Bound by the chain score product - softmax - output
// product of each tile, at about the rate of the exponentials.  Two forms:
//
// Dense (kExpandBlocks row blocks or more, whose every CTA would expand the
// same keys again): the cache is expanded once to 16 bits in scratch, as
// phew_kv_fetch does, and tiles arrive by TMA.  One pass of HBM over the keys
// against 0.5 us for each CTA and tile (measured: 256 CTAs x 56 tiles).
//
// Packed (few row blocks): producer warps load packed rows (two units of 32
// keys ahead, in registers), expand them as T(scale * code + bias) - two
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
//                 load Q and write O
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
// Keys and values are rounded to the type, as mx.dequantize gives them, and so
// are the softmax weights, as in the dense attention: what the tensor core
// takes.  Together 3.2e-3 to 3.7e-3 of an output's norm in bf16 (1.7e-3 is its
// own rounding), 4e-4 in f16 (2.1e-4).  Scores, maxima and sums are 32-bit.
//
// Measured, causal, heads of 128 in bf16: two prompts of 4096 tokens on 32
// heads, 334 us (823 TFLOP/s); the last 2048 of 8192 tokens on 32 heads over 8,
// 248 us (970 TFLOP/s).
//
// Every wait is bounded; one that runs out sets error_flag[1] and the CTA
// winds down with its TMEM freed.
#include "attn_softmax.cuh"
#include "kv_attn_tc.cuh"

namespace phew {
namespace kv {
namespace {

using namespace tc;
using attn::compute_p;
using attn::ex2;
using attn::pack2;
using attn::row_max;

constexpr int kTileRows = 128;
constexpr int kTcTile = 128;       // keys of a tile
constexpr int kProducers = 3;      // warps 1 .. 3 of the packed form
constexpr int kTmemCols = 512;
constexpr float kTcFloor = -1.0e38f;
constexpr float kTcGrow = 8.0f;    // log2 units: the running maximum moves when a tile passes it by more

template <int D_, int G_> struct TcShape {
  static constexpr int D = D_, G = G_, NG = D / G;
  static constexpr int HALVES = D / 64;
  static constexpr int HALF_BYTES = kTcTile * 128;           // 64 columns of 16 bits, 128-byte rows
  static constexpr int TILE_BYTES = HALF_BYTES * HALVES;
  static constexpr int QT = D <= 128 ? 2 : 1;                // query tiles of a CTA
  static constexpr int ROWS = QT * kTileRows;
  static constexpr int RING = D <= 128 ? 2 : 1;              // tiles of K, and of V, in flight
  static constexpr int SMEM = (QT + 2 * RING) * TILE_BYTES + 1024 + 256;
  // slot and phase of key tile j in the rings
  static __device__ __forceinline__ int slot(int j) { return RING == 2 ? j & 1 : 0; }
  static __device__ __forceinline__ uint32_t phase(int j) { return (RING == 2 ? j >> 1 : j) & 1; }
};

constexpr int tc_threads(bool dense, int tiles) { return 32 * ((dense ? 2 : 1 + kProducers) + 4 * tiles); }

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
  bool q_tma;  // dense: tiles of queries arrive by TMA too
  FastDiv by_per;
  float scale_log2;  // > 0
  bool causal;
  float* part;     // [segment][split][256][D] when splits > 1
  float* part_ml;  // [segment][split][256][2]
  int* error_flag;
  unsigned long long wait_ns;
  int withhold;  // test hook: the V tile of this key tile is never announced (-1: none)
};

// code pairs (U, U + 4) of a word as 16-bit floats, exactly
template <bool BF16, int U> __device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  uint32_t d, x;
  if constexpr (BF16) {
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(x) : "r"(w >> (4 * U)), "r"(0x000f000fu), "r"(0x43004300u));
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0x43004300u));  // 128 + n - 128
  } else {
    const uint32_t y = U == 0 ? w << 4 : w >> (U == 0 ? 0 : 4 * U - 4);
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(x) : "r"(y), "r"(0x00f000f0u), "r"(0x54005400u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(0x54005400u));  // 64 + n - 64
  }
  return d;
}
template <bool BF16> __device__ __forceinline__ uint32_t fma_pair(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  if constexpr (BF16)
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ bool finite16(uint32_t bits, bool bf16) {
  const uint32_t e = bf16 ? 0x7f80u : 0x7c00u;
  return (bits & e) != e;
}
__device__ __forceinline__ void store_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// shared-memory writes of this thread become visible to the tensor core
__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <typename S, bool BF16, bool DENSE>
__global__ void __launch_bounds__(tc_threads(DENSE, S::QT), 1)
    attn_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const TcParams p) {
  constexpr int D = S::D, NG = S::NG;
  constexpr int FIRST = DENSE ? 2 : 1 + kProducers;  // softmax warp
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
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 17);
  int* s_poison = reinterpret_cast<int*>(tmem_slot + 1);  // first key whose values are not finite
  int* wait_flag = p.error_flag + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // ---- which rows and which keys ----
  // Cache heads in groups of 16, so that the CTAs running at one time share few heads' keys in the L2; within a
  // group row blocks from the last (the longest under a causal mask) down, a block's heads and splits together.
  const int kv_heads = p.c.map.kv_heads;
  const int all_heads = p.batch * kv_heads, in_group = 16 * p.blocks * p.splits;
  const int group = static_cast<int>(blockIdx.x) / in_group, rem = static_cast<int>(blockIdx.x) % in_group;
  const int wide = min(16, all_heads - 16 * group) * p.splits;
  const int rb = p.blocks - 1 - rem / wide;
  const int split = rem % wide % p.splits, bh = 16 * group + rem % wide / p.splits;
  const int b = bh / kv_heads, h = bh % kv_heads;
  const int count = p.counts ? clamp_count(__ldg(p.counts + b), p.tokens) : p.tokens;
  const int length = clamp_count(__ldg(p.lengths + b), capacity(p.c.map));
  if (threadIdx.x == 0 && length != __ldg(p.lengths + b)) atomicExch(p.error_flag, PHEW_ERR_INVALID);
  const int row0 = rb * S::ROWS;
  // key tiles that each query tile needs, and this CTA's share of them
  int need[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int first = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(row0 + t * kTileRows)));
    const int last = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(row0 + t * kTileRows + kTileRows - 1)));
    const int end = first >= count ? 0 : seen_end(length, count, last < count ? last : count - 1, p.causal);
    need[t] = t < S::QT ? (end + kTcTile - 1) / kTcTile : 0;
  }
  const int all = max(need[0], need[1]);
  const int j0 = static_cast<int>(static_cast<int64_t>(all) * split / p.splits);
  const int n_max = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / p.splits) - j0;
  const int n_t[2] = {min(max(need[0] - j0, 0), n_max), min(max(need[1] - j0, 0), n_max)};

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], DENSE && p.q_tma ? 1 : 4);
      mbar_init(&k_full[i], DENSE ? 1 : 4);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], DENSE ? 1 : 4);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(drain, 1);
    *s_poison = 0x7fffffff;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (DENSE && p.q_tma) {
      // rows token * per + head: boxes of `per` heads x 128 / per tokens
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (n_t[t] > 0) {
          mbar_expect_tx(&q_full[t], S::TILE_BYTES);
          const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(row0 + t * kTileRows)));
#pragma unroll
          for (int i = 0; i < S::HALVES; ++i)
            tma_load_4d(sQ + t * S::TILE_BYTES + i * S::HALF_BYTES, &tm_q, &q_full[t], i * 64, h * p.per, tok, b);
        }
    }
  }
  if (warp == 0) tmem_alloc(tmem_slot, kTmemCols);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  int k_last[2] = {-1, -1}, v_last[2] = {-1, -1};  // dense: the key tile whose load each ring slot received last

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t id_qk = instr_desc_f16(BF16 ? 1 : 0, 0, kTileRows, kTcTile);
      constexpr uint32_t id_pv = instr_desc_f16(BF16 ? 1 : 0, 1, kTileRows, D);
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
      uint32_t sc[NG], bi[NG];  // each twice in a register
      bool fine = true, past = false;  // parts finite; values past the type's range (held at its end)
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        sc[g] = __byte_perm(x.sb[0][g / 2], 0, g & 1 ? 0x3232 : 0x1010);
        bi[g] = __byte_perm(x.sb[1][g / 2], 0, g & 1 ? 0x3232 : 0x1010);
        fine = fine && finite16(sc[g], BF16) && finite16(bi[g], BF16);
        past = past || !finite16(fma_pair<BF16>(sc[g], BF16 ? 0x41704170u : 0x4b804b80u, bi[g]), BF16);  // code 15
      }
      past = past && fine;
      if (side == 1 && !fine) {
        // a weight of zero times infinity is no number, and a later query's keys may not touch an earlier
        // one: the values count as zero here and as "no number" for every row that sees the key
        atomicMin(s_poison, (j0 + j) * kTcTile + row);
#pragma unroll
        for (int g = 0; g < NG; ++g) sc[g] = bi[g] = 0;
      }
      uint64_t* full = side == 0 ? &k_full[slot] : &v_full[slot];
      uint64_t* empty = side == 0 ? &k_empty[slot] : &v_empty[slot];
      if (lane == 0 && !mbar_wait(empty, S::phase(j) ^ 1, wait_flag, p.wait_ns)) ok = false;
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok) return;
      const uint32_t dst = smem_u32((side == 0 ? sK : sV) + slot * S::TILE_BYTES) + row * 128;
      const bool any_past = __any_sync(0xffffffffu, past);
#pragma unroll
      for (int ch = 0; ch < D / 32; ++ch) {
        const uint32_t word[4] = {x.code[ch].x, x.code[ch].y, x.code[ch].z, x.code[ch].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int g = (ch * 32 + i * 8) / S::G, c16 = ch * 4 + i;
          uint32_t v[4] = {fma_pair<BF16>(sc[g], code_pair<BF16, 0>(word[i]), bi[g]),
                           fma_pair<BF16>(sc[g], code_pair<BF16, 1>(word[i]), bi[g]),
                           fma_pair<BF16>(sc[g], code_pair<BF16, 2>(word[i]), bi[g]),
                           fma_pair<BF16>(sc[g], code_pair<BF16, 3>(word[i]), bi[g])};
          if (any_past)
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = past ? hold_pair<BF16>(v[k]) : v[k];
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
    const float c = p.scale_log2;
    int lim;
    {
      const int r = row0 + t * kTileRows + row;
      const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(r)));
      lim = seen_end(length, count, tok, p.causal) - j0 * kTcTile;
      if (nkv > 0 && !(DENSE && p.q_tma)) {
        const bool have = tok < count;
        const uint4* q = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + b * p.st[2] +
                                                        (h * p.per + (r - tok * p.per)) * p.st[1] + tok * p.st[0]);
        const uint32_t dst = smem_u32(sQ + t * S::TILE_BYTES) + row * 128;
#pragma unroll
        for (int c16 = 0; c16 < D / 8; ++c16) {
          const uint4 x = have ? __ldg(q + c16) : make_uint4(0, 0, 0, 0);
          const uint32_t at = dst + (c16 >> 3) * S::HALF_BYTES + (((c16 & 7) ^ (row & 7)) << 4);
          if constexpr (DENSE)
            store_shared16(at, x.x, x.y, x.z, x.w);
          else
            store_shared16(at, __byte_perm(x.x, x.z, 0x5410), __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410),
                           __byte_perm(x.y, x.w, 0x7632));
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[t]);
      }
    }
    float m_ref = kTcFloor, l = 0.f;
    for (int j = 0; j < nkv && ok; ++j) {
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
        m_ref = fmaxf(row_max(raw) * c, kTcFloor);
        tile_sum = compute_p<BF16>(raw, c, m_ref, s_addr);
      } else {
        // weights against the running maximum while this tile's is reduced, redone if it grew too far
        tile_sum = compute_p<BF16>(raw, c, m_ref, s_addr);
        const float m_tile = row_max(raw) * c;
        if (m_tile > m_ref + kTcGrow) {
          alpha = ex2(m_ref - m_tile);
          m_ref = m_tile;
          rescale = true;
        }
      }
      if (__any_sync(0xffffffffu, rescale)) {
        tmem_st_wait();
        tile_sum = compute_p<BF16>(raw, c, m_ref, s_addr);
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
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (DENSE && p.q_tma && n_t[t] > 0) mbar_wait(&q_full[t], 0, nullptr, p.wait_ns);
      commit(drain);
      mbar_wait(drain, 0, nullptr, p.wait_ns);
    } else if (DENSE && warp == 1 && lane == 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (k_last[i] >= 0) mbar_wait(&k_full[i], S::phase(k_last[i]), nullptr, p.wait_ns);
        if (v_last[i] >= 0) mbar_wait(&v_full[i], S::phase(v_last[i]), nullptr, p.wait_ns);
      }
    }
    fence_before_sync();
    __syncthreads();
  }
  if (warp == 0) {
    fence_after_sync();
    tmem_dealloc(tmem, kTmemCols);
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

// CTAs of a call, how many ways each row block's keys are split (enough to give
// every SM a CTA, two tiles of the longest possible sequence or more each), and
// whether the cache is expanded first.
// Query rows to a cache head above which the kernel is taken: up to there the mma.sync kernel's passes of 16 rows
// (8 of heads of 256) over the cache cost less than a tile of 128 that is mostly empty.  Measured, mma.sync against
// this kernel, 8 cache heads of 8192 keys / 16 x 8 of 2048 / 8 of 65536: at 48 rows 22 : 31, 49 : 57, 81 : 106 us,
// at 64 rows 24 : 31, 61 : 57, 103 : 106, at 96 rows 30 : 32, 84 : 57, 146 : 107.  Heads of 256, 8 of 8192 keys /
// 8 x 8 of 2048: at 64 rows 44 : 55, 77 : 82, at 96 rows 58 : 56, 105 : 84.
constexpr int64_t kTcAbove = 64;
// Row blocks from which one expansion beats one per CTA.  Expanded against packed, the same three caches: 2 blocks
// 44 : 45, 126 : 123, 216 : 209 us, 3 blocks 50 : 56, 162 : 180, 274 : 306, 4 blocks 59 : 69, 198 : 234, 357 : 428.
// Heads of 256 are always expanded.
constexpr int64_t kExpandBlocks = 3;
constexpr int64_t kExpandBytes = int64_t(1) << 30;  // scratch that a call may take for it

int rows_of(int head_dim) { return head_dim <= 128 ? TcShape<128, 128>::ROWS : TcShape<256, 128>::ROWS; }

struct TcPlan {
  int64_t blocks, splits, ctas;
  int64_t rows;  // token rows of a cache head in the expanded cache; 0: packed
  size_t part_bytes, side_bytes;
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
  return t;
}

// [batch * kv_heads * rows][D] of 16-bit values; box of 64 columns x 128 rows, 128-byte swizzle.
int dense_map(CUtensorMap* tm, const void* base, bool bf16_type, int64_t rows, int D) {
  const uint64_t dims[2] = {static_cast<uint64_t>(D), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(D) * 2};
  const uint32_t box[2] = {64, static_cast<uint32_t>(kTcTile)};
  return make_map_16bit(tm, base, bf16_type, 2, dims, strides, box);
}

struct Maps {
  CUtensorMap q, k, v;  // dense
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
  PHEW_CHECK_CUDA(cudaLaunchKernelEx(&cfg, attn_tc_kernel<S, BF16, DENSE>, m.q, m.k, m.v, p));
  if (int s = launch_status("kv attn_tc_kernel")) return s;
  if (p.splits == 1) return PHEW_OK;
  cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(p.batch) * p.c.map.kv_heads * p.blocks * (S::ROWS / 8)));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
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
  return 2 * t.side_bytes + t.part_bytes;
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
  p.q_tma = false;
  if (t.rows) {
    const int64_t rows = static_cast<int64_t>(a.batch) * a.c.map.kv_heads * t.rows;
    if (int s = dense_map(&m.k, scratch, bf16_type, rows, D)) return s;
    if (int s = dense_map(&m.v, scratch + t.side_bytes, bf16_type, rows, D)) return s;
    // tiles of queries are boxes where a tile holds whole tokens and every axis has a stride
    p.q_tma = kTileRows % a.per == 0 && a.st[0] > 0 && a.st[1] > 0 && a.st[2] > 0;
    if (p.q_tma) {
      const uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a.heads), static_cast<uint64_t>(a.tokens),
                                static_cast<uint64_t>(a.batch)};
      const uint64_t strides[3] = {static_cast<uint64_t>(a.st[1]) * 2, static_cast<uint64_t>(a.st[0]) * 2,
                                   static_cast<uint64_t>(a.st[2]) * 2};
      const uint32_t box[4] = {64, static_cast<uint32_t>(a.per), static_cast<uint32_t>(kTileRows / a.per), 1};
      if (int s = make_map_16bit(&m.q, a.q, bf16_type, 4, dims, strides, box)) return s;
    }
    if (int s = expand(a.c, bf16_type, scratch, scratch + t.side_bytes, a.batch, t.rows, a.lengths, a.error_flag, st)) return s;
  }
  p.part = reinterpret_cast<float*>(scratch + 2 * t.side_bytes);
  p.part_ml = p.part + static_cast<size_t>(t.ctas) * rows_of(D) * D;
  p.error_flag = a.error_flag;
  const tc::TestStall stall = tc::take_test_stall();
  p.wait_ns = stall.wait_ns;
  p.withhold = stall.withhold;
  const unsigned grid = static_cast<unsigned>(t.ctas);
  return bf16_type ? dispatch_tc<true>(m, p, grid, st) : dispatch_tc<false>(m, p, grid, st);
}

}  // namespace kv
}  // namespace phew
