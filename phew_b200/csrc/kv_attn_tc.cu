// Attention of many query rows over a 4-bit cache (chunks of a prompt), on the
// tcgen05 tensor cores.
//
// The rows of a cache head are r = token * per + head over its `per` query
// heads; a CTA takes 256 of them (two 128-row tiles a and b) and walks the
// keys in tiles of 128.  Bound by the tensor cores and, at the same rate, by
// the exponentials; the cache is read once per 256 rows.  What the dense kernel
// fetches as 16-bit tiles by TMA is made here from codes: four producer warps
// copy packed rows (cp.async, three half-steps ahead), expand them as
// T(scale * code + bias) - two instructions a value: a shift and a logic
// operation per pair of codes, an exact subtraction, a packed multiply-add -
// and store them in the 128-byte swizzle that the tensor core reads.  That is
// a fifth of the SM's issue slots beside the softmax, so the packed cache
// costs no time over a dense one.
//
//   warps 0-3    warp 0: TMEM owner and MMA issuer: per key tile j and query
//                tile t, O_t += P_t V_j, then S_t = Q_t K_{j+1}^T
//   warps 4-7    producers: warp w expands keys 32 w .. 32 w + 31 of each tile,
//                K_j and V_j in turn, into two-deep rings
//   warps 8-15   softmax of tile a and b, one query row per thread; they also
//                load Q and write O
//
// Registers move from the first two groups to the softmax (40 + 72 + 2 x 200
// = 4 x 128).  TMEM: S_a, S_b, O_a, O_b of 128 columns each.
//
// Within eight neighbouring head dimensions tiles hold them in the order
// 0 4 1 5 2 6 3 7, which is how pairs fall out of a word of codes; queries are
// stored to match and outputs read back through the same order.
//
// Long caches with few rows are split: a CTA takes a share of the key tiles
// and leaves partial sums, joined in a fixed order by the combine kernel.
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
constexpr int kTcRows = 256;       // query rows of a CTA
constexpr int kTcThreads = 512;
constexpr int kTmemCols = 512;
constexpr float kTcFloor = -1.0e38f;
constexpr float kTcGrow = 8.0f;    // log2 units: the running maximum moves when a tile passes it by more

template <int D_, int G_> struct TcShape {
  static constexpr int D = D_, G = G_, NG = D / G;
  static constexpr int HALVES = D / 64;
  static constexpr int HALF_BYTES = kTcTile * 128;           // 64 columns of 16 bits, 128-byte rows
  static constexpr int TILE_BYTES = HALF_BYTES * HALVES;
  static constexpr int SB = NG * 2, SROW = SB < 4 ? 4 : SB;  // a key's scales
  static constexpr int WARP_CODES = 32 * D / 2;              // one warp's share of a side's codes
  static constexpr int WARP_STAGE = WARP_CODES + 2 * 32 * SROW;
  static constexpr int STAGES = 3;
  static constexpr int SMEM = 6 * TILE_BYTES + 4 * STAGES * WARP_STAGE + 1024 + 256;
};

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
  FastDiv by_per;
  float scale_log2;  // > 0
  bool causal;
  float* part;     // [segment][split][256][D] when splits > 1
  float* part_ml;  // [segment][split][256][2]
  int* error_flag;
  unsigned long long wait_ns;
  int withhold;  // test hook: the V tile of this key tile is never announced (-1: none)
};

template <int N> __device__ __forceinline__ void copy16(uint32_t dst, const void* src, int valid) {
  if constexpr (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(valid) : "memory");
}

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

template <typename S, bool BF16>
__global__ void __launch_bounds__(kTcThreads, 1) attn_tc_kernel(const TcParams p) {
  constexpr int D = S::D, NG = S::NG;
  using T = typename std::conditional<BF16, bf16, f16>::type;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                          // [2] tiles
  uint8_t* sK = smem + 2 * S::TILE_BYTES;      // [2]
  uint8_t* sV = smem + 4 * S::TILE_BYTES;      // [2]
  uint8_t* stage = smem + 6 * S::TILE_BYTES;   // [4 warps][STAGES]
  uint64_t* bars = reinterpret_cast<uint64_t*>(stage + 4 * S::STAGES * S::WARP_STAGE);
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
  // Row blocks from the last (the longest under a causal mask) down; the heads and sequences of one row
  // block side by side.
  const int kv_heads = p.c.map.kv_heads;
  const int per_block = p.batch * kv_heads * p.splits;
  const int rb = p.blocks - 1 - static_cast<int>(blockIdx.x) / per_block;
  const int rest = static_cast<int>(blockIdx.x) % per_block;
  const int split = rest % p.splits, bh = rest / p.splits;
  const int b = bh / kv_heads, h = bh % kv_heads;
  const int count = p.counts ? clamp_count(__ldg(p.counts + b), p.tokens) : p.tokens;
  const int length = clamp_count(__ldg(p.lengths + b), capacity(p.c.map));
  if (threadIdx.x == 0 && length != __ldg(p.lengths + b)) atomicExch(p.error_flag, PHEW_ERR_INVALID);
  const int row0 = rb * kTcRows;
  // key tiles that each query tile needs, and this CTA's share of them
  int need[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int first = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(row0 + t * kTileRows)));
    const int last = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(row0 + t * kTileRows + kTileRows - 1)));
    const int end = first >= count ? 0 : seen_end(length, count, last < count ? last : count - 1, p.causal);
    need[t] = (end + kTcTile - 1) / kTcTile;
  }
  const int all = max(need[0], need[1]);
  const int j0 = static_cast<int>(static_cast<int64_t>(all) * split / p.splits);
  const int n_max = static_cast<int>(static_cast<int64_t>(all) * (split + 1) / p.splits) - j0;
  const int n_t[2] = {min(max(need[0] - j0, 0), n_max), min(max(need[1] - j0, 0), n_max)};
  const int key_end = max(0, length);  // rows behind it are never read

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 4);
      mbar_init(&k_full[i], 4);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 4);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(drain, 1);
    *s_poison = 0x7fffffff;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) tmem_alloc(tmem_slot, kTmemCols);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0 && lane == 0) {
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
        const int s = j & 1, s1 = (j + 1) & 1;
        const bool more = j + 1 < n_max;
        if (!mbar_wait(&v_full[s], (j >> 1) & 1, wait_flag, p.wait_ns)) { ok = false; break; }
        if (more && !mbar_wait(&k_full[s1], ((j + 1) >> 1) & 1, wait_flag, p.wait_ns)) { ok = false; break; }
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
  } else if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    // ---------------- producers ----------------
    const int w = warp - 4;
    const uint32_t ring = smem_u32(stage + w * S::STAGES * S::WARP_STAGE);
    const int row = w * 32 + lane;  // of the tile
    const int steps = 2 * n_max;    // K_0, V_0, K_1, ...
    // page lookup one tile ahead of its copies
    int look_page = -1, look_r = 0;
    bool look_any = false;
    auto look_up = [&](int j) {
      const int key = (j0 + j) * kTcTile + row;
      look_any = j < n_max && key < key_end;
      if (look_any) {
        const int col = static_cast<int>(div_by(p.c.map.by_page, static_cast<uint32_t>(key)));
        look_r = key - col * p.c.map.page_size;
        look_page = page_at(p.c.map, b, col);
      }
    };
    uint32_t src_row = kNoRow;
    uint32_t odd = 0;  // per stage (byte): the key's scales are the upper half of the loaded word
    auto start_copy = [&](int q) {
      if (q < steps) {
        const int side = q & 1, s = q % S::STAGES;
        if (side == 0) {
          src_row = kNoRow;
          if (look_any) {
            if (page_ok(p.c.map, look_page))
              src_row = row_at(p.c.map, look_page, h, look_r);
            else
              atomicExch(p.error_flag, PHEW_ERR_INVALID);
          }
          look_up((q >> 1) + 1);
        }
        const uint32_t at = ring + s * S::WARP_STAGE;
        constexpr int CH = D / 32;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int id = i * 32 + lane, r = id / CH, ch = id % CH;
          const uint32_t src = __shfl_sync(0xffffffffu, src_row, r);
          const bool have = src != kNoRow;
          const int sw = CH == 4 ? ch ^ ((r >> 1) & 3) : ch ^ ((r >> 2) & 1);  // eight rows' same chunk: eight bank groups
          copy16<16>(at + r * (D / 2) + sw * 16, p.c.codes[side] + (have ? static_cast<int64_t>(src) * (D / 8) + ch * 4 : 0),
                     have ? 16 : 0);
        }
        const bool have = src_row != kNoRow;
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          const char* arr = static_cast<const char*>(a ? p.c.biases[side] : p.c.scales[side]);
          const uint32_t dst = at + S::WARP_CODES + (a * 32 + lane) * S::SROW;
          if constexpr (S::SB == 2) {
            const int64_t off = (static_cast<int64_t>(have ? src_row : 0) * 2) & ~3ll;
            const uint32_t rows = static_cast<uint32_t>(p.c.map.pages) * static_cast<uint32_t>(p.c.map.kv_heads) *
                                  static_cast<uint32_t>(p.c.map.page_size);
            copy16<4>(dst, arr + off, !have ? 0 : (src_row | 1u) < rows ? 4 : 2);
          } else {
            copy16<S::SB>(dst, arr + (have ? static_cast<int64_t>(src_row) * S::SB : 0), have ? S::SB : 0);
          }
        }
        odd = (odd & ~(1u << s)) | ((have ? src_row & 1u : 0u) << s);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    look_up(0);
    start_copy(0);
    start_copy(1);
    for (int q = 0; q < steps && ok; ++q) {
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
      start_copy(q + 2);  // into the stage read in step q - 1
      const int j = q >> 1, side = q & 1, s = q % S::STAGES;
      const int slot = j & 1;
      const uint32_t at = ring + s * S::WARP_STAGE;
      // this key's scales and biases, each twice in a register
      uint32_t sc[NG], bi[NG];
      bool fine = true;
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const uint32_t src = at + S::WARP_CODES + (a * 32 + lane) * S::SROW;
        uint32_t v[S::SROW / 4];
#pragma unroll
        for (int i = 0; i < S::SROW / 4; ++i) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[i]) : "r"(src + 4 * i));
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const bool upper = S::SB == 2 ? (odd >> s) & 1 : g & 1;
          const uint32_t x = __byte_perm(v[g / 2], 0, upper ? 0x3232 : 0x1010);
          fine = fine && finite16(x, BF16);
          (a ? bi[g] : sc[g]) = x;
        }
      }
      if (side == 1 && !fine) {
        // a weight of zero times infinity is no number, and a later query's keys may not touch an earlier
        // one: the values count as zero here and as "no number" for every row that sees the key
        atomicMin(s_poison, (j0 + j) * kTcTile + row);
#pragma unroll
        for (int g = 0; g < NG; ++g) sc[g] = bi[g] = 0;
      }
      uint64_t* full = side == 0 ? &k_full[slot] : &v_full[slot];
      uint64_t* empty = side == 0 ? &k_empty[slot] : &v_empty[slot];
      if (!mbar_wait(empty, ((j >> 1) & 1) ^ 1, wait_flag, p.wait_ns)) { ok = false; break; }
      const uint32_t dst = smem_u32((side == 0 ? sK : sV) + slot * S::TILE_BYTES) + row * 128;
#pragma unroll
      for (int ch = 0; ch < D / 32; ++ch) {
        const int sw = D == 128 ? ch ^ ((lane >> 1) & 3) : ch ^ ((lane >> 2) & 1);
        uint32_t word[4];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(word[0]), "=r"(word[1]), "=r"(word[2]), "=r"(word[3])
                     : "r"(at + lane * (D / 2) + sw * 16));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int g = (ch * 32 + i * 8) / S::G, c16 = ch * 4 + i;
          store_shared16(dst + (c16 >> 3) * S::HALF_BYTES + (((c16 & 7) ^ (row & 7)) << 4),
                         fma_pair<BF16>(sc[g], code_pair<BF16, 0>(word[i]), bi[g]),
                         fma_pair<BF16>(sc[g], code_pair<BF16, 1>(word[i]), bi[g]),
                         fma_pair<BF16>(sc[g], code_pair<BF16, 2>(word[i]), bi[g]),
                         fma_pair<BF16>(sc[g], code_pair<BF16, 3>(word[i]), bi[g]));
        }
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0 && !(side == 1 && j == p.withhold)) mbar_arrive(full);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // ---------------- softmax and output ----------------
    const int t = (warp - 8) >> 2;
    const int quarter = warp & 3;             // TMEM lanes this warp may access
    const int row = quarter * 32 + lane;      // of the query tile
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lane_addr + t * 128;
    const uint32_t o_addr = tmem + lane_addr + 256 + t * 128;
    const int r = row0 + t * kTileRows + row;
    const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(r)));
    const int head = h * p.per + (r - tok * p.per);
    const int nkv = t ? n_t[1] : n_t[0];
    const float c = p.scale_log2;
    const int lim = seen_end(length, count, tok, p.causal);
    if (nkv > 0) {
      const bool have = tok < count;
      const uint4* q = reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + b * p.st[2] + head * p.st[1] + tok * p.st[0]);
      const uint32_t dst = smem_u32(sQ + t * S::TILE_BYTES) + row * 128;
#pragma unroll
      for (int c16 = 0; c16 < D / 8; ++c16) {
        const uint4 x = have ? __ldg(q + c16) : make_uint4(0, 0, 0, 0);
        store_shared16(dst + (c16 >> 3) * S::HALF_BYTES + (((c16 & 7) ^ (row & 7)) << 4), __byte_perm(x.x, x.z, 0x5410),
                       __byte_perm(x.x, x.z, 0x7632), __byte_perm(x.y, x.w, 0x5410), __byte_perm(x.y, x.w, 0x7632));
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[t]);
    }
    float m_ref = kTcFloor, l = 0.f;
    for (int j = 0; j < nkv && ok; ++j) {
      if (!mbar_wait(&s_full[t], j & 1, wait_flag, p.wait_ns)) { ok = false; break; }
      fence_after_sync();
      uint32_t raw[128];
#pragma unroll
      for (int k = 0; k < 4; ++k) tmem_ld32(s_addr + k * 32, raw + k * 32);
      tmem_ld_wait();
      const int left = lim - (j0 + j) * kTcTile;  // keys of this tile that the row sees
      if (left < kTcTile) {
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i >= left) raw[i] = __float_as_uint(-INFINITY);
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
        if (!mbar_wait(&o_done[t], (j - 1) & 1, wait_flag, p.wait_ns)) ok = false;
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
      tmem_st_wait();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
    }
    if (ok && nkv > 0 && !mbar_wait(&o_done[t], (nkv - 1) & 1, wait_flag, p.wait_ns)) ok = false;
    fence_after_sync();
    if (ok) {
      if (lim > *reinterpret_cast<volatile int*>(s_poison)) l = __int_as_float(0x7fc00000);
      const bool live = nkv > 0 && lim > 0;
      const bool split_up = p.splits > 1;
      const float inv = !live || l == 0.f ? 0.f : 1.f / l;
      const int64_t at = (static_cast<int64_t>(bh) * p.blocks + rb) * p.splits + split;
      float* part = split_up ? p.part + (at * kTcRows + t * kTileRows + row) * D : nullptr;
      T* out = static_cast<T*>(p.o) + ((static_cast<int64_t>(b) * p.heads + head) * p.tokens + tok) * D;
      const bool mine = tok < p.tokens;
      if (split_up && mine) {
        float* ml = p.part_ml + (at * kTcRows + t * kTileRows + row) * 2;
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
          const uint32_t* e = o + 8 * i;  // head dimensions 0 4 1 5 2 6 3 7 of eight
          if (split_up) {
            float4* dst = reinterpret_cast<float4*>(part + k * 32 + i * 8);
            dst[0] = make_float4(__uint_as_float(e[0]), __uint_as_float(e[2]), __uint_as_float(e[4]), __uint_as_float(e[6]));
            dst[1] = make_float4(__uint_as_float(e[1]), __uint_as_float(e[3]), __uint_as_float(e[5]), __uint_as_float(e[7]));
          } else {
            float f[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) f[x] = __uint_as_float(e[x]) * inv;
            *reinterpret_cast<uint4*>(out + k * 32 + i * 8) = make_uint4(pack2<BF16>(f[0], f[2]), pack2<BF16>(f[4], f[6]),
                                                                         pack2<BF16>(f[1], f[3]), pack2<BF16>(f[5], f[7]));
          }
        }
      }
    }
  }
  if (!ok) atomicExch(wait_flag, PHEW_ERR_TIMEOUT);
  fence_before_sync();
  if (__syncthreads_or(!ok)) {
    // a wait ran out somewhere: let the issued products finish before the TMEM and shared memory go
    if (warp == 0 && lane == 0) {
      commit(drain);
      mbar_wait(drain, 0, nullptr, p.wait_ns);
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
template <int D, bool BF16>
__global__ void __launch_bounds__(256) combine_tc_kernel(const TcParams p) {
  using T = typename std::conditional<BF16, bf16, f16>::type;
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t slot = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);  // (bh, block, row)
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int row = static_cast<int>(slot % kTcRows);
  const int64_t seg = slot / kTcRows;
  const int rb = static_cast<int>(seg % p.blocks);
  const int bh = static_cast<int>(seg / p.blocks);
  const int r = rb * kTcRows + row;
  const int tok = static_cast<int>(div_by(p.by_per, static_cast<uint32_t>(r)));
  if (tok >= p.tokens) return;
  const int b = bh / p.c.map.kv_heads, head = (bh % p.c.map.kv_heads) * p.per + (r - tok * p.per);
  float m = kTcFloor;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, p.part_ml[((seg * p.splits + s) * kTcRows + row) * 2]);
  float o[E], l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const int64_t at = (seg * p.splits + s) * kTcRows + row;
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

// CTAs of a call and how many ways each row block's keys are split: enough to
// give every SM a CTA, at most a tile of the longest possible sequence each.
struct TcPlan {
  int64_t blocks, splits, ctas;
};
TcPlan tc_plan(int64_t batch, int kv_heads, int64_t rows, int64_t cap) {
  TcPlan t;
  t.blocks = (rows + kTcRows - 1) / kTcRows;
  const int64_t base = batch * kv_heads * t.blocks, sms = sm_count_current();
  const int64_t tiles = (cap + kTcTile - 1) / kTcTile;
  t.splits = base >= sms ? 1 : sms / base;
  if (t.splits > tiles / 2) t.splits = tiles / 2;
  if (t.splits < 1) t.splits = 1;
  t.ctas = base * t.splits;
  return t;
}

template <typename S, bool BF16> int launch_tc(TcParams p, unsigned grid, cudaStream_t st) {
  static SmemAllowed allowed;
  if (int s = allow_smem(allowed, attn_tc_kernel<S, BF16>, S::SMEM)) return s;
  attn_tc_kernel<S, BF16><<<grid, kTcThreads, S::SMEM, st>>>(p);
  if (int s = launch_status("kv attn_tc_kernel")) return s;
  if (p.splits == 1) return PHEW_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(p.batch) * p.c.map.kv_heads * p.blocks * (kTcRows / 8)));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  PHEW_CHECK_CUDA(cudaLaunchKernelEx(&cfg, combine_tc_kernel<S::D, BF16>, p));
  return launch_status("kv combine_tc_kernel");
}

template <bool BF16> int dispatch_tc(const TcParams& p, unsigned grid, cudaStream_t st) {
  if (p.c.head_dim == 64)
    return p.c.group == 32 ? launch_tc<TcShape<64, 32>, BF16>(p, grid, st) : launch_tc<TcShape<64, 64>, BF16>(p, grid, st);
  if (p.c.group == 32) return launch_tc<TcShape<128, 32>, BF16>(p, grid, st);
  if (p.c.group == 64) return launch_tc<TcShape<128, 64>, BF16>(p, grid, st);
  return launch_tc<TcShape<128, 128>, BF16>(p, grid, st);
}

}  // namespace

size_t tc_bytes(int64_t batch, int kv_heads, int head_dim, int64_t rows, int64_t cap) {
  const TcPlan t = tc_plan(batch, kv_heads, rows, cap);
  return t.splits == 1 ? 0 : static_cast<size_t>(t.ctas) * kTcRows * (static_cast<size_t>(head_dim) + 2) * 4;
}

int run_attn_tc(const AttnParams& a, bool bf16_type, void* workspace, cudaStream_t st) {
  const TcPlan t = tc_plan(a.batch, a.c.map.kv_heads, static_cast<int64_t>(a.tokens) * a.per, capacity(a.c.map));
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
  p.by_per = a.by_per;
  p.scale_log2 = a.scale_log2;
  p.causal = a.causal;
  p.part = static_cast<float*>(workspace);
  p.part_ml = p.part + static_cast<size_t>(t.ctas) * kTcRows * a.c.head_dim;
  p.error_flag = a.error_flag;
  const tc::TestStall stall = tc::take_test_stall();
  p.wait_ns = stall.wait_ns;
  p.withhold = stall.withhold;
  const unsigned grid = static_cast<unsigned>(t.ctas);
  return bf16_type ? dispatch_tc<true>(p, grid, st) : dispatch_tc<false>(p, grid, st);
}

}  // namespace kv
}  // namespace phew
