// What the kernels of the quantised key/value cache share.
#pragma once

#include "common.cuh"
#include "kv_cache.h"

namespace phew {
namespace kv {

// A cache as kernels see it; index 0 is the key side, 1 the value side.
struct Cache {
  uint32_t* codes[2];
  void* scales[2];
  void* biases[2];
  int head_dim, group, bits;
  PageMap map;
};

// Checks a caller's cache and block table and fills *out.
int make_cache(const phew_kv_cache* c, const int* table, int64_t table_stride, int64_t columns, int64_t batch,
               const char* who, Cache* out);

constexpr int64_t kMaxRows = (1ll << 31) - (1 << 16);  // row numbers of a block past the last one stay 32-bit

#ifdef __CUDACC__
// A pair of 16-bit floats, infinities replaced by the type's largest value.
template <bool BF16> __device__ __forceinline__ uint32_t hold_pair(uint32_t x) {
  if constexpr (BF16) {
    asm("min.NaN.bf16x2 %0, %0, %1;" : "+r"(x) : "r"(0x7f7f7f7fu));
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(x) : "r"(0xff7fff7fu));
  } else {
    asm("min.NaN.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0x7bff7bffu));
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(x) : "r"(0xfbfffbffu));
  }
  return x;
}
#endif

// Values of a cache of 16-bit type as [batch][kv_heads][rows][head_dim]
// arrays, for attention's tiles of 128 keys: written up to a sequence's last
// tile, zero behind its last key.  What rounds past the type's range is held
// at its largest value (a masked weight of zero would make a NaN of an
// infinity).  For the same reason a key whose value's scale or bias is not
// finite gets zero for a value and NaN for a key: rows that see it get one
// through their score.
// Launched so that a programmatic dependent may be set up meanwhile.
int expand(const Cache& c, bool bf16_type, void* k, void* v, int64_t batch, int64_t rows, const int32_t* lengths,
           int* error_flag, cudaStream_t st);

}  // namespace kv
}  // namespace phew
