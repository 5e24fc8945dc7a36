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

}  // namespace kv
}  // namespace phew
