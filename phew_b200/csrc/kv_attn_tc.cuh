// The tcgen05 form of attention over a 4-bit cache, as kv_attn.cu reaches it.
#pragma once

#include "kv_attn.cuh"

namespace phew {
namespace kv {

// Whether a call of `rows` query rows to a cache head over sequences of at most `cap` tokens goes here (a
// positive scale aside).
bool takes_tc(int64_t batch, int kv_heads, int head_dim, int dtype, int64_t rows, int64_t cap);

// Its scratch bytes.
size_t tc_bytes(int64_t batch, int kv_heads, int head_dim, int64_t rows, int64_t cap);

int run_attn_tc(const AttnParams& p, bool bf16_type, void* workspace, cudaStream_t st);

}  // namespace kv
}  // namespace phew
