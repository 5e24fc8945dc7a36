// The tcgen05 form of attention over a 4-bit cache, as kv_attn.cu reaches it.
#pragma once

#include "kv_attn.cuh"

namespace phew {
namespace kv {

// Scratch bytes for `rows` query rows to a cache head over sequences of at most `cap` tokens.
size_t tc_bytes(int64_t batch, int kv_heads, int head_dim, int64_t rows, int64_t cap);

// Needs 16-bit types, head_dim 64 or 128 and a positive scale.
int run_attn_tc(const AttnParams& p, bool bf16_type, void* workspace, cudaStream_t st);

}  // namespace kv
}  // namespace phew
