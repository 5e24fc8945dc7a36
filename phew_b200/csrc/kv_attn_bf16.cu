// Attention of few query rows over a 4-bit cache: the bf16 kernels.
#define PHEW_KV_ATTN_TYPE bf16
#include "kv_attn.cuh"

namespace phew {
namespace kv {

template size_t attn_bytes<PHEW_KV_ATTN_TYPE>(int64_t, int, int, int, int64_t);
template int run_attn<PHEW_KV_ATTN_TYPE>(const AttnParams&, void*, cudaStream_t);

}  // namespace kv
}  // namespace phew
