// Attention over int8 pools, whose scales are the blocks'.

#include "block_attention.h"

namespace rlt_attn {

int block_chunk_log2() { return __builtin_ctz(kBlockChunk); }

int block_groups_per_cu(int head_dim, int nt) {
  return 4 * (head_dim <= 128 && nt == 1 ? block_waves_per_simd<128, 1>() : block_waves_per_simd<128, 2>()) /
         kBlockParts;
}

int launch_block_int8(const AttnParams& P, int q_dtype, dim3 grid, int nt, bool whole, hipStream_t stream) {
  return launch_block<RLT_INT8>(P, q_dtype, grid, nt, whole, stream);
}

void launch_block_prefill_int8(const AttnParams& P, int q_dtype, dim3 grid, bool whole, hipStream_t stream) {
  launch_block_prefill<RLT_INT8>(P, q_dtype, grid, whole, stream);
}

}  // namespace rlt_attn
