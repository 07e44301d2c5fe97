// Attention over e4m3 pools with block scales.

#include "block_attention.h"

namespace rlt_attn {

int launch_block_fp8(const AttnParams& P, int q_dtype, dim3 grid, int nt, bool whole, hipStream_t stream) {
  return launch_block<RLT_FP8_E4M3>(P, q_dtype, grid, nt, whole, stream);
}

void launch_block_prefill_fp8(const AttnParams& P, int q_dtype, dim3 grid, bool whole, hipStream_t stream) {
  launch_block_prefill<RLT_FP8_E4M3>(P, q_dtype, grid, whole, stream);
}

}  // namespace rlt_attn
