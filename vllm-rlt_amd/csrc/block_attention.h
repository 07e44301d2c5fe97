// Attention over 8-bit pools with one scale per block of tokens and kv head: the MFMA tilings of
// paged_attention.h built for scale mode 3, one source file per code type.
#pragma once

#include "paged_attention.h"

namespace rlt_attn {

// The verify kernels (`whole`: blocks hold whole 16-position tiles and a lane's offset within
// one fits 32 bits; other blocks take their scales position by position, int8 only: e4m3 pools
// have that form already) and the prefill tiling.
int launch_block_fp8(const AttnParams& P, int q_dtype, dim3 grid, int nt, hipStream_t stream);
int launch_block_int8(const AttnParams& P, int q_dtype, dim3 grid, int nt, bool whole, hipStream_t stream);
void launch_block_prefill_fp8(const AttnParams& P, int q_dtype, dim3 grid, bool whole, hipStream_t stream);
void launch_block_prefill_int8(const AttnParams& P, int q_dtype, dim3 grid, bool whole, hipStream_t stream);

}  // namespace rlt_attn

namespace {

template <int QT, int KVT, int D>
int launch_block_d(const AttnParams& P, dim3 grid, int nt, bool whole, hipStream_t stream) {
  if (whole) {
    if (P.compensate) return launch_mfma_ub<QT, KVT, D, 3, true, true>(P, grid, nt, stream);
    return launch_mfma_ub<QT, KVT, D, 3, true, false>(P, grid, nt, stream);
  }
  if constexpr (KVT == RLT_INT8)
    if (!P.compensate) return launch_mfma_ub<QT, KVT, D, 2, false, false>(P, grid, nt, stream);
  return RLT_ERR_UNSUPPORTED;
}

template <int QT, int KVT>
int launch_block_q(const AttnParams& P, dim3 grid, int nt, bool whole, hipStream_t stream) {
  switch (P.head_dim) {
    case 64: return launch_block_d<QT, KVT, 64>(P, grid, nt, whole, stream);
    case 96: return launch_block_d<QT, KVT, 96>(P, grid, nt, whole, stream);
    case 128: return launch_block_d<QT, KVT, 128>(P, grid, nt, whole, stream);
    case 256: return launch_block_d<QT, KVT, 256>(P, grid, nt, whole, stream);
    default: return RLT_ERR_UNSUPPORTED;
  }
}

template <int KVT>
int launch_block(const AttnParams& P, int q_dtype, dim3 grid, int nt, bool whole, hipStream_t stream) {
  return q_dtype == RLT_BF16 ? launch_block_q<RLT_BF16, KVT>(P, grid, nt, whole, stream)
                             : launch_block_q<RLT_F16, KVT>(P, grid, nt, whole, stream);
}

template <int QT, int KVT, int D>
void launch_block_prefill_d(const AttnParams& P, dim3 grid, bool whole, hipStream_t stream) {
  if (whole) rlt_prefill_kernel<QT, KVT, D, 3, true><<<grid, kPfThreads, 0, stream>>>(P);
  else rlt_prefill_kernel<QT, KVT, D, 3, false><<<grid, kPfThreads, 0, stream>>>(P);
}

template <int QT, int KVT>
void launch_block_prefill_q(const AttnParams& P, dim3 grid, bool whole, hipStream_t stream) {
  if (P.head_dim == 64) launch_block_prefill_d<QT, KVT, 64>(P, grid, whole, stream);
  else if (P.head_dim == 96) launch_block_prefill_d<QT, KVT, 96>(P, grid, whole, stream);
  else launch_block_prefill_d<QT, KVT, 128>(P, grid, whole, stream);
}

template <int KVT>
void launch_block_prefill(const AttnParams& P, int q_dtype, dim3 grid, bool whole, hipStream_t stream) {
  if (q_dtype == RLT_BF16) launch_block_prefill_q<RLT_BF16, KVT>(P, grid, whole, stream);
  else launch_block_prefill_q<RLT_F16, KVT>(P, grid, whole, stream);
}

}  // namespace
