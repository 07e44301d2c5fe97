// Attention of a tree of drafted tokens over a paged KV pool: entry point, and the vector
// form of the types and layouts that the MFMA kernels (tree_attention.h) do not take.

#include "rlt_mi355x.h"

#include "tree_attention.h"

#include <type_traits>

namespace tree {

// ---------------------------------------------------------------- vector form

constexpr int kVecDims = 256;
constexpr int64_t kMaxLaunch = UINT32_MAX;  // threads of a launch along one axis

// float32 q, other head sizes, unaligned pools or blocks that split an 8-position group: one
// workgroup per (node, q head), its four waves taking 64-position tiles in turn.  Lane = key
// position for the scores (float32 dot products), lane = dims for the values.  A correctness
// path: every key is read once per q row.
template <int QT, int KVT>
__global__ __launch_bounds__(256) void rlt_tree_vec_kernel(Params P) {
  __shared__ float q[kVecDims];
  __shared__ float wgt[kWaves][64];
  __shared__ int64_t vbase[kWaves][64];
  __shared__ float ml[kWaves][2];
  __shared__ float acc_sh[kWaves][kVecDims];
  const int t = threadIdx.x, lane = t & 63, w = t >> 6;
  const int seq = blockIdx.x;
  const Seq sv = seq_of(P, seq);
  const int node = blockIdx.y / P.hq, head = blockIdx.y % P.hq, kvh = head / P.group;
  if (node >= sv.nodes) return;
  const int D = P.head_dim;
  const int64_t qrow = sv.q_begin + node;
  for (int d = t; d < D; d += 256)
    q[d] = load_as_f32<QT>(P.q, qrow * P.q_row_stride + (int64_t)head * P.q_head_stride + d);
  uint64_t words[kWords];
  const int lo = node_mask(P, sv, node, words);
  __syncthreads();
  float qk = P.qk_scale_log2, v_mul = 1.f;
  if (P.scale_mode == 1) {
    qk *= P.k_scale[0];
    v_mul = P.v_scale[0];
  }
  const int32_t* const table = P.tables + (int64_t)seq * P.table_stride;
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int tb = (lo & ~255) + 64 * w; tb < sv.len; tb += 64 * kWaves) {
    const int pos = tb + lane;
    bool seen = pos >= lo && pos < sv.len;
    if (pos >= sv.base) {
      const int j = pos - sv.base;
      const uint64_t word = j < 64 ? words[0] : j < 128 ? words[1] : j < 192 ? words[2] : words[3];
      seen = pos < sv.len && ((word >> (j & 63)) & 1);
    }
    float s = -INFINITY, vs = 1.f;
    if (seen) {
      const int32_t e = table[pos / P.block_size];
      const int64_t blk = e >= 0 && e < P.num_blocks ? e : 0, off = pos % P.block_size;
      const int64_t kb = blk * P.k_block_stride + off * P.k_token_stride + (int64_t)kvh * P.k_head_stride;
      float x = 0.f;
      for (int d = 0; d < D; ++d) x = __builtin_fmaf(load_as_f32<KVT>(P.k, kb + d), q[d], x);
      if (P.scale_mode == 2) {
        const int64_t so = blk * P.s_block_stride + off * P.s_token_stride + (int64_t)kvh * P.s_head_stride;
        x *= P.k_scale[so];
        vs = P.v_scale[so];
      }
      s = x * qk;
      vbase[w][lane] = blk * P.v_block_stride + off * P.v_token_stride + (int64_t)kvh * P.v_head_stride;
    } else {
      vbase[w][lane] = -1;
    }
    float mx = s;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, RLT_WAVE));
    const float m_new = fmaxf(m, mx);
    const float use = m_new == -INFINITY ? 0.f : m_new;
    const float corr = m_new == m ? 1.f : exp2f(m - use);
    const float p = seen ? exp2f(s - use) : 0.f;
    float sum = p;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum += __shfl_xor(sum, o, RLT_WAVE);
    l = l * corr + sum;
    m = m_new;
    wgt[w][lane] = p * vs;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= corr;
    for (int j = 0; j < 64; ++j) {
      const int64_t vb = vbase[w][j];
      if (vb < 0) continue;
      const float pj = wgt[w][j];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < D) acc[i] = __builtin_fmaf(pj, load_as_f32<KVT>(P.v, vb + lane + 64 * i), acc[i]);
    }
    __builtin_amdgcn_wave_barrier();
  }
  if (lane == 0) {
    ml[w][0] = m;
    ml[w][1] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) acc_sh[w][lane + 64 * i] = acc[i];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int g = 0; g < kWaves; ++g) top = fmaxf(top, ml[g][0]);
  float x[kWaves];
  for (int g = 0; g < kWaves; ++g) {
    const bool live = ml[g][0] != -INFINITY || ml[g][1] != 0.f;
    x[g] = ml[g][0] == -INFINITY ? (live ? ml[g][1] : 0.f) : exp2f(ml[g][0] - top);
    if (live) sum += ml[g][1] * x[g];
  }
  const float inv = sum == 0.f ? 0.f : v_mul / sum;
  for (int d = t; d < D; d += 256) {
    float o = 0.f;
    for (int g = 0; g < kWaves; ++g)
      if (ml[g][0] != -INFINITY || ml[g][1] != 0.f) o += acc_sh[g][d] * x[g];
    store_from_f32<QT>(P.out, qrow * P.out_row_stride + (int64_t)head * P.out_head_stride + d, o * inv);
  }
}

// ---------------------------------------------------------------- launches

template <int QT, int KVT, int D, int SM, int RW>
void launch(const Params& P, hipStream_t stream) {
  using G = Geometry<QT, KVT, D, RW>;
  const dim3 grid(grid_of<D>()), block(64 * kWaves);
  if (P.compensate)
    hipLaunchKernelGGL((rlt_tree_kernel<QT, KVT, D, SM, RW, true>), grid, block, 0, stream, P);
  else
    hipLaunchKernelGGL((rlt_tree_kernel<QT, KVT, D, SM, RW, false>), grid, block, 0, stream, P);
  // few pairs have many contributions each: more workgroups a pair, more threads a row (8 / 32 / 56
  // pairs: 8.0 / 9.6 / 5.1 us against 19.9 / 20.8 / 6.1; 128 / 512 / 880 pairs with one group of
  // threads: 11.0 / 11.5 / 17.8 against 16.5 / 18.8 / 45 with four)
  const int64_t pairs = (int64_t)P.num_seqs * P.hkv * P.max_blocks;
  const int rows = P.max_q * P.group < G::RB ? P.max_q * P.group : G::RB;
  auto merge = [&](auto cg) {
    constexpr int CG = decltype(cg)::value, R = merge_rows<D, CG>();
    hipLaunchKernelGGL((rlt_tree_merge_kernel<QT, D, G::RB, CG>),
                       dim3((unsigned)pairs, (unsigned)((rows + R - 1) / R)), dim3(kMergeThreads), 0,
                       stream, P);
  };
  if (pairs < 64) merge(std::integral_constant<int, 4>{});
  else merge(std::integral_constant<int, 1>{});
}

// Row waves: the fewest that hold the rows of a kv head, at most four (further rows are further
// blocks, which read the keys again: 80 to 128 rows at up to 8192 positions 76 us with four, 98
// with two; 64 rows of 55 heads 163 us with two, 248 with one).  More waves than rows need lose
// the free run of single ones (32 rows in fp8: 645 us with one, 697 with two).
int row_waves(int rows, int head_dim, bool fp8) {
  if (head_dim == 256 && !fp8) return 4;  // two stages of its tiles fit one kv group only
  return rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
}

template <int QT, int KVT, int D, int SM>
void launch_rows(const Params& P, hipStream_t stream) {
  constexpr bool fp8 = KVT != QT;
  const int rw = row_waves(P.max_q * P.group, D, fp8);
  if constexpr (D != 256 || fp8) {
    if (rw == 1) return launch<QT, KVT, D, SM, 1>(P, stream);
    if (rw == 2) return launch<QT, KVT, D, SM, 2>(P, stream);
  }
  return launch<QT, KVT, D, SM, 4>(P, stream);
}

template <int QT, int KVT, int SM>
void launch_dim(const Params& P, hipStream_t stream) {
  switch (P.head_dim) {
    case 64: return launch_rows<QT, KVT, 64, SM>(P, stream);
    case 96: return launch_rows<QT, KVT, 96, SM>(P, stream);
    case 128: return launch_rows<QT, KVT, 128, SM>(P, stream);
    default: return launch_rows<QT, KVT, 256, SM>(P, stream);
  }
}

template <int QT>
void launch_mfma(const Params& P, int kv_dtype, hipStream_t stream) {
  if (kv_dtype != RLT_FP8_E4M3) launch_dim<QT, QT, 0>(P, stream);
  else if (P.scale_mode == 1) launch_dim<QT, RLT_FP8_E4M3, 1>(P, stream);
  else launch_dim<QT, RLT_FP8_E4M3, 2>(P, stream);
}

template <int QT>
int launch_vec(const Params& P, int kv_dtype, hipStream_t stream) {
  const dim3 grid((unsigned)P.num_seqs, (unsigned)(P.max_q * P.hq));
  if (kv_dtype == RLT_FP8_E4M3)
    hipLaunchKernelGGL((rlt_tree_vec_kernel<QT, RLT_FP8_E4M3>), grid, dim3(256), 0, stream, P);
  else
    hipLaunchKernelGGL((rlt_tree_vec_kernel<QT, QT>), grid, dim3(256), 0, stream, P);
  return RLT_OK;
}

bool mfma_dim(int d) { return d == 64 || d == 96 || d == 128 || d == 256; }

}  // namespace tree

extern "C" {

size_t rlt_tree_attention_workspace_size(int32_t num_seqs, int32_t max_q_len, int32_t num_q_heads,
                                         int32_t num_kv_heads, int32_t head_dim, int32_t kv_dtype) {
  if (num_seqs <= 0 || max_q_len <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 ||
      !tree::mfma_dim(head_dim))
    return 0;
  const int64_t rows = (int64_t)max_q_len * (num_q_heads / num_kv_heads);
  const int rb = 32 * tree::row_waves((int)(rows < 1024 ? rows : 1024), head_dim, kv_dtype == RLT_FP8_E4M3);
  const int64_t pairs = (int64_t)num_seqs * num_kv_heads * ((rows + rb - 1) / rb);
  return rlt_align_up((size_t)pairs * sizeof(tree::Split), 256) +
         (size_t)2 * tree::kGrid * tree::kPartRows * (head_dim + 2) * sizeof(float);
}

int rlt_tree_attention_flags(const void* q, int64_t q_row_stride, int64_t q_head_stride,
                             const void* key_cache, const void* value_cache, int64_t k_block_stride,
                             int64_t k_token_stride, int64_t k_head_stride, int64_t v_block_stride,
                             int64_t v_token_stride, int64_t v_head_stride, int32_t num_blocks,
                             const int32_t* block_tables, int64_t table_stride, int32_t table_width,
                             const int32_t* context_lengths, const int32_t* cu_seqlens_q,
                             const int64_t* tree_mask, int64_t mask_stride, int32_t mask_words,
                             int32_t num_seqs, int32_t max_q_len, int32_t num_q_rows,
                             const float* key_scale, const float* value_scale, int32_t scale_mode,
                             int64_t s_block_stride, int64_t s_token_stride, int64_t s_head_stride,
                             int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                             int32_t block_size, int32_t q_dtype, int32_t kv_dtype, int32_t window,
                             int32_t flags, void* out, int64_t out_row_stride, int64_t out_head_stride,
                             void* workspace, size_t workspace_bytes, hipStream_t stream) {
  using namespace tree;
  if (num_seqs < 0 || num_q_rows < 0 || max_q_len < 0 || table_width < 0 || window < 0 ||
      (flags & ~RLT_ATTN_COMPENSATE))
    return RLT_ERR_ARGUMENT;
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads || head_dim <= 0 ||
      block_size <= 0 || num_blocks <= 0)
    return RLT_ERR_ARGUMENT;
  if (q_dtype != RLT_F32 && q_dtype != RLT_F16 && q_dtype != RLT_BF16) return RLT_ERR_ARGUMENT;
  if (kv_dtype != q_dtype && kv_dtype != RLT_FP8_E4M3) return RLT_ERR_UNSUPPORTED;
  if (scale_mode < 0 || scale_mode > 2 || (scale_mode && (!key_scale || !value_scale)) ||
      (kv_dtype == RLT_FP8_E4M3) != (scale_mode != 0))
    return RLT_ERR_ARGUMENT;
  if (num_seqs == 0 || num_q_rows == 0 || max_q_len == 0) return RLT_OK;
  if (!q || !key_cache || !value_cache || (!block_tables && table_width) || !context_lengths ||
      !cu_seqlens_q || !tree_mask || !out)
    return RLT_ERR_ARGUMENT;
  if (head_dim > kVecDims || max_q_len > kMaxNodes || num_q_heads > 1024) return RLT_ERR_UNSUPPORTED;
  if (mask_words <= 0 || (int64_t)mask_words * 64 < max_q_len || mask_stride < mask_words ||
      (uintptr_t)tree_mask % 8)
    return RLT_ERR_ARGUMENT;
  // positions, and a sequence's macro tiles over its kv heads and row blocks, in 32 bits
  const int64_t cap = (int64_t)table_width * block_size;
  const int64_t blocks = ((int64_t)max_q_len * (num_q_heads / num_kv_heads) + 31) / 32;
  if (cap > INT32_MAX - 4096 || (cap / kTile + 1) * num_kv_heads * blocks > INT32_MAX)
    return RLT_ERR_UNSUPPORTED;
  const size_t need = rlt_tree_attention_workspace_size(
      num_seqs, max_q_len, num_q_heads, num_kv_heads, head_dim, kv_dtype);
  if (workspace_bytes < need || (need && (!workspace || (uintptr_t)workspace % 16))) return RLT_ERR_WORKSPACE;

  Params P;
  P.q = q;
  P.q_row_stride = q_row_stride;
  P.q_head_stride = q_head_stride;
  P.k = key_cache;
  P.v = value_cache;
  P.k_block_stride = k_block_stride;
  P.k_token_stride = k_token_stride;
  P.k_head_stride = k_head_stride;
  P.v_block_stride = v_block_stride;
  P.v_token_stride = v_token_stride;
  P.v_head_stride = v_head_stride;
  P.tables = block_tables;
  P.table_stride = table_stride;
  P.table_width = table_width;
  P.num_blocks = num_blocks;
  P.lengths = context_lengths;
  P.cu_q = cu_seqlens_q;
  P.mask = (const uint64_t*)tree_mask;
  P.mask_stride = mask_stride;
  P.mask_words = mask_words;
  P.k_scale = key_scale;
  P.v_scale = value_scale;
  P.s_block_stride = s_block_stride;
  P.s_token_stride = s_token_stride;
  P.s_head_stride = s_head_stride;
  P.num_seqs = num_seqs;
  P.num_rows = num_q_rows;
  P.max_q = max_q_len;
  P.hq = num_q_heads;
  P.hkv = num_kv_heads;
  P.group = num_q_heads / num_kv_heads;
  P.head_dim = head_dim;
  P.block_size = block_size;
  // (one that covers the table hides nothing; a smaller one keeps 32-bit positions, down to the
  // -256 of a tree longer than its cache, above -2^31)
  P.window = window < cap ? window : 0;
  P.qk_scale_log2 = 1.4426950408889634f / sqrtf((float)head_dim);
  P.scale_mode = scale_mode;
  P.compensate = (flags & RLT_ATTN_COMPENSATE) ? 1 : 0;
  P.out = out;
  P.out_row_stride = out_row_stride;
  P.out_head_stride = out_head_stride;

  // MFMA kernels: 16-byte pieces of q and of the pools, whole 8-position groups per block,
  // lane offsets of 32 bits, 8-byte output stores
  const int64_t elt = kv_dtype == RLT_FP8_E4M3 ? 1 : 2;
  const int64_t strides = k_block_stride | k_token_stride | k_head_stride | v_block_stride |
                          v_token_stride | v_head_stride;
  const int64_t far = (int64_t)1 << 26;
  const bool mfma =
      q_dtype != RLT_F32 && mfma_dim(head_dim) && block_size % 8 == 0 && table_width > 0 &&
      (((uintptr_t)key_cache | (uintptr_t)value_cache | (uintptr_t)q) % 16) == 0 &&
      (strides * elt) % 16 == 0 && ((q_row_stride | q_head_stride) * 2) % 16 == 0 &&
      (uintptr_t)out % 8 == 0 && ((out_row_stride | out_head_stride) * 2) % 8 == 0 &&
      k_token_stride >= 0 && k_token_stride < far && v_token_stride >= 0 && v_token_stride < far;
  if (mfma) {
    const int rb = 32 * row_waves(P.max_q * P.group, head_dim, kv_dtype == RLT_FP8_E4M3);
    P.max_blocks = (P.max_q * P.group + rb - 1) / rb;
    const int64_t pairs = (int64_t)num_seqs * num_kv_heads * P.max_blocks;
    if (pairs > kMaxLaunch / kMergeThreads) return RLT_ERR_UNSUPPORTED;
    P.splits = (Split*)workspace;
    P.part = (float*)((char*)workspace + rlt_align_up((size_t)pairs * sizeof(Split), 256));
    if (q_dtype == RLT_BF16) launch_mfma<RLT_BF16>(P, kv_dtype, stream);
    else launch_mfma<RLT_F16>(P, kv_dtype, stream);
    return rlt_launch_status();
  }
  P.splits = nullptr;
  P.max_blocks = 0;
  P.part = nullptr;
  if ((int64_t)P.max_q * num_q_heads > 65535 || num_seqs > kMaxLaunch / 256) return RLT_ERR_UNSUPPORTED;
  switch (q_dtype) {
    case RLT_F32: launch_vec<RLT_F32>(P, kv_dtype, stream); break;
    case RLT_F16: launch_vec<RLT_F16>(P, kv_dtype, stream); break;
    default: launch_vec<RLT_BF16>(P, kv_dtype, stream); break;
  }
  return rlt_launch_status();
}

int rlt_tree_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride,
                       const void* key_cache, const void* value_cache, int64_t k_block_stride,
                       int64_t k_token_stride, int64_t k_head_stride, int64_t v_block_stride,
                       int64_t v_token_stride, int64_t v_head_stride, int32_t num_blocks,
                       const int32_t* block_tables, int64_t table_stride, int32_t table_width,
                       const int32_t* context_lengths, const int32_t* cu_seqlens_q,
                       const int64_t* tree_mask, int64_t mask_stride, int32_t mask_words,
                       int32_t num_seqs, int32_t max_q_len, int32_t num_q_rows,
                       const float* key_scale, const float* value_scale, int32_t scale_mode,
                       int64_t s_block_stride, int64_t s_token_stride, int64_t s_head_stride,
                       int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                       int32_t block_size, int32_t q_dtype, int32_t kv_dtype, int32_t window,
                       void* out, int64_t out_row_stride, int64_t out_head_stride,
                       void* workspace, size_t workspace_bytes, hipStream_t stream) {
  return rlt_tree_attention_flags(
      q, q_row_stride, q_head_stride, key_cache, value_cache, k_block_stride, k_token_stride,
      k_head_stride, v_block_stride, v_token_stride, v_head_stride, num_blocks, block_tables,
      table_stride, table_width, context_lengths, cu_seqlens_q, tree_mask, mask_stride, mask_words,
      num_seqs, max_q_len, num_q_rows, key_scale, value_scale, scale_mode, s_block_stride,
      s_token_stride, s_head_stride, num_q_heads, num_kv_heads, head_dim, block_size, q_dtype,
      kv_dtype, window, 0, out, out_row_stride, out_head_stride, workspace, workspace_bytes, stream);
}

}  // extern "C"
