// Entry points of the paged attention: the vector path, the merge of a row's chunks, the window
// store ahead of the prefill tiling, and the dispatch.  The tilings are in paged_attention.h.

#include "block_attention.h"

namespace {

// ============================================================ vector path

constexpr int kVecRows = 8;  // rows per row-group on the vector path

struct VecShared {
  float q[kVecRows][256];
  float p[kWaves][kVecRows][kTileTok];
  float ml[2][kVecRows][2];
  float o[2][kVecRows][256];
};

// Scores: lane (position l16, dim quarter grp) dots its quarter with every row's
// q (LDS broadcast) and reduces across quarters.  P * V: lane owns dims
// lane + 64e and reads the tile's 16 value vectors straight from memory.
template <int QT, int KVT>
__global__ __launch_bounds__(256) void rlt_attn_vec_kernel(AttnParams P) {
  __shared__ VecShared sh;
  const int D = P.head_dim;
  const int DQ = (D + 3) / 4;
  const WorkItem wi = work_item(P, blockIdx.x);
  const int seq = wi.seq;
  const int rg = wi.rg;
  const int kvh = wi.hg;  // one kv head per workgroup on this path
  const int chunk = wi.chunk;
  const int wave = threadIdx.x >> 6;
  const int lane = threadIdx.x & 63;
  const int l16 = lane & 15;
  const int grp = lane >> 4;

  const SeqView sv = seq_view(P, seq);
  const int rows_total = sv.q_len * P.group;
  const int rg_begin = rg * kVecRows;
  if (rg_begin >= rows_total) return;
  const int rg_rows = min(kVecRows, rows_total - rg_begin);
  int lo_first, hi_first, lo_last, hi_last;
  group_range(P, sv, rg_begin, rg_rows, lo_first, hi_first, lo_last, hi_last);
  const int c_begin = chunk * kChunk;
  if (c_begin >= hi_last || c_begin + kChunk <= lo_first) return;

  int rlo[kVecRows], rhi[kVecRows];
#pragma unroll
  for (int r = 0; r < kVecRows; ++r) {
    if (r < rg_rows) row_range(P, sv, (rg_begin + r) / P.group, rlo[r], rhi[r]);
    else rlo[r] = rhi[r] = 0;
  }
  for (int idx = threadIdx.x; idx < kVecRows * D; idx += blockDim.x) {
    const int r = idx / D, d = idx % D;
    float x = 0.f;
    if (r < rg_rows) {
      const int rho = rg_begin + r;
      const int head = kvh * P.group + rho % P.group;
      x = load_as_f32<QT>(P.q, (int64_t)(sv.q_begin + rho / P.group) * P.q_row_stride +
                                   (int64_t)head * P.q_head_stride + d);
    }
    sh.q[r][d] = x;
  }
  __syncthreads();

  float qk_scale = P.qk_scale_log2;
  float v_mul = 1.f;
  if (P.scale_mode == 1) {
    qk_scale *= P.k_scale[0];
    v_mul = P.v_scale[0];
  }
  float m_run[kVecRows], l_run[kVecRows], acc[kVecRows][4];
#pragma unroll
  for (int r = 0; r < kVecRows; ++r) {
    m_run[r] = -INFINITY;
    l_run[r] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[r][e] = 0.f;
  }
  const int w_begin = c_begin + wave * kWaveSpan;
  const int span_lo = max(w_begin, lo_first & ~(kTileTok - 1));
  const int span_hi = min(w_begin + kWaveSpan, hi_last);
  const int t0 = span_lo <= w_begin ? 0 : (span_lo - w_begin) / kTileTok;
  const int t1 = span_hi <= w_begin ? 0 : (span_hi - w_begin + kTileTok - 1) / kTileTok;
  for (int t = t0; t < t1; ++t) {
    const int tb = w_begin + t * kTileTok;
    const int pos = tb + l16;
    const bool ok = pos < hi_last;
    int64_t kb = 0;
    float ksc = 1.f;
    if (ok) {
      kb = kv_token_base(P, seq, pos, P.k_block_stride, P.k_token_stride) + (int64_t)kvh * P.k_head_stride;
      if (P.scale_mode == 2) ksc = scale_at(P, P.k_scale, seq, pos, kvh);
    }
    float s_row[kVecRows];
#pragma unroll
    for (int r = 0; r < kVecRows; ++r) s_row[r] = 0.f;
    for (int e = 0; e < DQ; ++e) {
      const int d = grp * DQ + e;
      if (d < D) {
        const float kx = ok ? load_as_f32<KVT>(P.k, kb + d) * ksc : 0.f;
#pragma unroll
        for (int r = 0; r < kVecRows; ++r) s_row[r] = fmaf(kx, sh.q[r][d], s_row[r]);
      }
    }
    float corr[kVecRows];
#pragma unroll
    for (int r = 0; r < kVecRows; ++r) {
      float s = s_row[r];
      s += __shfl_xor(s, 16, RLT_WAVE);
      s += __shfl_xor(s, 32, RLT_WAVE);
      const bool vis = pos >= rlo[r] && pos < rhi[r];
      s = vis ? s * qk_scale : -INFINITY;
      float mx = s;
      for (int off = 1; off < 16; off <<= 1) mx = fmaxf(mx, __shfl_xor(mx, off, RLT_WAVE));
      const float m_new = fmaxf(m_run[r], mx);
      float pr = 0.f;
      corr[r] = 1.f;
      if (m_new != -INFINITY) {
        corr[r] = exp2f(m_run[r] - m_new);
        pr = exp2f(s - m_new);
      }
      float rs = pr;
      for (int off = 1; off < 16; off <<= 1) rs += __shfl_xor(rs, off, RLT_WAVE);
      l_run[r] = l_run[r] * corr[r] + rs;
      m_run[r] = m_new;
      if (grp == 0) sh.p[wave][r][l16] = pr;
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < kVecRows; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[r][e] *= corr[r];
    // P * V over the tile's 16 positions; lane owns dims lane + 64e.
    for (int j = 0; j < kTileTok; ++j) {
      const int pj = tb + j;
      if (pj >= hi_last) break;
      const int64_t vb =
          kv_token_base(P, seq, pj, P.v_block_stride, P.v_token_stride) + (int64_t)kvh * P.v_head_stride;
      const float vsc = P.scale_mode == 2 ? scale_at(P, P.v_scale, seq, pj, kvh) : 1.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = lane + 64 * e;
        if (d < D) {
          const float vx = load_as_f32<KVT>(P.v, vb + d) * vsc;
#pragma unroll
          for (int r = 0; r < kVecRows; ++r) acc[r][e] = fmaf(sh.p[wave][r][j], vx, acc[r][e]);
        }
      }
    }
    __builtin_amdgcn_wave_barrier();
  }

  auto publish = [&](int buf) {
    if (lane < kVecRows) {
      float mv = 0.f, lv = 0.f;
#pragma unroll
      for (int r = 0; r < kVecRows; ++r)
        if (r == lane) { mv = m_run[r]; lv = l_run[r]; }
      sh.ml[buf][lane][0] = mv;
      sh.ml[buf][lane][1] = lv;
    }
#pragma unroll
    for (int r = 0; r < kVecRows; ++r)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = lane + 64 * e;
        if (d < D) sh.o[buf][r][d] = acc[r][e];
      }
  };
  auto absorb = [&](int buf) {
#pragma unroll
    for (int r = 0; r < kVecRows; ++r) {
      float mo, s1, s2;
      merge_scales(m_run[r], sh.ml[buf][r][0], mo, s1, s2);
      m_run[r] = mo;
      l_run[r] = l_run[r] * s1 + sh.ml[buf][r][1] * s2;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = lane + 64 * e;
        if (d < D) acc[r][e] = acc[r][e] * s1 + sh.o[buf][r][d] * s2;
      }
    }
  };
  __syncthreads();
  if (wave >= 2) publish(wave - 2);
  __syncthreads();
  if (wave < 2) absorb(wave);
  __syncthreads();
  if (wave == 1) publish(0);
  __syncthreads();
  if (wave != 0) return;
  absorb(0);
#pragma unroll
  for (int r = 0; r < kVecRows; ++r) {
    if (r >= rg_rows) continue;
    const int lo_c = rlo[r] / kChunk;
    const int hi_c = (rhi[r] + kChunk - 1) / kChunk;
    if (chunk < lo_c || chunk >= hi_c) continue;
    const int rho = rg_begin + r;
    const int qrow = sv.q_begin + rho / P.group;
    const int head = kvh * P.group + rho % P.group;
    const int64_t slot = ((int64_t)qrow * P.hq + head) * P.max_chunks + chunk;
    if (lane == 0) {
      P.part_ml[2 * slot] = m_run[r];
      P.part_ml[2 * slot + 1] = l_run[r];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int d = lane + 64 * e;
      if (d < D) P.part_o[slot * D + d] = acc[r][e] * v_mul;
    }
  }
}

// ============================================================ merge

// grid (sequences x max_q, ceil(hq / 4)), 256 threads: one wave per (row, head).
// Combines the row's chunks: the (max, sum) of up to kMergeBatch chunks and
// their head-dim values are loaded together (one memory round trip), the scale
// exp2(m_c - M) of chunk c comes from lane c, and every lane accumulates its dims
// over the chunks in chunk order.  The order depends only on the row's own chunk
// range.  reference: triton_attention.py:145-173 (empty rows give zeros; 1e-30
// floor).
constexpr int kMergeBatch = 16;

// Lane c's value of x in every lane (c wave-uniform).
__device__ __forceinline__ float lane_value(float x, int c) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), c));
}

// E: head dims per lane (ceil(head_dim / 64)).
template <int OT, int E>
__global__ __launch_bounds__(256) void rlt_merge_kernel(AttnParams P) {
  const int head = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (head >= P.hq) return;
  int seq, qi;
  if (P.cu_q) {
    seq = blockIdx.x / P.max_q;
    qi = blockIdx.x % P.max_q;
  } else {
    seq = blockIdx.x;
    qi = 0;
  }
  const SeqView sv = seq_view(P, seq);
  if (qi >= sv.q_len) return;
  const int row = sv.q_begin + qi;
  int lo, hi;
  row_range(P, sv, qi, lo, hi);
  const int c0 = lo >> P.chunk_log2, c1 = (hi + (1 << P.chunk_log2) - 1) >> P.chunk_log2;
  const int nc = c1 - c0;
  if (P.direct && nc <= 1) return;  // (written by the attention kernel)
  const int64_t base = ((int64_t)row * P.hq + head) * P.max_chunks + c0;
  const int64_t out_off = (int64_t)row * P.out_row_stride + (int64_t)head * P.out_head_stride;
  const int D = P.head_dim;
  if (nc <= 0) {
    for (int d = lane; d < D; d += 64) store_from_f32<OT>(P.out, out_off + d, 0.f);
    return;
  }
  if (nc <= kMergeBatch) {
    // statistics (lane c) and values (every lane, dims lane + 64e) of all chunks
    float m = -INFINITY, l = 0.f;
    if (lane < nc) {
      m = P.part_ml[2 * (base + lane)];
      l = P.part_ml[2 * (base + lane) + 1];
    }
    float v[kMergeBatch][E];
#pragma unroll
    for (int c = 0; c < kMergeBatch; ++c)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int d = lane + 64 * e;
        v[c][e] = (c < nc && d < D) ? P.part_o[(base + c) * D + d] : 0.f;
      }
    float mmax = -INFINITY;
    for (int c = 0; c < nc; ++c) mmax = fmaxf(mmax, lane_value(m, c));
    const float sc = (lane < nc && m != -INFINITY) ? exp2f(m - mmax) : 0.f;
    float lsum = 0.f;
    const float ls = l * sc;
    for (int c = 0; c < nc; ++c) lsum += lane_value(ls, c);
    const float inv_den = 1.f / fmaxf(lsum, 1.0e-30f);
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    // chunks past nc have scale 0 and values 0: adding them changes nothing
#pragma unroll
    for (int c = 0; c < kMergeBatch; ++c) {
      const float sv = lane_value(sc, c);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += v[c][e] * sv;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int d = lane + 64 * e;
      if (d < D) store_from_f32<OT>(P.out, out_off + d, acc[e] * inv_den);
    }
    return;
  }
  // long rows: chunk statistics 64 at a time, then values chunk by chunk
  float mmax = -INFINITY;
  for (int c = lane; c < nc; c += 64) mmax = fmaxf(mmax, P.part_ml[2 * (base + c)]);
  for (int off = 32; off >= 1; off >>= 1) mmax = fmaxf(mmax, __shfl_xor(mmax, off, RLT_WAVE));
  float l = 0.f;
  for (int c0p = 0; c0p < nc; c0p += 64) {
    const int c = c0p + lane;
    float part = 0.f;
    if (c < nc) {
      const float m = P.part_ml[2 * (base + c)];
      const float s = m == -INFINITY ? 0.f : exp2f(m - mmax);
      part = P.part_ml[2 * (base + c) + 1] * s;
    }
    for (int off = 32; off >= 1; off >>= 1) part += __shfl_xor(part, off, RLT_WAVE);
    l += part;
  }
  const float inv_den = 1.f / fmaxf(l, 1.0e-30f);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int c0p = 0; c0p < nc; c0p += 64) {
    const int cn = min(64, nc - c0p);
    float my_s = 0.f;
    if (lane < cn) {
      const float m = P.part_ml[2 * (base + c0p + lane)];
      my_s = m == -INFINITY ? 0.f : exp2f(m - mmax);
    }
    int c = 0;
    for (; c + 4 <= cn; c += 4) {  // four chunks of loads in flight
      float v[4][4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int d = lane + 64 * e;
          v[u][e] = d < D ? P.part_o[(base + c0p + c + u) * D + d] : 0.f;
        }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float s = __shfl(my_s, c + u, RLT_WAVE);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += v[u][e] * s;
      }
    }
    for (; c < cn; ++c) {
      const float s = __shfl(my_s, c, RLT_WAVE);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int d = lane + 64 * e;
        if (d < D) acc[e] += P.part_o[(base + c0p + c) * D + d] * s;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int d = lane + 64 * e;
    if (d < D) store_from_f32<OT>(P.out, out_off + d, acc[e] * inv_den);
  }
}


// Window store ahead of the prefill tiling (a store-and-attend call whose window takes
// it).  A group of 8 or 16 lanes takes one vector -- a window row's key or value of one kv
// head, 16 bytes a lane -- and a workgroup kStoreVectors consecutive vectors of a sequence
// (kv heads innermost, keys before values), with the loads of all of a lane's vectors in
// flight before the first is quantized.  The bits are store_rows' (the verify kernels'
// fused store).
//
// What bounds it: memory latency on short chunks, then HBM.  A wave that took 16 rows of a
// kv head one after the other waited for a row's load, its table entry and its reduction
// 16 times over: 2820 rows of 8 heads, D = 128, quantized with per-vector scales 37.9 us,
// here 15.3; 8 x 2048 rows of 4 heads in bf16, 13.9.
constexpr int kStoreThreads = 256;
constexpr int kStoreDepth = 4;  // vectors per lane group
template <int D>
constexpr int store_lanes() { return D <= 64 ? 8 : 16; }
template <int D>
constexpr int store_vectors() { return kStoreThreads / store_lanes<D>() * kStoreDepth; }
// Workgroups of one launch: a grid holds fewer than 2^32 threads, and a call may ask for more
// (its windows are padded to the longest).
constexpr int64_t kStoreGrid = (int64_t)1 << 23;

// NaN-propagating maximum over a group of L (8 or 16) lanes, in every lane.
template <int L>
__device__ __forceinline__ float group_nan_max(float x) {
  auto at = [](float v, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value,
                                                      0xf, 0xf, false));
  };
  x = rlt_fp8::nan_max(x, at(x, std::integral_constant<int, 0xB1>{}));   // lane ^ 1
  x = rlt_fp8::nan_max(x, at(x, std::integral_constant<int, 0x4E>{}));   // lane ^ 2
  x = rlt_fp8::nan_max(x, at(x, std::integral_constant<int, 0x141>{}));  // 8 lanes mirrored
  if (L == 16) x = rlt_fp8::nan_max(x, at(x, std::integral_constant<int, 0x140>{}));
  return x;
}

template <int QT, int KVT, int D, int SM>
__global__ __launch_bounds__(kStoreThreads) void rlt_window_store_kernel(AttnParams P, uint32_t per_seq,
                                                                         uint32_t first_wg) {
  constexpr int LPV = store_lanes<D>();
  constexpr int kPieces = D / 8;  // 16-byte pieces of a vector
  constexpr int kAtOnce = kStoreThreads / LPV;
  const uint32_t wg = first_wg + blockIdx.x;
  const int seq = (int)(wg / per_seq);
  const int64_t first = (int64_t)(wg - seq * per_seq) * store_vectors<D>();
  const SeqView sv = seq_view(P, seq);
  const uint32_t vectors = 2 * P.hkv;  // of one row
  const int row0 = (int)(first / vectors);
  if (row0 >= sv.q_len) return;
  const uint32_t off0 = (uint32_t)(first - (int64_t)row0 * vectors);
  const int sub = threadIdx.x / LPV, piece = threadIdx.x % LPV;
  uint4 raw[kStoreDepth];
  int32_t entry[kStoreDepth];
  int head[kStoreDepth], off[kStoreDepth];
  bool value[kStoreDepth];
#pragma unroll
  for (int u = 0; u < kStoreDepth; ++u) {
    const uint32_t at = off0 + sub + u * kAtOnce;
    const int i = row0 + (int)(at / vectors);
    const uint32_t vec = at % vectors;
    value[u] = vec >= (uint32_t)P.hkv;
    head[u] = (int)(value[u] ? vec - P.hkv : vec);
    // positions before the sequence, past the block table or outside the pool are not
    // written
    const int pos = sv.kv_len - sv.q_len + i;
    const int idx = pos / P.block_size;
    off[u] = pos % P.block_size;
    const bool live = i < sv.q_len && pos >= 0 && idx < P.table_width;
    entry[u] = live ? P.tables[(int64_t)seq * P.table_stride + idx] : -1;
    raw[u] = make_uint4(0, 0, 0, 0);
    if (live && piece < kPieces)
      raw[u] = ((const uint4*)((const uint16_t*)(value[u] ? P.new_v : P.new_k) +
                               (int64_t)(sv.q_begin + i) * P.new_row_stride +
                               (int64_t)head[u] * P.new_head_stride))[piece];
  }
#pragma unroll
  for (int u = 0; u < kStoreDepth; ++u) {
    const bool store = entry[u] >= 0 && entry[u] < P.num_blocks;
    const int64_t at = (int64_t)entry[u] * (value[u] ? P.v_block_stride : P.k_block_stride) +
                       (int64_t)off[u] * (value[u] ? P.v_token_stride : P.k_token_stride) +
                       (int64_t)head[u] * (value[u] ? P.v_head_stride : P.k_head_stride);
    uint8_t* pool = (uint8_t*)(value[u] ? P.v : P.k);
    if constexpr (KVT == QT) {
      if (store && piece < kPieces) ((uint4*)(pool + 2 * at))[piece] = raw[u];
    } else {
      const uint32_t w4[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
      float x[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = Mfma<QT>::lo_f32(w4[j]);
        x[2 * j + 1] = Mfma<QT>::hi_f32(w4[j]);
      }
      float* scales = const_cast<float*>(value[u] ? P.v_scale : P.k_scale);
      float scale;
      if constexpr (SM == 2) {
        float amax = 0.f;  // (lanes past the vector hold zeros)
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = rlt_fp8::nan_max(amax, fabsf(x[j]));
        scale = rlt_fp8::dynamic_scale(group_nan_max<LPV>(amax));
      } else {
        scale = scales[0];
      }
      if (store && piece < kPieces) {
        uint32_t lo = 0, hi = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          lo |= rlt_fp8::encode(x[j], scale) << (8 * j);
          hi |= rlt_fp8::encode(x[4 + j], scale) << (8 * j);
        }
        *(uint2*)(pool + at + 8 * piece) = make_uint2(lo, hi);
        if (SM == 2 && piece == 0)
          scales[(int64_t)entry[u] * P.s_block_stride + (int64_t)off[u] * P.s_token_stride +
                 (int64_t)head[u] * P.s_head_stride] = scale;
      }
    }
  }
}

// ============================================================ dispatch

// Blocks hold whole 16-position tiles and a lane's offset within a tile fits 32 bits.
bool whole_tiles(const AttnParams& P) {
  const int64_t most = (int64_t)1 << 26;
  return P.block_size % kTileTok == 0 && P.k_token_stride >= 0 && P.k_token_stride < most &&
         P.v_token_stride >= 0 && P.v_token_stride < most;
}

// UB: whole_tiles.  Compensated P V is built for such block sizes only (the reference pools' block size 16
// and its multiples).
template <int QT, int KVT, int D, int SM>
int launch_mfma_sm(const AttnParams& P, dim3 grid, int nt, hipStream_t stream) {
  const bool ub = whole_tiles(P);
  if (P.compensate) {
    if (P.block_size % kTileTok != 0) return RLT_ERR_UNSUPPORTED;
    if (ub) return launch_mfma_ub<QT, KVT, D, SM, true, true>(P, grid, nt, stream);
    return launch_mfma_ub<QT, KVT, D, SM, false, true>(P, grid, nt, stream);
  }
  if (ub) return launch_mfma_ub<QT, KVT, D, SM, true, false>(P, grid, nt, stream);
  return launch_mfma_ub<QT, KVT, D, SM, false, false>(P, grid, nt, stream);
}

template <int QT, int KVT, int D>
int launch_mfma_d(const AttnParams& P, dim3 grid, int nt, hipStream_t stream) {
  // 16-bit pools are read unscaled (scale_mode applies to fp8 pools only)
  if constexpr (KVT == QT) {
    return launch_mfma_sm<QT, KVT, D, 0>(P, grid, nt, stream);
  } else {
    if (P.scale_mode == 1) return launch_mfma_sm<QT, KVT, D, 1>(P, grid, nt, stream);
    return launch_mfma_sm<QT, KVT, D, 2>(P, grid, nt, stream);
  }
}

template <int QT, int KVT>
int launch_mfma(const AttnParams& P, dim3 grid, int nt, hipStream_t stream) {
  switch (P.head_dim) {
    case 64: return launch_mfma_d<QT, KVT, 64>(P, grid, nt, stream);
    case 96: return launch_mfma_d<QT, KVT, 96>(P, grid, nt, stream);
    case 128: return launch_mfma_d<QT, KVT, 128>(P, grid, nt, stream);
    case 256: return launch_mfma_d<QT, KVT, 256>(P, grid, nt, stream);
    default: return RLT_ERR_UNSUPPORTED;
  }
}

bool mfma_head_dim(int d) { return d == 64 || d == 96 || d == 128 || d == 256; }

template <int QT>
int launch_vec_q(const AttnParams& P, int kv_dtype, dim3 grid, hipStream_t stream) {
  switch (kv_dtype) {
    case RLT_F32: rlt_attn_vec_kernel<QT, RLT_F32><<<grid, 256, 0, stream>>>(P); break;
    case RLT_F16: rlt_attn_vec_kernel<QT, RLT_F16><<<grid, 256, 0, stream>>>(P); break;
    case RLT_BF16: rlt_attn_vec_kernel<QT, RLT_BF16><<<grid, 256, 0, stream>>>(P); break;
    case RLT_FP8_E4M3: rlt_attn_vec_kernel<QT, RLT_FP8_E4M3><<<grid, 256, 0, stream>>>(P); break;
    case RLT_INT8: rlt_attn_vec_kernel<QT, RLT_INT8><<<grid, 256, 0, stream>>>(P); break;
    default: return RLT_ERR_ARGUMENT;
  }
  return RLT_OK;
}

template <int QT, int KVT, int D, int SM>
void launch_prefill_sm(const AttnParams& P, dim3 grid, int max_q, hipStream_t stream) {
  if (P.new_k) {
    const int64_t per_seq = ((int64_t)max_q * 2 * P.hkv + store_vectors<D>() - 1) / store_vectors<D>();
    const int64_t wgs = P.num_seqs * per_seq;  // (attention_impl: below 2^32)
    for (int64_t at = 0; at < wgs; at += kStoreGrid)
      rlt_window_store_kernel<QT, KVT, D, SM>
          <<<(unsigned)(wgs - at < kStoreGrid ? wgs - at : kStoreGrid), kStoreThreads, 0, stream>>>(
              P, (uint32_t)per_seq, (uint32_t)at);
  }
  if (whole_tiles(P))
    rlt_prefill_kernel<QT, KVT, D, SM, true><<<grid, kPfThreads, 0, stream>>>(P);
  else
    rlt_prefill_kernel<QT, KVT, D, SM, false><<<grid, kPfThreads, 0, stream>>>(P);
}

template <int QT, int KVT, int D>
void launch_prefill_d(const AttnParams& P, dim3 grid, int max_q, hipStream_t stream) {
  if constexpr (KVT == QT) launch_prefill_sm<QT, KVT, D, 0>(P, grid, max_q, stream);
  else if (P.scale_mode == 1) launch_prefill_sm<QT, KVT, D, 1>(P, grid, max_q, stream);
  else launch_prefill_sm<QT, KVT, D, 2>(P, grid, max_q, stream);
}

// max_q: the longest window (the store of the rows, when the call has one, goes first)
template <int QT, int KVT>
void launch_prefill(const AttnParams& P, int head_dim, dim3 grid, int max_q, hipStream_t stream) {
  if (head_dim == 64) launch_prefill_d<QT, KVT, 64>(P, grid, max_q, stream);
  else if (head_dim == 96) launch_prefill_d<QT, KVT, 96>(P, grid, max_q, stream);
  else launch_prefill_d<QT, KVT, 128>(P, grid, max_q, stream);
}

template <int OT>
void launch_merge(const AttnParams& P, dim3 grid, hipStream_t stream) {
  switch ((P.head_dim + 63) / 64) {
    case 1: rlt_merge_kernel<OT, 1><<<grid, 256, 0, stream>>>(P); break;
    case 2: rlt_merge_kernel<OT, 2><<<grid, 256, 0, stream>>>(P); break;
    case 3: rlt_merge_kernel<OT, 3><<<grid, 256, 0, stream>>>(P); break;
    default: rlt_merge_kernel<OT, 4><<<grid, 256, 0, stream>>>(P); break;
  }
}

// Compute units of the current device (cached per device).
int compute_units() {
  static int cached[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) return 256;
  if (dev < 64 && cached[dev] > 0) return cached[dev];
  int n = 0;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
    n = 256;
  if (dev < 64) cached[dev] = n;
  return n;
}

int max_chunks_for(int32_t table_width, int32_t block_size, int chunk = kChunk) {
  const int64_t tokens = (int64_t)table_width * block_size;
  return (int)((tokens + chunk - 1) / chunk);
}

}  // namespace

extern "C" {

int rlt_abi_version(void) { return RLT_MI355X_ABI_VERSION; }

int rlt_paged_attention_uses_mfma(int32_t q_dtype, int32_t kv_dtype, int32_t head_dim) {
  const bool qok = q_dtype == RLT_BF16 || q_dtype == RLT_F16;
  const bool kvok = kv_dtype == q_dtype || kv_dtype == RLT_FP8_E4M3 || kv_dtype == RLT_INT8;
  return qok && kvok && mfma_head_dim(head_dim);
}

int rlt_paged_attention_uses_prefill(int32_t q_dtype, int32_t kv_dtype, int32_t head_dim,
                                     int32_t max_q_len) {
  return rlt_paged_attention_uses_mfma(q_dtype, kv_dtype, head_dim) &&
         (head_dim == 64 || head_dim == 96 || head_dim == 128) && max_q_len >= kPfMinQ;
}

size_t rlt_paged_attention_workspace_size(int32_t num_q_rows, int32_t num_q_heads, int32_t head_dim,
                                          int32_t table_width, int32_t block_size) {
  const int64_t slots = (int64_t)num_q_rows * num_q_heads * max_chunks_for(table_width, block_size);
  return rlt_align_up(sizeof(float) * slots * 2, 256) + rlt_align_up(sizeof(float) * slots * head_dim, 256);
}

}  // extern "C"

namespace {

struct WindowStore {
  const void* k;
  const void* v;
  int64_t row_stride, head_stride;
};

int attention_impl(const void* q, int64_t q_row_stride, int64_t q_head_stride,
                             const void* key_cache, const void* value_cache, int64_t k_block_stride,
                             int64_t k_token_stride, int64_t k_head_stride, int64_t v_block_stride,
                             int64_t v_token_stride, int64_t v_head_stride, int32_t num_blocks,
                             const int32_t* block_tables, int64_t table_stride, int32_t table_width,
                             const int32_t* context_lengths, const int32_t* row_lengths,
                             const int32_t* cu_seqlens_q, int32_t num_seqs, int32_t max_q_len,
                             int32_t num_q_rows, const float* key_scale, const float* value_scale,
                             int32_t scale_mode, int64_t s_block_stride, int64_t s_token_stride,
                             int64_t s_head_stride, int32_t num_q_heads, int32_t num_kv_heads,
                             int32_t head_dim, int32_t block_size, int32_t q_dtype, int32_t kv_dtype,
                             int32_t window, int32_t flags, void* out, int64_t out_row_stride,
                             int64_t out_head_stride, void* workspace, size_t workspace_bytes,
                             hipStream_t stream, const WindowStore* store) {
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads) return RLT_ERR_ARGUMENT;
  if (head_dim <= 0 || head_dim > 256 || block_size <= 0 || window < 0) return RLT_ERR_ARGUMENT;
  if (num_seqs < 0 || num_q_rows < 0 || max_q_len < 0 || table_width < 0) return RLT_ERR_ARGUMENT;
  if (scale_mode < 0 || scale_mode > 3 || (scale_mode && (!key_scale || !value_scale)))
    return RLT_ERR_ARGUMENT;
  if (kv_dtype == RLT_FP8_E4M3 && scale_mode == 0) return RLT_ERR_ARGUMENT;
  // block scales: 8-bit pools, and all that int8 pools take
  if (scale_mode == 3 ? kv_dtype != RLT_FP8_E4M3 && kv_dtype != RLT_INT8 : kv_dtype == RLT_INT8)
    return RLT_ERR_ARGUMENT;
  if (q_dtype == RLT_FP8_E4M3 || q_dtype == RLT_INT8) return RLT_ERR_ARGUMENT;
  if (scale_mode == 3 && store) return RLT_ERR_UNSUPPORTED;  // rlt_kv_append, then the attention
  if (flags & ~RLT_ATTN_COMPENSATE) return RLT_ERR_ARGUMENT;
  if (num_blocks <= 0) return RLT_ERR_ARGUMENT;
  if (num_q_rows == 0 || num_seqs == 0) return RLT_OK;
  if (!cu_seqlens_q && num_seqs != num_q_rows) return RLT_ERR_ARGUMENT;
  if (cu_seqlens_q && max_q_len <= 0) return RLT_ERR_ARGUMENT;
  if (row_lengths && !cu_seqlens_q) return RLT_ERR_ARGUMENT;
  const size_t need = rlt_paged_attention_workspace_size(num_q_rows, num_q_heads, head_dim,
                                                         table_width, block_size);
  if (!workspace || workspace_bytes < need) return RLT_ERR_WORKSPACE;

  AttnParams P;
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
  P.row_len = row_lengths;
  P.k_scale = key_scale;
  P.v_scale = value_scale;
  P.s_block_stride = s_block_stride;
  P.s_token_stride = scale_mode == 3 ? 0 : s_token_stride;
  P.s_head_stride = s_head_stride;
  P.scale_mode = scale_mode;
  P.compensate = (flags & RLT_ATTN_COMPENSATE) ? 1 : 0;
  P.direct = 0;
  P.first_group = 0;
  P.num_seqs = num_seqs;
  P.num_rows = num_q_rows;
  P.hq = num_q_heads;
  P.hkv = num_kv_heads;
  P.group = num_q_heads / num_kv_heads;
  P.head_dim = head_dim;
  P.block_size = block_size;
  P.window = window;
  // chunk size: 1024 for 8-bit KV on the MFMA path (unit_chunk), 512 otherwise; the
  // workspace query sizes the partials for 512, an upper bound
  const bool code8 = kv_dtype == RLT_FP8_E4M3 || kv_dtype == RLT_INT8;
  const bool code8_mfma = code8 && rlt_paged_attention_uses_mfma(q_dtype, kv_dtype, head_dim);
  P.chunk_log2 = !code8_mfma ? 9 : scale_mode == 3 && whole_tiles(P) ? rlt_attn::block_chunk_log2() : 10;
  P.max_chunks = max_chunks_for(table_width, block_size, 1 << P.chunk_log2);
  P.qk_scale_log2 = kLog2e / sqrtf((float)head_dim);
  P.out = out;
  P.out_row_stride = out_row_stride;
  P.out_head_stride = out_head_stride;
  const int64_t slots = (int64_t)num_q_rows * num_q_heads * P.max_chunks;
  P.part_ml = (float*)workspace;
  P.part_o = (float*)((char*)workspace + rlt_align_up(sizeof(float) * slots * 2, 256));
  if (P.max_chunks == 0) P.max_chunks = 1;  // zero-width tables: every row is empty
  P.new_k = store ? store->k : nullptr;
  P.new_v = store ? store->v : nullptr;
  P.new_row_stride = store ? store->row_stride : 0;
  P.new_head_stride = store ? store->head_stride : 0;
  if (store) {
    // the fused window store, on the verify kernels only: 16-bit pools (no scales), or
    // fp8 pools with per-tensor or per-vector scales; the rows are bf16 / fp16 like q
    const bool fp8 = kv_dtype == RLT_FP8_E4M3;
    if (!cu_seqlens_q || (q_dtype != RLT_BF16 && q_dtype != RLT_F16) ||
        !(kv_dtype == q_dtype || fp8) ||
        !rlt_paged_attention_uses_mfma(q_dtype, kv_dtype, head_dim))
      return RLT_ERR_UNSUPPORTED;
    if (fp8 != (scale_mode != 0)) return RLT_ERR_ARGUMENT;
    const int64_t piece = fp8 ? 8 : 16;  // bytes each lane stores into the pool
    const int64_t elt = fp8 ? 1 : 2;
    if (!store->k || !store->v || ((uintptr_t)store->k | (uintptr_t)store->v) % 16 ||
        (store->row_stride * 2) % 16 || (store->head_stride * 2) % 16 ||
        (k_token_stride * elt) % piece || (v_token_stride * elt) % piece ||
        (k_head_stride * elt) % piece || (v_head_stride * elt) % piece ||
        (k_block_stride * elt) % piece || (v_block_stride * elt) % piece)
      return RLT_ERR_ARGUMENT;
  }

  const int rows_per_seq = max_q_len * P.group;
  const bool mfma = rlt_paged_attention_uses_mfma(q_dtype, kv_dtype, head_dim);
  int st = RLT_OK;
  if (mfma) {
    // 16-byte vector loads of q and of every lane's KV slice.
    const int64_t kv_elt = code8 ? 1 : 2;
    // (8-bit keys with head_dim % 64 == 0 are read 16 bytes per lane: RawSlice::kWide)
    const int64_t kv_align = code8 && head_dim % 64 != 0 ? 8 : 16;
    const bool aligned =
        ((uintptr_t)q % 16 == 0) && (q_row_stride * 2) % 16 == 0 && (q_head_stride * 2) % 16 == 0 &&
        ((uintptr_t)key_cache % 16 == 0) && ((uintptr_t)value_cache % 16 == 0) &&
        (k_block_stride * kv_elt) % kv_align == 0 && (k_token_stride * kv_elt) % kv_align == 0 &&
        (k_head_stride * kv_elt) % kv_align == 0 && (v_block_stride * kv_elt) % kv_align == 0 &&
        (v_token_stride * kv_elt) % kv_align == 0 && (v_head_stride * kv_elt) % kv_align == 0;
    if (!aligned) return RLT_ERR_ARGUMENT;
    // (compensated calls stay on the verify kernels at every q_len)
    if (cu_seqlens_q && !row_lengths && !P.compensate &&
        rlt_paged_attention_uses_prefill(q_dtype, kv_dtype, head_dim, max_q_len)) {
      // long q windows: the prefill tiling, normalized in one launch
      P.rows_per_rg = kPfRows;
      P.rowgroups = (rows_per_seq + kPfRows - 1) / kPfRows;
      const int64_t wgs = (int64_t)num_seqs * P.rowgroups * num_kv_heads;
      if (wgs >= ((int64_t)1 << 31)) return RLT_ERR_UNSUPPORTED;
      const dim3 grid((unsigned)wgs);
      // the window store's workgroups: 64 vectors or more each, two vectors per row and kv
      // head, so at most twice this many
      const int64_t swgs = (int64_t)num_seqs * num_kv_heads * (((int64_t)max_q_len + 63) / 64);
      if (swgs >= ((int64_t)1 << 31)) return RLT_ERR_UNSUPPORTED;
      const bool fp8 = kv_dtype == RLT_FP8_E4M3;
      if (scale_mode == 3) {
        if (fp8) rlt_attn::launch_block_prefill_fp8(P, q_dtype, grid, whole_tiles(P), stream);
        else rlt_attn::launch_block_prefill_int8(P, q_dtype, grid, whole_tiles(P), stream);
      } else if (q_dtype == RLT_BF16) {
        if (fp8) launch_prefill<RLT_BF16, RLT_FP8_E4M3>(P, head_dim, grid, max_q_len, stream);
        else launch_prefill<RLT_BF16, RLT_BF16>(P, head_dim, grid, max_q_len, stream);
      } else {
        if (fp8) launch_prefill<RLT_F16, RLT_FP8_E4M3>(P, head_dim, grid, max_q_len, stream);
        else launch_prefill<RLT_F16, RLT_F16>(P, head_dim, grid, max_q_len, stream);
      }
      return rlt_launch_status();
    }
    const int nt = (rows_per_seq > 16 && head_dim <= 128) ? 2 : 1;
    P.rows_per_rg = 16 * nt;
    P.rowgroups = (rows_per_seq + P.rows_per_rg - 1) / P.rows_per_rg;
    if (P.rowgroups < 1) P.rowgroups = 1;
    // Persistent workgroups, one per CU, unless the pair index does not fit in LDS.
    P.head_groups = num_kv_heads;
    const int64_t pairs = (int64_t)num_seqs * P.rowgroups;
    const bool blocks = scale_mode == 3 && whole_tiles(P);
    P.direct = blocks;
    P.persistent = pairs <= (blocks ? rlt_attn::kMaxBlockPairs : kMaxPairs);
    // (not with an fp8 store of 32 rows or more: quantizing them is a good part of its unit's time,
    // and neighbouring heads of the chunk that holds the window put such units on the same
    // workgroups.  8 windows of up to 24 / 32 / 48 / 63 rows behind 3000, 55 heads of 96, apart
    // and together: 111 / 130 / 198 / 214 and 111 / 130 / 238 / 272 us, 24 at 2000: 207 / 220 / 394
    // / 422 and 204 / 233 / 402 / 439; 24 windows of up to 5 / 16 rows: 162 / 188 and 147 / 178)
    const bool long_store = store && kv_dtype == RLT_FP8_E4M3 && max_q_len >= 32;
    P.shared_lines = num_kv_heads > 1 && !long_store &&
                     ((k_head_stride * kv_elt) % 128 != 0 || (v_head_stride * kv_elt) % 128 != 0 ||
                      (scale_mode == 2 && s_head_stride * 4 < 128));
    int64_t wgs = (int64_t)num_seqs * P.rowgroups * num_kv_heads * P.max_chunks;
    if (P.persistent)
      wgs = (int64_t)compute_units() * (blocks ? rlt_attn::block_groups_per_cu(head_dim, nt) : 1);
    if (wgs >= ((int64_t)1 << 31)) return RLT_ERR_UNSUPPORTED;
    dim3 grid((unsigned)wgs);
    if (kv_dtype == RLT_INT8)
      st = rlt_attn::launch_block_int8(P, q_dtype, grid, nt, whole_tiles(P), stream);
    else if (scale_mode == 3 && (whole_tiles(P) || !P.compensate))
      st = rlt_attn::launch_block_fp8(P, q_dtype, grid, nt, whole_tiles(P), stream);
    else if (q_dtype == RLT_BF16)
      st = kv_dtype == RLT_BF16 ? launch_mfma<RLT_BF16, RLT_BF16>(P, grid, nt, stream)
                                : launch_mfma<RLT_BF16, RLT_FP8_E4M3>(P, grid, nt, stream);
    else
      st = kv_dtype == RLT_F16 ? launch_mfma<RLT_F16, RLT_F16>(P, grid, nt, stream)
                               : launch_mfma<RLT_F16, RLT_FP8_E4M3>(P, grid, nt, stream);
  } else {
    if (scale_mode == 3) P.scale_mode = 2;  // (token stride 0)
    P.rows_per_rg = kVecRows;
    P.rowgroups = (rows_per_seq + kVecRows - 1) / kVecRows;
    if (P.rowgroups < 1) P.rowgroups = 1;
    P.head_groups = num_kv_heads;
    P.persistent = 0;
    P.shared_lines = 0;
    const int64_t wgs = (int64_t)num_seqs * P.rowgroups * P.head_groups * P.max_chunks;
    if (wgs >= ((int64_t)1 << 31)) return RLT_ERR_UNSUPPORTED;
    dim3 grid((unsigned)wgs);
    switch (q_dtype) {
      case RLT_F32: st = launch_vec_q<RLT_F32>(P, kv_dtype, grid, stream); break;
      case RLT_F16: st = launch_vec_q<RLT_F16>(P, kv_dtype, grid, stream); break;
      case RLT_BF16: st = launch_vec_q<RLT_BF16>(P, kv_dtype, grid, stream); break;
      default: st = RLT_ERR_ARGUMENT;
    }
  }
  if (st != RLT_OK) return st;
  if (P.direct && P.max_chunks <= 1) return rlt_launch_status();
  P.max_q = cu_seqlens_q ? max_q_len : 1;
  const int64_t merge_rows = cu_seqlens_q ? (int64_t)num_seqs * max_q_len : num_q_rows;
  if (merge_rows >= ((int64_t)1 << 31)) return RLT_ERR_UNSUPPORTED;
  dim3 mgrid((unsigned)merge_rows, (unsigned)((num_q_heads + 3) / 4));
  switch (q_dtype) {
    case RLT_F32: launch_merge<RLT_F32>(P, mgrid, stream); break;
    case RLT_F16: launch_merge<RLT_F16>(P, mgrid, stream); break;
    case RLT_BF16: launch_merge<RLT_BF16>(P, mgrid, stream); break;
  }
  return rlt_launch_status();
}

}  // namespace

extern "C" {

int rlt_paged_attention_rows(const void* q, int64_t q_row_stride, int64_t q_head_stride,
                             const void* key_cache, const void* value_cache, int64_t k_block_stride,
                             int64_t k_token_stride, int64_t k_head_stride, int64_t v_block_stride,
                             int64_t v_token_stride, int64_t v_head_stride, int32_t num_blocks,
                             const int32_t* block_tables, int64_t table_stride, int32_t table_width,
                             const int32_t* context_lengths, const int32_t* row_lengths,
                             const int32_t* cu_seqlens_q, int32_t num_seqs, int32_t max_q_len,
                             int32_t num_q_rows, const float* key_scale, const float* value_scale,
                             int32_t scale_mode, int64_t s_block_stride, int64_t s_token_stride,
                             int64_t s_head_stride, int32_t num_q_heads, int32_t num_kv_heads,
                             int32_t head_dim, int32_t block_size, int32_t q_dtype, int32_t kv_dtype,
                             int32_t window, int32_t flags, void* out, int64_t out_row_stride,
                             int64_t out_head_stride, void* workspace, size_t workspace_bytes,
                             hipStream_t stream) {
  return attention_impl(q, q_row_stride, q_head_stride, key_cache, value_cache, k_block_stride,
                        k_token_stride, k_head_stride, v_block_stride, v_token_stride,
                        v_head_stride, num_blocks, block_tables, table_stride, table_width,
                        context_lengths, row_lengths, cu_seqlens_q, num_seqs, max_q_len,
                        num_q_rows, key_scale, value_scale, scale_mode, s_block_stride,
                        s_token_stride, s_head_stride, num_q_heads, num_kv_heads, head_dim,
                        block_size, q_dtype, kv_dtype, window, flags, out, out_row_stride,
                        out_head_stride, workspace, workspace_bytes, stream, nullptr);
}

int rlt_paged_attention_store(const void* q, int64_t q_row_stride, int64_t q_head_stride,
                              void* key_cache, void* value_cache, int64_t k_block_stride,
                              int64_t k_token_stride, int64_t k_head_stride, int64_t v_block_stride,
                              int64_t v_token_stride, int64_t v_head_stride, int32_t num_blocks,
                              const int32_t* block_tables, int64_t table_stride,
                              int32_t table_width, const int32_t* context_lengths,
                              const int32_t* cu_seqlens_q, int32_t num_seqs, int32_t max_q_len,
                              int32_t num_q_rows, int32_t num_q_heads, int32_t num_kv_heads,
                              int32_t head_dim, int32_t block_size, int32_t dtype,
                              const void* new_k, const void* new_v, int64_t new_row_stride,
                              int64_t new_head_stride, void* out, int64_t out_row_stride,
                              int64_t out_head_stride, void* workspace, size_t workspace_bytes,
                              hipStream_t stream) {
  const WindowStore st{new_k, new_v, new_row_stride, new_head_stride};
  return attention_impl(q, q_row_stride, q_head_stride, key_cache, value_cache, k_block_stride,
                        k_token_stride, k_head_stride, v_block_stride, v_token_stride,
                        v_head_stride, num_blocks, block_tables, table_stride, table_width,
                        context_lengths, nullptr, cu_seqlens_q, num_seqs, max_q_len, num_q_rows,
                        nullptr, nullptr, 0, 0, 0, 0, num_q_heads, num_kv_heads, head_dim,
                        block_size, dtype, dtype, 0, 0, out, out_row_stride, out_head_stride,
                        workspace, workspace_bytes, stream, &st);
}

int rlt_paged_attention_store_scaled(
    const void* q, int64_t q_row_stride, int64_t q_head_stride, void* key_cache,
    void* value_cache, int64_t k_block_stride, int64_t k_token_stride, int64_t k_head_stride,
    int64_t v_block_stride, int64_t v_token_stride, int64_t v_head_stride, int32_t num_blocks,
    const int32_t* block_tables, int64_t table_stride, int32_t table_width,
    const int32_t* context_lengths, const int32_t* row_lengths, const int32_t* cu_seqlens_q,
    int32_t num_seqs, int32_t max_q_len, int32_t num_q_rows, float* key_scale, float* value_scale,
    int32_t scale_mode, int64_t s_block_stride, int64_t s_token_stride, int64_t s_head_stride,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
    int32_t q_dtype, int32_t kv_dtype, int32_t flags, const void* new_k, const void* new_v,
    int64_t new_row_stride, int64_t new_head_stride, void* out, int64_t out_row_stride,
    int64_t out_head_stride, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  const WindowStore st{new_k, new_v, new_row_stride, new_head_stride};
  return attention_impl(q, q_row_stride, q_head_stride, key_cache, value_cache, k_block_stride,
                        k_token_stride, k_head_stride, v_block_stride, v_token_stride,
                        v_head_stride, num_blocks, block_tables, table_stride, table_width,
                        context_lengths, row_lengths, cu_seqlens_q, num_seqs, max_q_len,
                        num_q_rows, key_scale, value_scale, scale_mode, s_block_stride,
                        s_token_stride, s_head_stride, num_q_heads, num_kv_heads, head_dim,
                        block_size, q_dtype, kv_dtype, 0, flags, out, out_row_stride,
                        out_head_stride, workspace, workspace_bytes, stream, &st);
}

int rlt_paged_attention(const void* q, int64_t q_row_stride, int64_t q_head_stride,
                        const void* key_cache, const void* value_cache, int64_t k_block_stride,
                        int64_t k_token_stride, int64_t k_head_stride, int64_t v_block_stride,
                        int64_t v_token_stride, int64_t v_head_stride, int32_t num_blocks,
                        const int32_t* block_tables, int64_t table_stride, int32_t table_width,
                        const int32_t* context_lengths,
                        const int32_t* cu_seqlens_q, int32_t num_seqs, int32_t max_q_len,
                        int32_t num_q_rows, const float* key_scale, const float* value_scale,
                        int32_t scale_mode, int64_t s_block_stride, int64_t s_token_stride,
                        int64_t s_head_stride, int32_t num_q_heads, int32_t num_kv_heads,
                        int32_t head_dim, int32_t block_size, int32_t q_dtype, int32_t kv_dtype,
                        int32_t window, void* out, int64_t out_row_stride, int64_t out_head_stride,
                        void* workspace, size_t workspace_bytes, hipStream_t stream) {
  return rlt_paged_attention_rows(
      q, q_row_stride, q_head_stride, key_cache, value_cache, k_block_stride, k_token_stride,
      k_head_stride, v_block_stride, v_token_stride, v_head_stride, num_blocks, block_tables,
      table_stride, table_width, context_lengths, nullptr, cu_seqlens_q, num_seqs, max_q_len,
      num_q_rows, key_scale, value_scale, scale_mode, s_block_stride, s_token_stride,
      s_head_stride, num_q_heads, num_kv_heads, head_dim, block_size, q_dtype, kv_dtype, window, 0,
      out, out_row_stride, out_head_stride, workspace, workspace_bytes, stream);
}

}  // extern "C"
