// Attention over 8-bit pools (e4m3 or int8 codes) with one scale per block of tokens and kv head,
// for single rows and verify windows; prompts take the prefill tiling of paged_attention.h.
//
//   out = sum_t w_t s_v[b(t)] c_v(t) / sum_t w_t,  w_t = exp(q . c_k(t) s_k[b(t)] / sqrt(D) - m)
//
// What bounds it: HBM reads.  64 rows at 16k-32k positions of 8 heads in int8, 3.18 GB: 611 us with
// the merge, 5.2 TB/s (1 GB: 218 us), whatever the kv heads, block size, loads in flight (one or
// two pairs of tiles) and waves (8 or 12 a CU); a unit's first loads issued before the one
// ahead of it is combined gain nothing (616), non-temporal loads are slower (629).  Windows of 5
// over GQA 4, 157 MB, 47 us: one or two units a workgroup, each a chain of lengths -> table ->
// tiles -> combine; one row at 700 positions 11.9 us.
//
// Work.  A unit is (sequence, row-group, kv head, chunk): 1024 absolute key positions, a quarter
// of them to each of a workgroup's four waves, whose softmax states (maximum, sum,
// unnormalized output) are combined through LDS in part order.  (Chunks of 512 leave twice the
// partials: 611 -> 656 us; a wave alone on a chunk, 36 us for the one row.)  A row whose keys lie in one chunk
// is normalized there; others leave a partial per chunk for rlt_merge_kernel.  Persistent
// workgroups, as many as share the CUs' registers, take the units of all sequences in turn, as
// rlt_attn_mfma_kernel does; a row's arithmetic depends on its own keys and absolute positions
// alone, so that packed rows equal single rows bit for bit, whatever the batch.
//
// A wave takes pairs of 16-position tiles: S^T = K Q^T by v_mfma_f32_16x16x32, straight from
// memory (paged_attention.h's operand orders); O^T += V^T P^T by the same instruction, the pair's
// 32 positions as one contraction.  A lane holds the place and the two scales of one tile of
// its span, looked up once, which a tile takes by lane reads into scalar registers: no table, no
// division and no scale load inside the stream.  The key scale enters with the exponent's one
// fma.  The product with the values is fp16's whatever q's type: codes are exact in it, and it rounds
// a weight to 11 bits (outputs 1.05 times as far from float64 as one of float32 weights, rounded to
// bf16; with bf16 weights 1.42 times).  Its weights take the value scale over a power of two near
// the largest that their row sees in the span (the row's own, as the maximum, or rows would
// round by what those beside them see: 0.4 us of the one row's 12), which the output takes back, and
// lie 2^kBlockLift above their place, since fp16's normal numbers end at 2^-14.  The running maximum moves only when it is passed by
// 2^kBlockLazy, and sums stay with the lanes until the end.
#pragma once

#include "paged_attention.h"

namespace rlt_attn {

// Positions of a chunk (their log2), and persistent workgroups that share a CU.
int block_chunk_log2();
int block_groups_per_cu(int head_dim, int nt);
// The verify kernels (`whole`: blocks hold whole 16-position tiles and a lane's offset within
// one fits 32 bits; other blocks take their scales position by position) and the prefill tiling.
int launch_block_fp8(const AttnParams& P, int q_dtype, dim3 grid, int nt, bool whole, hipStream_t stream);
int launch_block_int8(const AttnParams& P, int q_dtype, dim3 grid, int nt, bool whole, hipStream_t stream);
void launch_block_prefill_fp8(const AttnParams& P, int q_dtype, dim3 grid, bool whole, hipStream_t stream);
void launch_block_prefill_int8(const AttnParams& P, int q_dtype, dim3 grid, bool whole, hipStream_t stream);

// (sequence, row-group) pairs that the persistent form lists
constexpr int kMaxBlockPairs = 1024;
// Workgroups of one launch: a grid holds fewer than 2^32 threads, and a call may ask for more (its
// tables and windows are padded to the longest); those behind go into further launches.
constexpr unsigned kBlockGrid = 1u << 23;

}  // namespace rlt_attn

namespace {

constexpr int kBlockParts = 4;                           // waves of a unit
constexpr int kBlockChunk = 1024;
constexpr int kBlockSpan = kBlockChunk / kBlockParts;    // positions of a wave
constexpr float kBlockLazy = 4.f;                        // log2 headroom before the running maximum moves
constexpr int kBlockLift = 15 - (int)kBlockLazy;
// registers: 168 hold one row tile of up to 128 dims, 256 the others
template <int D, int NT>
constexpr int block_waves_per_simd() { return D <= 128 && NT == 1 ? 3 : 2; }

template <int NT, int D>
struct BlockShared {
  static constexpr int kStride = D + 4;  // floats of a row: 16-byte accesses of 16 rows meet all banks
  alignas(16) float o[kBlockParts][16 * NT * kStride];
  float ml[kBlockParts][16 * NT][2];
  int64_t out_at[16 * NT], slot[16 * NT];
  int chunks[16 * NT];  // of the row: 0, 1 (written here), more; -1: the chunk is not among them
  int32_t first[rlt_attn::kMaxBlockPairs + 1], c0[rlt_attn::kMaxBlockPairs];
  int32_t wave_total[kBlockParts];
};

// Keys as paged_attention.h's slices, but for 96 dims, whose 96-byte vectors take fewer loads in other
// pieces: a lane group's 24 consecutive key codes in two (three 8-byte ones).  With the values'
// (BlockValues), 16 windows of 16 rows, 2048 positions, 55 heads: 133 -> 96 us.
template <int QT, int KVT, int D>
struct BlockKeys : RawSlice<QT, KVT, D> {};
template <int QT, int KVT>
struct BlockKeys<QT, KVT, 96> {
  static constexpr int kGroupElems = 24;
  uint32_t w[6];
  __device__ static constexpr int element(int s, int g) { return 24 * g + 8 * s; }
  __device__ __forceinline__ void load(const uint8_t* p) { __builtin_memcpy(w, __builtin_assume_aligned(p, 8), 24); }
  __device__ __forceinline__ uint4 op(int s) const {
    const uint2 a = codes_to_16<QT, KVT>(w[2 * s]), b = codes_to_16<QT, KVT>(w[2 * s + 1]);
    return make_uint4(a.x, a.y, b.x, b.y);
  }
};

// A row-group's chunks [c0, c1); one that sees nothing takes chunk 0, which writes its zeros.
__device__ __forceinline__ void block_chunks(const AttnParams& P, int p, int& c0, int& c1) {
  pair_chunks<kBlockChunk>(P, p, c0, c1);
  if (c0 == c1) {
    const int seq = p / P.rowgroups;
    const bool rows = (p - seq * P.rowgroups) * P.rows_per_rg < seq_view(P, seq).q_len * P.group;
    c0 = 0;
    c1 = rows ? 1 : 0;
  }
}

// One wave's part of a unit; its state goes to sh.o / sh.ml[part].
template <int QT, int KVT, int D, int NT, bool CP>
__device__ __forceinline__ void block_part(const AttnParams& P, const SeqView& sv, int seq, int rg_begin, int rg_rows,
                                           int kvh, int w_begin, int part, BlockShared<NT, D>& sh) {
  using M = Mfma<QT>;
  using W = Mfma<RLT_F16>;  // weights and values
  using KeySlice = BlockKeys<QT, KVT, D>;
  using VQ = BlockValues<RLT_F16, KVT, D>;
  constexpr int NQS = D / 32;  // 32-wide contraction slices
  constexpr int ND = D / 16;   // 16-wide output column tiles (= dims per lane)
  const int lane = threadIdx.x & 63, l16 = lane & 15, grp = lane >> 4;

  int lo_first, hi_first, lo_last, hi_last;
  group_range(P, sv, rg_begin, rg_rows, lo_first, hi_first, lo_last, hi_last);
  // visible tiles [v0, t1) of the span, as absolute 16-position tiles from w_begin on; pairs begin
  // at even ones, so that a row's pairs do not depend on the rows beside it
  const int v0 = __builtin_amdgcn_readfirstlane(max(0, (lo_first - w_begin) >> 4));
  const int t1 = __builtin_amdgcn_readfirstlane(
      (min(kBlockSpan, max(0, min(hi_last - w_begin, kBlockSpan))) + kTileTok - 1) / kTileTok);
  if (v0 >= t1) {
    if (lane < 16) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        sh.ml[part][nt * 16 + lane][0] = -INFINITY;
        sh.ml[part][nt * 16 + lane][1] = 0.f;
      }
    }
    return;
  }
  const int t0 = v0 & ~1, tl = t1 - 1;

  // this lane's tile: where its keys and values begin, and its scales
  int64_t k_at, v_at, s_at;
  {
    const int pos = w_begin + min(max(lane, v0), tl) * kTileTok, idx = pos / P.block_size;
    const int32_t e = P.tables[(int64_t)seq * P.table_stride + min(idx, P.table_width - 1)];
    const int64_t blk = (e >= 0 && e < P.num_blocks) ? e : 0;
    const int off = pos - idx * P.block_size;
    k_at = blk * P.k_block_stride + off * P.k_token_stride + (int64_t)kvh * P.k_head_stride;
    v_at = blk * P.v_block_stride + off * P.v_token_stride + (int64_t)kvh * P.v_head_stride;
    s_at = blk * P.s_block_stride + (int64_t)kvh * P.s_head_stride;
  }
  auto tile_at = [&](int64_t x, int t) {
    const int tt = min(t, tl);  // (past the last tile: that one again)
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, tt);
    return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), tt) << 32) | lo);
  };
  auto tile_scale = [&](float x, int t) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), min(t, tl)));
  };
  KeySlice kb[2];
  VQ vq[2];
  const uint32_t k_lane = (uint32_t)(l16 * (uint32_t)P.k_token_stride + grp * KeySlice::kGroupElems);
  const uint32_t v_lane = (uint32_t)(4 * grp * (uint32_t)P.v_token_stride + VQ::lane_bytes(l16));
  auto issue_k = [&](int t, int b) { kb[b].load((const uint8_t*)P.k + tile_at(k_at, t) + k_lane); };
  auto issue_v = [&](int t, int b) {
    const uint8_t* base = (const uint8_t*)P.v + tile_at(v_at, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) vq[b].load(i, base + (int64_t)i * P.v_token_stride + v_lane);
  };
#pragma unroll
  for (int b = 0; b < 2; ++b) issue_k(t0 + b, b);
  float k_tile = P.k_scale[s_at], v_tile = P.v_scale[s_at];
#pragma unroll
  for (int b = 0; b < 2; ++b) issue_v(t0 + b, b);

  // this lane's rows (one per 16-row tile): B operand of S^T = K Q^T
  uint4 qreg[NT][NQS];
  int row_lo[NT], row_hi[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int rho = rg_begin + nt * 16 + l16;
    row_lo[nt] = row_hi[nt] = 0;
    if (nt * 16 + l16 < rg_rows) {
      const int qi = rho / P.group;
      row_range(P, sv, qi, row_lo[nt], row_hi[nt]);
      const uint16_t* qp = (const uint16_t*)P.q + (int64_t)(sv.q_begin + qi) * P.q_row_stride +
                           (int64_t)(kvh * P.group + rho % P.group) * P.q_head_stride;
#pragma unroll
      for (int s = 0; s < NQS; ++s) qreg[nt][s] = *(const uint4*)(qp + KeySlice::element(s, grp));
    } else {
#pragma unroll
      for (int s = 0; s < NQS; ++s) qreg[nt][s] = make_uint4(0, 0, 0, 0);
    }
  }

  f32x4 oacc[NT][ND];
  float m_run[NT], l_run[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m_run[nt] = -INFINITY;
    l_run[nt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt) oacc[nt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // (scales are positive; one of 0 counts as the smallest normal number: a masked score times it
  // stays -inf)
  k_tile *= P.qk_scale_log2;
  k_tile = k_tile < 1.17549435e-38f ? 1.17549435e-38f : k_tile;
  // the power of two that a row's weights are taken over: of the largest value scale among the tiles
  // that it sees itself, whatever the rows beside it see
  int v_exp[NT];
  {
    float most[NT];
    if (lo_last < w_begin + (v0 + 1) * kTileTok && hi_first > w_begin + tl * kTileTok) {
      // (every row sees some of the first and the last tile, and so all, which lanes 0 to 15 hold)
      float all = fabsf(v_tile);
      auto turned = [&](auto ctrl) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(all), decltype(ctrl)::value, 0xf, 0xf, false));
      };
      all = fmaxf(all, turned(std::integral_constant<int, 0x128>{}));  // lanes 8 on, of 16
      all = fmaxf(all, turned(std::integral_constant<int, 0x124>{}));
      all = fmaxf(all, turned(std::integral_constant<int, 0x122>{}));
      all = fmaxf(all, turned(std::integral_constant<int, 0x121>{}));
      all = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(all)));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) most[nt] = all;
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) most[nt] = 0.f;
#pragma unroll 1
      for (int t = v0; t < t1; ++t) {
        const float x = fabsf(tile_scale(v_tile, t));
        const int tb = w_begin + t * kTileTok;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          most[nt] = tb < row_hi[nt] && tb + kTileTok > row_lo[nt] ? fmaxf(most[nt], x) : most[nt];
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      v_exp[nt] = (most[nt] > 0.f ? __builtin_amdgcn_frexp_expf(most[nt]) : 0) - kBlockLift;
  }

  // pairs inside [full_lo, full_hi) are visible to every row
  const int span_end = w_begin + kBlockSpan;
  const int full_lo = lo_last, full_hi = min(hi_first, span_end);
  auto pair = [&](int t) {
    const int tb = w_begin + t * kTileTok;
    const bool full = tb >= full_lo && tb + 2 * kTileTok <= full_hi;
    // ---- S^T = K Q^T : lane holds (positions tb + 16 b + 4 * grp + r, row l16 of tile nt)
    f32x4 sc[2][NT];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sc[b][nt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < NQS; ++s) {
        const uint4 a = kb[b].op(s);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) sc[b][nt] = M::qk(a, qreg[nt][s], sc[b][nt]);
      }
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) issue_k(t + 2 + b, b);
    __builtin_amdgcn_sched_barrier(0);
    // ---- weights: contraction slot 8 grp + 4 b + r of P^T is position 16 b + 4 grp + r
    if (!full) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int pos = tb + b * kTileTok + 4 * grp + r;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            sc[b][nt][r] = (pos >= row_lo[nt] && pos < min(row_hi[nt], span_end)) ? sc[b][nt][r] : -INFINITY;
        }
    }
    const float f0 = tile_scale(k_tile, t), f1 = tile_scale(k_tile, t + 1);
    const float s0 = tile_scale(v_tile, t), s1 = tile_scale(v_tile, t + 1);
    float g0[NT], g1[NT], mx[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      g0[nt] = __builtin_amdgcn_ldexpf(s0, -v_exp[nt]);
      g1[nt] = __builtin_amdgcn_ldexpf(s1, -v_exp[nt]);
      if (!full) {
        // (the scale of a tile that the row does not see is any multiple of its largest)
        const int lo = row_lo[nt] - tb, hi = row_hi[nt] - tb;
        g0[nt] = hi > 0 && lo < kTileTok ? g0[nt] : 0.f;
        g1[nt] = hi > kTileTok && lo < 2 * kTileTok ? g1[nt] : 0.f;
      }
    }
    bool grow = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const f32x4 &a = sc[0][nt], &b = sc[1][nt];
      mx[nt] = group_max(fmaxf(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])) * f0,
                               fmaxf(fmaxf(b[0], b[1]), fmaxf(b[2], b[3])) * f1));
      grow |= mx[nt] > m_run[nt] + kBlockLazy;
    }
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const bool up = mx[nt] > m_run[nt] + kBlockLazy;
        const float corr = up ? __builtin_amdgcn_exp2f(m_run[nt] - mx[nt]) : 1.f;
        m_run[nt] = up ? mx[nt] : m_run[nt];
        l_run[nt] *= corr;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) oacc[nt][dt] *= corr;
      }
    }
    uint4 p[NT], dropped[CP ? NT : 1];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // (a row that has seen no key keeps weights of 0)
      const float m = m_run[nt] == -INFINITY ? 0.f : m_run[nt];
      float x[2][4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[0][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[0][nt][r], f0, -m));
        x[1][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[1][nt][r], f1, -m));
      }
      l_run[nt] += ((x[0][0] + x[0][1]) + (x[0][2] + x[0][3])) + ((x[1][0] + x[1][1]) + (x[1][2] + x[1][3]));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[0][r] *= g0[nt];
        x[1][r] *= g1[nt];
      }
      p[nt] = make_uint4(W::pack2(x[0][0], x[0][1]), W::pack2(x[0][2], x[0][3]),
                         W::pack2(x[1][0], x[1][1]), W::pack2(x[1][2], x[1][3]));
      if (CP) {
        auto rest = [&](uint32_t w, float a, float b) { return W::pack2(a - W::lo_f32(w), b - W::hi_f32(w)); };
        dropped[nt] = make_uint4(rest(p[nt].x, x[0][0], x[0][1]), rest(p[nt].y, x[0][2], x[0][3]),
                                 rest(p[nt].z, x[1][0], x[1][1]), rest(p[nt].w, x[1][2], x[1][3]));
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int b = 0; b < 2; ++b) vq[b].arrange(l16);
    // codes that no row sees may be any (NaN included)
    if (!full) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int pos = tb + b * kTileTok + 4 * grp + i;
          if (pos < lo_first || pos >= hi_last) vq[b].zero(i);
        }
    }
    // ---- O^T += V^T P^T : A = V^T (dims ND * l16 + dt, positions as in P^T)
    for_pairs<ND, NT>([&](auto kc) {
      constexpr int K = decltype(kc)::value;
      if (D > 128) __builtin_amdgcn_sched_barrier(0);  // (no registers left to run ahead)
      uint2 a0, a1, b0, b1;
      vq[0].template op2<K>(a0, a1);
      vq[1].template op2<K>(b0, b1);
      const uint4 v0 = make_uint4(a0.x, a0.y, b0.x, b0.y), v1 = make_uint4(a1.x, a1.y, b1.x, b1.y);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        oacc[nt][2 * K] = W::qk(v0, p[nt], oacc[nt][2 * K]);
        oacc[nt][2 * K + 1] = W::qk(v1, p[nt], oacc[nt][2 * K + 1]);
        if (CP) {
          oacc[nt][2 * K] = W::qk(v0, dropped[nt], oacc[nt][2 * K]);
          oacc[nt][2 * K + 1] = W::qk(v1, dropped[nt], oacc[nt][2 * K + 1]);
        }
      }
    });
#pragma unroll
    for (int b = 0; b < 2; ++b) issue_v(t + 2 + b, b);
  };
#pragma unroll 1
  for (int t = t0; t < t1; t += 2) pair(t);

#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const float back = __builtin_amdgcn_ldexpf(1.f, v_exp[nt]);
    const float l = group_sum(l_run[nt]);
    const int row = nt * 16 + l16;
    if (grp == 0) {
      sh.ml[part][row][0] = m_run[nt];
      sh.ml[part][row][1] = l;
    }
    // accumulator element r of column tile dt is dim ND * (4 * grp + r) + dt
    float* const to = sh.o[part] + row * BlockShared<NT, D>::kStride + 4 * grp * ND;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if constexpr (ND % 4 == 0) {
#pragma unroll
        for (int d = 0; d < ND; d += 4)
          *(f32x4*)(to + r * ND + d) = f32x4{oacc[nt][d][r] * back, oacc[nt][d + 1][r] * back,
                                             oacc[nt][d + 2][r] * back, oacc[nt][d + 3][r] * back};
      } else {
#pragma unroll
        for (int d = 0; d < ND; d += 2)
          *(float2*)(to + r * ND + d) = make_float2(oacc[nt][d][r] * back, oacc[nt][d + 1][r] * back);
      }
    }
  }
}

// Units as rlt_attn_mfma_kernel's: each full round of the grid takes consecutive ones on the
// workgroups of one XCD (b % 8), which share their scales' and narrow heads' cache lines; the
// last, when it is not full, spreads over the XCDs.
template <int QT, int KVT, int D, int NT, bool CP>
__global__ __launch_bounds__(64 * kBlockParts, (block_waves_per_simd<D, NT>()))
void rlt_block_attention_kernel(AttnParams P) {
  __shared__ BlockShared<NT, D> sh;
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int pairs = P.num_seqs * P.rowgroups;
  int units = 1, G = 1, b = 0;
  if (P.persistent) {
    // units before each pair: per thread over a run of pairs, then scans over lanes and waves
    const int per = (pairs + 64 * kBlockParts - 1) / (64 * kBlockParts);
    const int p_lo = min(pairs, t * per), p_hi = min(pairs, p_lo + per);
    int run = 0;
    for (int p = p_lo; p < p_hi; ++p) {
      int c0, c1;
      block_chunks(P, p, c0, c1);
      sh.c0[p] = c0;
      sh.first[p] = run;
      run += (c1 - c0) * P.hkv;
    }
    int incl = run;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(incl, off, RLT_WAVE);
      if (lane >= off) incl += y;
    }
    if (lane == 63) sh.wave_total[wave] = incl;
    __syncthreads();
    int base = incl - run;
    for (int w = 0; w < wave; ++w) base += sh.wave_total[w];
    for (int p = p_lo; p < p_hi; ++p) sh.first[p] += base;
    if (t == 64 * kBlockParts - 1) sh.first[pairs] = base + run;
    __syncthreads();
    units = sh.first[pairs];
    G = gridDim.x;
    b = blockIdx.x;
  }
  const int rounds = units / G, rest = units - rounds * G;
  for (int k = 0; k < rounds + (b < rest ? 1 : 0); ++k) {
    int seq, rg, kvh, chunk, c0;
    if (P.persistent) {
      const int u = k < rounds && G % 8 == 0 ? k * G + (b & 7) * (G / 8) + (b >> 3) : k * G + b;
      unit_of(P, sh.first, sh.c0, pairs, u, seq, rg, kvh, chunk);
      c0 = sh.c0[seq * P.rowgroups + rg];
    } else {
      // (more pairs than are listed: a workgroup each)
      const WorkItem wi = work_item(P, P.first_group + blockIdx.x);
      seq = wi.seq;
      rg = wi.rg;
      kvh = wi.hg;
      chunk = wi.chunk;
      int c1;
      block_chunks(P, seq * P.rowgroups + rg, c0, c1);
      if (chunk < c0 || chunk >= c1) return;
    }
    seq = __builtin_amdgcn_readfirstlane(seq);
    rg = __builtin_amdgcn_readfirstlane(rg);
    kvh = __builtin_amdgcn_readfirstlane(kvh);
    chunk = __builtin_amdgcn_readfirstlane(chunk);
    const SeqView sv = seq_view(P, seq);
    const int rg_begin = rg * P.rows_per_rg;
    const int rg_rows = min(P.rows_per_rg, sv.q_len * P.group - rg_begin);
    if (t < rg_rows) {
      const int qi = (rg_begin + t) / P.group, head = kvh * P.group + (rg_begin + t) % P.group;
      int lo, hi;
      row_range(P, sv, qi, lo, hi);
      const int first = lo / kBlockChunk, last = (hi + kBlockChunk - 1) / kBlockChunk;
      // (rows that see nothing are written once, by the row-group's first unit)
      sh.chunks[t] = hi <= lo ? (chunk == c0 ? 0 : -1) : chunk < first || chunk >= last ? -1 : last - first;
      sh.slot[t] = ((int64_t)(sv.q_begin + qi) * P.hq + head) * P.max_chunks + chunk;
      sh.out_at[t] = (int64_t)(sv.q_begin + qi) * P.out_row_stride + (int64_t)head * P.out_head_stride;
    }
    block_part<QT, KVT, D, NT, CP>(P, sv, seq, rg_begin, rg_rows, kvh, chunk * kBlockChunk + wave * kBlockSpan, wave, sh);
    __syncthreads();
    // ---- the parts' states combined, four dims a thread
    for (int e = t; e < rg_rows * (D / 4); e += 64 * kBlockParts) {
      const int row = e / (D / 4), d = 4 * (e % (D / 4));
      const int chunks = sh.chunks[row];
      if (chunks < 0) continue;
      float m = -INFINITY, l = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kBlockParts; ++i) m = fmaxf(m, sh.ml[i][row][0]);
#pragma unroll
      for (int i = 0; i < kBlockParts; ++i) {
        const float mi = sh.ml[i][row][0], li = sh.ml[i][row][1];
        if (mi == -INFINITY && li == 0.f) continue;  // (a part without a key)
        // (scores that are all NaN leave no maximum, and a NaN for a sum)
        const float s = mi == -INFINITY ? li : __builtin_amdgcn_exp2f(mi - m);
        l += li * s;
        o += *(const f32x4*)(sh.o[i] + row * BlockShared<NT, D>::kStride + d) * s;
      }
      if (chunks <= 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint16_t* const to = (uint16_t*)P.out + sh.out_at[row] + d;
        const uint32_t x = Mfma<QT>::pack2(o[0] * inv, o[1] * inv), y = Mfma<QT>::pack2(o[2] * inv, o[3] * inv);
        to[0] = (uint16_t)x;
        to[1] = (uint16_t)(x >> 16);
        to[2] = (uint16_t)y;
        to[3] = (uint16_t)(y >> 16);
      } else {
        *(f32x4*)(P.part_o + sh.slot[row] * D + d) = o;
        if (d == 0) *(float2*)(P.part_ml + 2 * sh.slot[row]) = make_float2(m, l);
      }
    }
    __syncthreads();  // the buffers are reused by the next unit
  }
}

// Where a workgroup for every (row-group, kv head, chunk) of the tables fits on the CUs at once,
// each takes its own, without the list of units (two barriers and the lengths of all sequences:
// one row at 700 positions 12.0 -> 11.4 us, 8 windows of 5 at 2-4k 23.2 -> 22.2); more of them
// than that would leave the order in which they read to the dispatcher (64 rows at 512-4096,
// 16 heads: 142 us, and 183 so).
template <int QT, int KVT, int D, bool CP>
int launch_block_cp(AttnParams P, dim3 grid, int nt, hipStream_t stream) {
  const int64_t all = (int64_t)P.num_seqs * P.rowgroups * P.hkv * P.max_chunks;
  if (P.persistent && all <= (int64_t)grid.x) {
    P.persistent = 0;
    grid = dim3((unsigned)all);
  }
  if (nt != 1 && D > 128) return RLT_ERR_UNSUPPORTED;
  for (unsigned left = grid.x; left; left -= grid.x, P.first_group += grid.x) {
    grid.x = left < rlt_attn::kBlockGrid ? left : rlt_attn::kBlockGrid;
    if (nt == 1) rlt_block_attention_kernel<QT, KVT, D, 1, CP><<<grid, 64 * kBlockParts, 0, stream>>>(P);
    else rlt_block_attention_kernel<QT, KVT, D, (D <= 128 ? 2 : 1), CP><<<grid, 64 * kBlockParts, 0, stream>>>(P);
  }
  return RLT_OK;
}

template <int QT, int KVT, int D>
int launch_block_d(const AttnParams& P, dim3 grid, int nt, bool whole, hipStream_t stream) {
  if (whole) {
    if (P.compensate) return launch_block_cp<QT, KVT, D, true>(P, grid, nt, stream);
    return launch_block_cp<QT, KVT, D, false>(P, grid, nt, stream);
  }
  if (!P.compensate) return launch_mfma_ub<QT, KVT, D, 3, false, false>(P, grid, nt, stream);
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
void launch_block_prefill_d(AttnParams P, dim3 grid, bool whole, hipStream_t stream) {
  for (unsigned left = grid.x; left; left -= grid.x, P.first_group += grid.x) {
    grid.x = left < rlt_attn::kBlockGrid ? left : rlt_attn::kBlockGrid;
    if (whole) rlt_prefill_kernel<QT, KVT, D, 3, true><<<grid, kPfThreads, 0, stream>>>(P);
    else rlt_prefill_kernel<QT, KVT, D, 3, false><<<grid, kPfThreads, 0, stream>>>(P);
  }
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
