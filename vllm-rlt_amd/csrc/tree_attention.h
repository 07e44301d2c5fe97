// Attention of a tree of drafted tokens over a paged KV pool on MI355X (gfx950).
//
// Sequence s owns the q rows cu[s] .. cu[s + 1] - 1, the nodes of its draft tree, whose keys
// and values lie at the last N positions of its cache (node j at position len - N + j).  Node
// i sees the prefix [0, len - N) and the nodes j whose bit is set in its mask, and
//   out_i = sum_t softmax_t(q_i . k_t / sqrt(D)) v_t
// over them.  The rows that read one kv head -- (node, q head of its group), R = N * group of
// them -- share every key and value, so a pass is R flops per byte of a 16-bit pool (2 R of an
// fp8 one): the KV stream bounds it up to R ~ 200.
//
// Tiling.  A workgroup is four waves on one CU: RW row waves times KW = 4 / RW kv waves.  A
// row wave holds NT column tiles of 32 rows (v_mfma_f32_32x32x16: S^T = K Q^T, O^T += V^T P^T);
// each kv wave (group of RW waves) streams its own 32-position tiles, every KW-th of the
// workgroup's span, through a ring of S stages in LDS filled by direct global -> LDS loads.
// With RW = 1 no wave ever waits for another inside the stream, and a key is read from LDS
// once for up to 64 rows; more rows take two row waves that share the tiles.
//
// Schedule.  The keys of all (sequence, kv head, row block) pairs are one line of macro tiles
// (KW tiles each), of which every workgroup takes an equal share, whatever the mix of lengths.
// A pair inside one share is normalized where it is computed; a pair that crosses shares
// leaves one partial (maximum, sum, unnormalized output) per workgroup and
// rlt_tree_merge_kernel combines them in order.  A share is found from the lengths on the
// device, so the grid is static and the launch can be captured.
#pragma once

#include "common.h"

#include <math.h>

namespace tree {

constexpr int kWaves = 4;
constexpr int kTile = 32;          // key positions per LDS tile
constexpr int kGrid = 256;         // persistent workgroups: one per CU
constexpr int kMaxNodes = 256;     // nodes of one sequence's tree
constexpr int kWords = kMaxNodes / 64;
constexpr int kRingBytes = 128 << 10;
constexpr int kBadWords = kMaxNodes / kTile + 3;  // tiles that a range of kMaxNodes meets
constexpr float kLazy = 8.f;       // log2 headroom before the running max moves

struct Params {
  const void* q;
  int64_t q_row_stride, q_head_stride;
  const void* k;
  const void* v;
  int64_t k_block_stride, k_token_stride, k_head_stride;
  int64_t v_block_stride, v_token_stride, v_head_stride;
  const int32_t* tables;
  int64_t table_stride;
  int32_t table_width, num_blocks;
  const int32_t* lengths;
  const int32_t* cu_q;
  const uint64_t* mask;   // [q rows, words]: bit j % 64 of word j / 64: the row sees node j
  int64_t mask_stride;
  int32_t mask_words;
  const float* k_scale;
  const float* v_scale;
  int64_t s_block_stride, s_token_stride, s_head_stride;
  int32_t num_seqs, num_rows, max_q;
  int32_t hq, hkv, group, head_dim, block_size, window;
  float qk_scale_log2;    // log2(e) / sqrt(head_dim)
  int32_t scale_mode;
  void* out;
  int64_t out_row_stride, out_head_stride;
  int64_t* starts;        // [num_seqs + 1]: first macro tile of each sequence; [num_seqs]: share
  float* part;            // [2 * kGrid][rows per block * (head_dim + 2)]
};

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;

// v_mfma_f32_32x32x16: A lane (m = lane % 32, h = lane / 32) holds contraction slots 8 h ..
// 8 h + 7, B the same with n; C / D lane holds column n = lane % 32, rows 8 (i / 4) + 4 h + i % 4
template <int QT>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (QT == RLT_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// two floats -> a packed pair, round to nearest even
template <int QT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (QT == RLT_BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
}
// four e4m3 codes -> four packed 16-bit values (exact)
template <int QT>
__device__ __forceinline__ uint2 widen(uint32_t w) {
  if constexpr (QT == RLT_BF16)
    return make_uint2(
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true)));
  else
    return make_uint2(
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true)));
}

// A word's elements (16-bit halves, or e4m3 codes, which have NaN but no infinities) with the
// non-finite ones cleared.
template <int QT, bool FP8>
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {
  if constexpr (FP8) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (((w >> (8 * i)) & 0x7fu) == 0x7fu) w &= ~(0xffu << (8 * i));
  } else {
    constexpr uint32_t E = QT == RLT_BF16 ? 0x7f80u : 0x7c00u;
    if ((w & E) == E) w &= 0xffff0000u;
    if (((w >> 16) & E) == E) w &= 0xffffu;
  }
  return w;
}

// Direct global -> LDS loads: lane L's 16 (4) bytes land at `lds` + 16 L (4 L).  In assembly,
// without a register result, because the compiler cannot tell these LDS writes from the stages
// that are read meanwhile and would wait for all of them before every LDS read; the caller
// waits with wait_loads<N>().  The s_nop covers a base register written by the vector unit
// just before and M0's own wait state.  No other instruction of the kernel reads M0.
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)(uintptr_t)(lds_void*)p;
}
__device__ __forceinline__ void load_lds16(const void* base, uint32_t lane_bytes, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(lane_bytes), "s"(base), "s"(lds)
               : "memory");
}
__device__ __forceinline__ void load_lds16(const void* lane_address, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(lane_address), "s"(lds)
               : "memory");
}
__device__ __forceinline__ void load_lds4(const void* lane_address, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 4\n\tglobal_load_lds_dword %0, off"
               :
               : "v"(lane_address), "s"(lds)
               : "memory");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// LDS reads done, before a stage is refilled; and the same of every wave
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void stage_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  const uint32_t lo = (uint32_t)uniform((int)(uint32_t)x), hi = (uint32_t)uniform((int)(x >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// A 32-row lane pair's (lane, lane ^ 32) values combined.
__device__ __forceinline__ float half_max(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// ---------------------------------------------------------------- sequences and shares

struct Seq {
  int32_t q_begin, nodes, len, base;  // base: position of node 0
};

__device__ __forceinline__ Seq seq_of(const Params& P, int s) {
  Seq v;
  const int32_t b = P.cu_q[s], e = P.cu_q[s + 1];
  v.q_begin = min(max(b, 0), P.num_rows);
  v.nodes = min(max(min(e, P.num_rows) - v.q_begin, 0), P.max_q);
  const int64_t cap = (int64_t)P.table_width * P.block_size;
  v.len = (int32_t)min((int64_t)max(P.lengths[s], 0), cap);
  v.base = v.len - v.nodes;
  return v;
}
// the same of a wave-uniform sequence, in scalar registers
__device__ __forceinline__ Seq uniform_seq(const Params& P, int s) {
  Seq v = seq_of(P, s);
  v.q_begin = uniform(v.q_begin);
  v.nodes = uniform(v.nodes);
  v.len = uniform(v.len);
  v.base = v.len - v.nodes;
  return v;
}

// Lowest position that any node of the sequence sees (a lower bound).
__device__ __forceinline__ int first_position(const Params& P, const Seq& v) {
  return P.window > 0 ? max(0, v.base - P.window) : 0;
}

// Macro tiles [m0, m0 + count) of one (kv head, row block) pair of the sequence, and its
// row blocks.
struct Span {
  int m0, count, blocks;
};
template <int RB, int MACRO>
__device__ __forceinline__ Span span_of(const Params& P, const Seq& v) {
  Span x;
  x.blocks = (v.nodes * P.group + RB - 1) / RB;
  x.m0 = first_position(P, v) / MACRO;
  x.count = x.blocks ? max(0, (v.len + MACRO - 1) / MACRO - x.m0) : 0;
  return x;
}

// 32 visibility bits of a node at positions tb .. tb + 31: the prefix from `lo` on, then the
// node's mask words (bits past the tree are clear).
__device__ __forceinline__ uint32_t tile_bits(const uint64_t* words, int base, int lo, int tb) {
  const int off = tb - base;
  uint32_t bits;
  if (off <= -kTile) {
    bits = ~0u;
  } else if (off < 0) {
    bits = ((1u << -off) - 1u) | ((uint32_t)words[0] << -off);
  } else if (off >= kMaxNodes) {
    bits = 0;
  } else {
    const int w = off >> 6, b = off & 63;
    uint64_t x = words[w] >> b;
    if (b > 32 && w + 1 < kWords) x |= words[w + 1] << (64 - b);
    bits = (uint32_t)x;
  }
  if (tb < lo) bits = lo - tb >= kTile ? 0u : bits & (~0u << (lo - tb));
  return bits;
}

// The mask words of a node inside the tree, and the lowest prefix position it sees: with a
// sliding window of w, the last w of the positions that it sees, so that a node with more
// than w visible nodes sees no prefix and drops its first ones.
__device__ __forceinline__ int node_mask(const Params& P, const Seq& v, int node, uint64_t* words) {
  const uint64_t* src = P.mask + (int64_t)(v.q_begin + node) * P.mask_stride;
  int seen = 0;
#pragma unroll
  for (int w = 0; w < kWords; ++w) {
    const int left = v.nodes - 64 * w;
    uint64_t x = w < P.mask_words && left > 0 ? src[w] : 0;
    if (left < 64 && left > 0) x &= (1ull << left) - 1;
    // (a tree longer than its cache: nodes before position 0 do not exist)
    const int cut = -v.base - 64 * w;
    if (cut > 0) x &= cut >= 64 ? 0ull : ~0ull << cut;
    words[w] = x;
    seen += __popcll(x);
  }
  if (P.window <= 0) return 0;
  int drop = seen - P.window;
  if (drop <= 0) return max(0, v.base + drop);
#pragma unroll
  for (int w = 0; w < kWords; ++w) {
    while (drop > 0 && words[w]) {
      words[w] &= words[w] - 1;
      --drop;
    }
  }
  return max(0, v.base);
}

// ---------------------------------------------------------------- MFMA kernel

template <int QT, int KVT, int D, int NT, int RW>
struct Geometry {
  static constexpr bool FP8 = KVT != QT;
  static constexpr int ELT = FP8 ? 1 : 2;
  static constexpr int KW = kWaves / RW;
  static constexpr int RB = 32 * NT * RW;            // rows per block
  static constexpr int MACRO = kTile * KW;           // positions per macro tile
  static constexpr int ROW = (D == 96 ? 128 : D) * ELT;  // bytes of an LDS row
  static constexpr int SLOTS = ROW / 16;
  static constexpr int PIECES = D * ELT / 16;        // 16-byte pieces of a row in the pool
  static constexpr int RPL = 64 / SLOTS;             // rows filled by one wave-wide load
  static constexpr int LOADS = kTile / RPL;          // such loads per K (V) tile
  static constexpr int TILE = kTile * ROW;           // bytes of a K (V) tile
  static constexpr int FIT = kRingBytes / (KW * 2 * TILE);
  static constexpr int S = FIT > 6 ? 6 : FIT;        // stages
  static_assert(S >= 2, "at least two stages");
  static_assert(LOADS % RW == 0, "the row waves share a tile's loads");
  static constexpr int RING = KW * S * 2 * TILE;
  static constexpr int OSTRIDE = D + 4;              // floats per row of the combine buffer
  static constexpr int COMBINE = KW * RB * OSTRIDE * 4;
  static constexpr int BODY = RING > COMBINE ? RING : COMBINE;
};

template <int QT, int KVT, int D, int NT, int RW>
struct Shared {
  using G = Geometry<QT, KVT, D, NT, RW>;
  alignas(16) uint8_t body[G::BODY];                 // the ring, then the combine buffer
  alignas(16) float scale[kWaves][G::S][64];         // per wave: 32 key, 32 value scales
  uint64_t words[G::RB][kWords];                     // mask words of the row block's nodes
  int lo[G::RB];
  float ml[G::KW][G::RB][2];
  uint32_t bad[2 * kBadWords];  // positions with a non-finite value in masked tiles
  int64_t totals[kWaves];
  int find_seq;
  int64_t find_start;
};

// LDS slot of a row's 16-byte piece.  Keys: XOR with the row, so that 16 rows of one piece
// column meet distinct bank groups.  Values: XOR so that the rows of one transpose read (4
// rows x a 64-byte dim tile of 16-bit values, 8 rows x 16 bytes of codes) cover the banks.
template <int SLOTS>
__device__ __forceinline__ int k_swz(int r) { return r & (SLOTS - 1); }
template <int SLOTS, bool FP8>
__device__ __forceinline__ int v_swz(int r) {
  if (FP8) return ((r & 3) | ((r >> 1) & 4)) & (SLOTS - 1);
  return SLOTS >= 16 ? 4 * (r & 3) : 4 * ((r >> 1) & 1);
}

template <int QT, int KVT, int D, int SM, int NT, int RW>
__global__ __launch_bounds__(64 * kWaves, 1) void rlt_tree_kernel(Params P) {
  using G = Geometry<QT, KVT, D, NT, RW>;
  constexpr bool FP8 = G::FP8;
  constexpr int ELT = G::ELT, KW = G::KW, RB = G::RB, MACRO = G::MACRO, S = G::S;
  constexpr int SLOTS = G::SLOTS, PIECES = G::PIECES, RPL = G::RPL;
  constexpr int NQ = D / 16;  // contraction slices of S^T
  constexpr int ND = D / 32;  // dim tiles of O^T
  constexpr int LPT = 2 * G::LOADS / RW + (SM == 2 ? 1 : 0);  // a wave's loads per tile
  __shared__ Shared<QT, KVT, D, NT, RW> sh;
  const int t = threadIdx.x, lane = t & 63, l32 = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int kg = w / RW, rw = w % RW;  // kv group, row wave

  // ---- this workgroup's share of the macro tiles
  const int per = (P.num_seqs + 64 * kWaves - 1) / (64 * kWaves);
  const int s_lo = min(t * per, P.num_seqs), s_hi = min(s_lo + per, P.num_seqs);
  int64_t run = 0;
  for (int s = s_lo; s < s_hi; ++s) {
    const Span x = span_of<RB, MACRO>(P, seq_of(P, s));
    run += (int64_t)x.count * x.blocks * P.hkv;
  }
  int64_t incl = run;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(incl, o, RLT_WAVE);
    if (lane >= o) incl += y;
  }
  if (lane == 63) sh.totals[w] = incl;
  __syncthreads();
  int64_t before = incl - run, total = 0;
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) before += sh.totals[i];
    total += sh.totals[i];
  }
  total = uniform(total);
  const int64_t share = (total + kGrid - 1) / kGrid;
  const int64_t f_begin = (int64_t)blockIdx.x * share;
  const int64_t f_end = min(f_begin + share, total);
  if (blockIdx.x == 0) {
    int64_t at = before;
    for (int s = s_lo; s < s_hi; ++s) {
      P.starts[s] = at;
      const Span x = span_of<RB, MACRO>(P, seq_of(P, s));
      at += (int64_t)x.count * x.blocks * P.hkv;
    }
    if (t == 0) P.starts[P.num_seqs] = share;
  }
  if (f_begin >= f_end) return;  // uniform over the workgroup
  if (before <= f_begin && f_begin < before + run) {
    int64_t at = before;
    for (int s = s_lo; s < s_hi; ++s) {
      const Span x = span_of<RB, MACRO>(P, seq_of(P, s));
      const int64_t n = (int64_t)x.count * x.blocks * P.hkv;
      if (f_begin < at + n) {
        sh.find_seq = s;
        sh.find_start = at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  int seq = uniform(sh.find_seq);
  int64_t seq_start = uniform(sh.find_start);
  Seq sv = uniform_seq(P, seq);
  Span sp = span_of<RB, MACRO>(P, sv);

  // ---- lane constants of the loads: lane L of load j fills row RPL j + L / SLOTS, slot L % SLOTS
  const int ld_row = lane / SLOTS, ld_slot = lane % SLOTS;
  const uint32_t k_tok = (uint32_t)P.k_token_stride * ELT, v_tok = (uint32_t)P.v_token_stride * ELT;
  uint8_t* const ring = sh.body + kg * (S * 2 * G::TILE);

  float qk_scale = P.qk_scale_log2, v_mul = 1.f;
  if (SM == 1) {
    qk_scale *= P.k_scale[0];
    v_mul = P.v_scale[0];
  }

  // ---- lane constants of the operand reads
  // S^T: row l32; 16-bit: piece 2 c + h of slice c; codes: piece 2 j + h holds slices 2 j, 2 j + 1
  const int k_x = (h ^ k_swz<SLOTS>(l32)) * 16;
  const int k_lane = l32 * G::ROW;
  // V^T, 16-bit: within a 16-lane group lane i receives element i % 4 of the 8-byte reads of
  // lanes i / 4 + 4 k, so lane i reads row i / 4 at dims 4 (i % 4); codes: lane i receives byte
  // i % 8 of the 8-byte reads of lanes 2 k + i / 8, so lane i reads row i / 2 at dims 8 (i % 2).
  // Rows are the positions in the order of the S^T accumulators: contraction slots 8 h + j of
  // chunk c are positions 16 c + 4 h + j (j < 4) and 16 c + 8 + 4 h + j - 4.
  const int i16 = lane & 15;
  const int vr16 = 4 * h + (i16 >> 2);
  const int vr8 = 4 * h + ((i16 >> 1) & 3) + ((i16 >> 3) << 3);

  int64_t f = f_begin;
  while (f < f_end) {
    // ---- the pair and the part [a, b) of its macro tiles that this share holds
    while (f >= seq_start + (int64_t)sp.count * sp.blocks * P.hkv) {
      seq_start += (int64_t)sp.count * sp.blocks * P.hkv;
      ++seq;
      sv = uniform_seq(P, seq);
      sp = span_of<RB, MACRO>(P, sv);
    }
    const int64_t in_seq = f - seq_start;
    const int pair = (int)(in_seq / sp.count);
    const int a = (int)(in_seq - (int64_t)pair * sp.count);
    const int b = (int)min((int64_t)sp.count, a + (f_end - f));
    const int rb = pair % sp.blocks, kvh = pair / sp.blocks;
    const int rows = min(RB, sv.nodes * P.group - rb * RB);
    const int node0 = rb * RB / P.group;

    // ---- loads of the tile at position tb into a stage
    const auto* table = (const __attribute__((address_space(4))) int32_t*)(
        P.tables + (int64_t)seq * P.table_stride);
    auto issue = [&](int macro, int stage) {
      const int tb = ((sp.m0 + macro) * KW + kg) * kTile;
      // blocks hold whole 8-position groups: four scalar (block, offset) pairs per tile
      int blk[4], off[4];
      int idx = tb / P.block_size, o = tb - idx * P.block_size;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int32_t e = table[min(idx, P.table_width - 1)];
        blk[g] = e >= 0 && e < P.num_blocks ? e : 0;
        off[g] = o;
        o += 8;
        if (o >= P.block_size) {
          o = 0;
          ++idx;
        }
      }
      uint8_t* const st = ring + stage * (2 * G::TILE);
      auto rows_of = [&](const void* pool, int64_t bs, int64_t ts, int64_t hs, uint32_t tok,
                         uint8_t* dst, auto swz) {
        const uint8_t* const head = (const uint8_t*)pool + (int64_t)kvh * hs * ELT;
#pragma unroll
        for (int i = 0; i < G::LOADS / RW; ++i) {
          const int j = i * RW + rw;  // wave-uniform
          const int r0 = RPL * j;
          const int piece = ld_slot ^ swz(r0 + ld_row);
          if (PIECES == SLOTS || piece < PIECES) {
            const uint32_t lds = uniform((int)(lds_offset(dst) + r0 * G::ROW));
            if constexpr (RPL <= 8) {
              const int g = r0 >> 3;
              const int64_t bk = g == 0 ? blk[0] : g == 1 ? blk[1] : g == 2 ? blk[2] : blk[3];
              const int og = g == 0 ? off[0] : g == 1 ? off[1] : g == 2 ? off[2] : off[3];
              const uint8_t* base = head + (bk * bs + (int64_t)(og + (r0 & 7)) * ts) * ELT;
              load_lds16(base, (uint32_t)ld_row * tok + piece * 16, lds);
            } else {
              // 16 rows per load: two groups
              const bool up = ld_row >= 8;
              const int64_t bk = r0 == 0 ? (up ? blk[1] : blk[0]) : (up ? blk[3] : blk[2]);
              const int og = r0 == 0 ? (up ? off[1] : off[0]) : (up ? off[3] : off[2]);
              load_lds16(head + (bk * bs + (int64_t)(og + (ld_row & 7)) * ts) * ELT + piece * 16, lds);
            }
          }
        }
      };
      rows_of(P.k, P.k_block_stride, P.k_token_stride, P.k_head_stride, k_tok, st,
              [](int r) { return k_swz<SLOTS>(r); });
      rows_of(P.v, P.v_block_stride, P.v_token_stride, P.v_head_stride, v_tok, st + G::TILE,
              [](int r) { return v_swz<SLOTS, FP8>(r); });
      if constexpr (SM == 2) {
        const int g = l32 >> 3;
        const int64_t bk = g == 0 ? blk[0] : g == 1 ? blk[1] : g == 2 ? blk[2] : blk[3];
        const int og = g == 0 ? off[0] : g == 1 ? off[1] : g == 2 ? off[2] : off[3];
        load_lds4((h ? P.v_scale : P.k_scale) + bk * P.s_block_stride +
                      (int64_t)(og + (l32 & 7)) * P.s_token_stride + (int64_t)kvh * P.s_head_stride,
                  uniform((int)lds_offset(sh.scale[w][stage])));
      }
    };
    const int n = b - a;
#pragma unroll 1
    for (int i = 0; i < S - 1 && i < n; ++i) issue(a + i, i);

    // ---- this wave's rows: B operands of S^T, and the masks of the block's nodes
    u32x4 qreg[NT][NQ];
    int local[NT];  // node within the block
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = (rw * NT + nt) * 32 + l32;
      const int rho = rb * RB + r;
      const int node = rho / P.group, head = kvh * P.group + rho % P.group;
      local[nt] = r < rows ? node - node0 : 0;
      const uint16_t* qp = (const uint16_t*)P.q + (int64_t)(sv.q_begin + node) * P.q_row_stride +
                           (int64_t)head * P.q_head_stride;
#pragma unroll
      for (int c = 0; c < NQ; ++c) {
        // (codes: slices 2 j and 2 j + 1 take a lane's 16 elements 32 j + 16 h ..)
        const int e = FP8 ? 32 * (c / 2) + 16 * h + 8 * (c % 2) : 16 * c + 8 * h;
        qreg[nt][c] = r < rows ? *(const u32x4*)(qp + e) : u32x4{0, 0, 0, 0};
      }
    }
    const int nodes_here = min(sv.nodes - node0, (rows + rb * RB - node0 * P.group + P.group - 1) / P.group);
    for (int i = t; i < nodes_here; i += 64 * kWaves) sh.lo[i] = node_mask(P, sv, node0 + i, sh.words[i]);
    if (t < 2 * kBadWords) sh.bad[t] = 0;
    // the masked tiles: of the tree, and where a sliding window begins
    const int tree_tile = max(sv.base, 0) / kTile, first_tile = first_position(P, sv) / kTile;
    __syncthreads();

    f32x16 oacc[NT][ND];
    float m_run[NT], m_use[NT], l_run[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m_run[nt] = -INFINITY;
      m_use[nt] = 0.f;
      l_run[nt] = 0.f;
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) oacc[nt][dt][i] = 0.f;
    }

    int stage = 0;
    for (int it = 0; it < n; ++it, stage = stage + 1 == S ? 0 : stage + 1) {
      if (it + S - 1 < n) {
        wait_loads<(S - 2) * LPT>();
        if (RW > 1) stage_barrier();
        issue(a + it + S - 1, stage == 0 ? S - 1 : stage - 1);
      } else {
        wait_loads<0>();
        if (RW > 1) stage_barrier();
      }
      const int tb = ((sp.m0 + a + it) * KW + kg) * kTile;
      if (tb >= sv.len) continue;  // wave-uniform: a macro tile's last tiles
      const uint8_t* const kt = ring + stage * (2 * G::TILE);
      uint8_t* const vt = ring + stage * (2 * G::TILE) + G::TILE;
      // no row hides any of the tile's positions
      const bool full = tb + kTile <= sv.base && (P.window <= 0 || tb >= sv.len - P.window);

      // ---- S^T = K Q^T
      f32x16 sc[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[nt][i] = 0.f;
      if constexpr (!FP8) {
#pragma unroll
        for (int c = 0; c < NQ; ++c) {
          const u32x4 ka = *(const u32x4*)(kt + k_lane + ((32 * c) ^ k_x));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) sc[nt] = mfma<QT>(ka, qreg[nt][c], sc[nt]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NQ / 2; ++j) {
          const u32x4 raw = *(const u32x4*)(kt + k_lane + ((32 * j) ^ k_x));
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const uint2 lo = widen<QT>(raw[2 * x]), hi = widen<QT>(raw[2 * x + 1]);
            const u32x4 ka = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) sc[nt] = mfma<QT>(ka, qreg[nt][2 * j + x], sc[nt]);
          }
        }
      }
      if constexpr (SM == 2) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 x = *(const f32x4*)(sh.scale[w][stage] + 8 * g + 4 * h);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[nt][4 * g + i] *= x[i];
        }
      }
      if (!full) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          // bit 8 g + i: position 8 g + 4 h + i of the tile
          const uint32_t sees = tile_bits(sh.words[local[nt]], sv.base, sh.lo[local[nt]], tb) >> (4 * h);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            sc[nt][i] = (sees >> (8 * (i >> 2) + (i & 3))) & 1 ? sc[nt][i] : -INFINITY;
        }
      }
      // ---- weights in the log2 domain.  The running maximum moves only when a tile's exceeds
      // it by kLazy (weights stay below 2^kLazy), so the accumulators are rarely rescaled.
      uint32_t p[NT][8];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float mx = sc[nt][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sc[nt][i]);
        mx = half_max(mx) * qk_scale;
        const bool grow = mx > m_run[nt] + kLazy;
        if (__builtin_amdgcn_ballot_w64(grow) != 0) {
          const float m_new = grow ? mx : m_run[nt];
          const float use = m_new == -INFINITY ? 0.f : m_new;
          const float corr = grow ? __builtin_amdgcn_exp2f(m_run[nt] - use) : 1.f;
          l_run[nt] *= corr;
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) oacc[nt][dt] *= corr;
          m_run[nt] = m_new;
          m_use[nt] = use;
        }
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[nt][i], qk_scale, -m_use[nt]));
#pragma unroll
        for (int g = 0; g < 4; ++g) l_run[nt] += (x[4 * g] + x[4 * g + 1]) + (x[4 * g + 2] + x[4 * g + 3]);
        if constexpr (SM == 2) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 y = *(const f32x4*)(sh.scale[w][stage] + 32 + 8 * g + 4 * h);
            // (a hidden position's scale may be anything, and its weight is 0)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[4 * g + i] = x[4 * g + i] == 0.f ? 0.f : x[4 * g + i] * y[i];
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) p[nt][i] = pack2<QT>(x[2 * i], x[2 * i + 1]);
      }
      // ---- O^T += V^T P^T.  In masked tiles a value may be hidden from some rows, and 0 times
      // a non-finite value would spoil them: such values are cleared (idempotent: the row waves
      // may both do it) and marked, and rows that see them get them behind the stream.  Rows
      // past the sequence belong to no row.
      if (!full) {
        const int tile = tb / kTile;
        const int word = tile >= tree_tile ? min(tile - tree_tile, kBadWords - 1)
                                           : kBadWords + min(max(tile - first_tile, 0), kBadWords - 1);
#pragma unroll
        for (int j = 0; j < G::LOADS; ++j) {
          const int r = RPL * j + ld_row;
          if (PIECES == SLOTS || (ld_slot ^ v_swz<SLOTS, FP8>(r)) < PIECES) {
            u32x4* const at = (u32x4*)(vt + r * G::ROW + ld_slot * 16);
            if (tb + r >= sv.len) {
              *at = u32x4{0, 0, 0, 0};
            } else {
              const u32x4 x = *at;
              const u32x4 y = {finite_part<QT, FP8>(x[0]), finite_part<QT, FP8>(x[1]),
                               finite_part<QT, FP8>(x[2]), finite_part<QT, FP8>(x[3])};
              if (x[0] != y[0] || x[1] != y[1] || x[2] != y[2] || x[3] != y[3]) {
                atomicOr(&sh.bad[word], 1u << r);
                *at = y;
              }
            }
          }
        }
        asm volatile("" ::: "memory");
      }
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          u32x4 va;
          if constexpr (!FP8) {
            const int piece = 2 * ((lane >> 4) & 1) + ((i16 >> 1) & 1);  // within the dim tile
            const uint8_t* vr = vt + (16 * c + vr16) * G::ROW +
                                ((4 * dt + piece) ^ v_swz<SLOTS, false>(vr16)) * 16 + (i16 & 1) * 8;
            const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(lds_void*)vr);
            const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) s16x4*)(lds_void*)(vr + 8 * G::ROW));
            __builtin_memcpy(&va, &x0, 8);
            __builtin_memcpy((char*)&va + 8, &x1, 8);
          } else {
            const int r = 16 * c + vr8;
            const uint8_t* vr = vt + r * G::ROW +
                                ((2 * dt + ((lane >> 4) & 1)) ^ v_swz<SLOTS, true>(r)) * 16 + (i16 & 1) * 8;
            const i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                (__attribute__((address_space(3))) i32x2*)(lds_void*)vr);
            const uint2 lo = widen<QT>((uint32_t)x[0]), hi = widen<QT>((uint32_t)x[1]);
            va = u32x4{lo.x, lo.y, hi.x, hi.y};
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const u32x4 pc = {p[nt][4 * c], p[nt][4 * c + 1], p[nt][4 * c + 2], p[nt][4 * c + 3]};
            oacc[nt][dt] = mfma<QT>(va, pc, oacc[nt][dt]);
          }
        }
      wait_lds();
    }
    wait_loads<0>();
    __syncthreads();  // every wave is done with the ring: the combine buffer takes its place

    // ---- the kv groups' states side by side in LDS, then combined in order
    float* const ob = (float*)sh.body;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = (rw * NT + nt) * 32 + l32;
      const float l = half_sum(l_run[nt]);
      if (h == 0) {
        sh.ml[kg][r][0] = m_run[nt];
        sh.ml[kg][r][1] = l;
      }
      float* const row = ob + (kg * RB + r) * G::OSTRIDE + 4 * h;
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x16& o = oacc[nt][dt];
          *(f32x4*)(row + 32 * dt + 8 * g) = f32x4{o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]};
        }
    }
    __syncthreads();
    // marked values, for the rows that see them
    uint32_t any_bad = 0;
    for (int i = 0; i < 2 * kBadWords; ++i) any_bad |= sh.bad[i];
    const bool whole = n == sp.count;
    const int slot = 2 * blockIdx.x + (f == f_begin ? 0 : 1);
    float* const part = P.part + (int64_t)slot * RB * (D + 2);
    for (int e = t; e < rows * (D / 4); e += 64 * kWaves) {
      const int r = e / (D / 4), d = 4 * (e % (D / 4));
      float m = -INFINITY;
#pragma unroll
      for (int g = 0; g < KW; ++g) m = fmaxf(m, sh.ml[g][r][0]);
      float l = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < KW; ++g) {
        const float mg = sh.ml[g][r][0];
        const float x = mg == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mg - m);
        // (a group whose sum is NaN spoils the row, as it should)
        const float lg = sh.ml[g][r][1];
        l += mg == -INFINITY && lg == 0.f ? 0.f : lg * x;
        const f32x4 og = *(const f32x4*)(ob + (g * RB + r) * G::OSTRIDE + d);
        if (mg != -INFINITY || lg != 0.f) o += og * x;
      }
      const int rho = rb * RB + r;
      if (any_bad) {
        const int local_node = rho / P.group - node0;
        for (int i = 0; i < 2 * kBadWords; ++i) {
          const int tb = (i < kBadWords ? tree_tile + i : first_tile + i - kBadWords) * kTile;
          uint32_t left = sh.bad[i];
          if (left) left &= tile_bits(sh.words[local_node], sv.base, sh.lo[local_node], tb);
          for (; left; left &= left - 1) {
            const int pos = tb + __builtin_ctz(left);
            const int32_t e = table[min(pos / P.block_size, P.table_width - 1)];
            const int64_t at = (int64_t)(e >= 0 && e < P.num_blocks ? e : 0) * P.v_block_stride +
                               (int64_t)(pos % P.block_size) * P.v_token_stride +
                               (int64_t)kvh * P.v_head_stride + d;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float x = load_as_f32<KVT>(P.v, at + c);
              if (!(fabsf(x) < INFINITY)) o[c] += x;
            }
          }
        }
      }
      if (whole) {
        const float inv = l == 0.f ? 0.f : v_mul / l;
        uint16_t* const op = (uint16_t*)P.out + (int64_t)(sv.q_begin + rho / P.group) * P.out_row_stride +
                             (int64_t)(kvh * P.group + rho % P.group) * P.out_head_stride + d;
        *(uint2*)op = make_uint2(pack2<QT>(o[0] * inv, o[1] * inv), pack2<QT>(o[2] * inv, o[3] * inv));
      } else {
        *(f32x4*)(part + r * D + d) = o;
        if (d == 0) {
          part[RB * D + 2 * r] = m;
          part[RB * D + 2 * r + 1] = l;
        }
      }
    }
    __syncthreads();  // the ring, the masks and the sums are reused by the next pair
    f += n;
  }
}

// The partials of pairs that cross shares, combined in order: one wave per (row, q head).
// Rows of sequences without a key become zeros here.
template <int QT, int RB, int MACRO>
__global__ __launch_bounds__(256) void rlt_tree_merge_kernel(Params P) {
  const int lane = threadIdx.x & 63;
  const int seq = blockIdx.x;
  const int item = blockIdx.y * 4 + (threadIdx.x >> 6);  // (node, q head)
  const Seq sv = seq_of(P, seq);
  const int node = item / P.hq, head = item % P.hq;
  if (node >= sv.nodes) return;
  const int D = P.head_dim;
  const Span sp = span_of<RB, MACRO>(P, sv);
  uint16_t* const op = (uint16_t*)P.out + (int64_t)(sv.q_begin + node) * P.out_row_stride +
                       (int64_t)head * P.out_head_stride;
  if (sp.count == 0) {
    for (int d = lane; d < D; d += 64) op[d] = 0;
    return;
  }
  const int rho = node * P.group + head % P.group;
  const int rb = rho / RB, r = rho % RB;
  const int64_t share = P.starts[P.num_seqs];
  const int64_t f0 = P.starts[seq] + ((int64_t)(head / P.group) * sp.blocks + rb) * sp.count;
  const int b0 = (int)(f0 / share), b1 = (int)((f0 + sp.count - 1) / share);
  if (b0 == b1) return;  // normalized where it was computed
  auto slot_of = [&](int b) { return 2 * b + (b == b0 && f0 != b * share ? 1 : 0); };
  const int64_t stride = (int64_t)RB * (D + 2);
  // the overall maximum: lanes take the contributions
  float m = -INFINITY;
  for (int b = b0 + lane; b <= b1; b += 64)
    m = fmaxf(m, P.part[slot_of(b) * stride + RB * D + 2 * r]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, RLT_WAVE));
  float acc[4] = {0.f, 0.f, 0.f, 0.f};  // dims lane, lane + 64, ..
  float l = 0.f;
#pragma unroll 4
  for (int b = b0; b <= b1; ++b) {
    const float* const part = P.part + slot_of(b) * stride;
    const float mb = part[RB * D + 2 * r], lb = part[RB * D + 2 * r + 1];
    const bool live = mb != -INFINITY || lb != 0.f;
    const float x = mb == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mb - m);
    if (live) l += lb * x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int d = lane + 64 * i;
      if (d < D) {
        const float o = part[r * D + d];
        if (live) acc[i] += o * x;
      }
    }
  }
  const float v_mul = P.scale_mode == 1 ? P.v_scale[0] : 1.f;
  const float inv = l == 0.f ? 0.f : v_mul / l;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int d = lane + 64 * i;
    if (d < D) store_from_f32<QT>(op, d, acc[i] * inv);
  }
}

}  // namespace tree
