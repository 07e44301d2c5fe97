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
// Tiling.  A workgroup is four waves, two workgroups share a CU: two waves per SIMD hide each
// other's chains of LDS reads, matrix instructions and exponentials.  The waves are RW row
// waves times KW = 4 / RW kv waves.  A row wave holds 32 rows (v_mfma_f32_32x32x16: S^T = K
// Q^T, O^T += V^T P^T); each kv wave (group of RW row waves) streams its own 32-position
// tiles, every KW-th of the workgroup's share, through LDS by direct global -> LDS loads.
// With RW = 1 (up to 32 rows) no wave waits for another inside the stream: a tile's keys are
// refilled as soon as its scores are taken, its values as soon as they are added.  More rows
// take 2 or 4 row waves that share the tiles, one barrier per tile.
//
// Measured (main kernel + merge, medians; bytes by counters): 32 sequences of 20 to 32 nodes, GQA 4,
// up to 8192 positions, bf16 76 + 11 us (296 MB read, 33 of partials written: 4.3 TB/s); 16
// sequences of 64 nodes, 55 heads of 96 163 + 18 us (835 MB read for 692 of keys and values, whose
// heads straddle lines, 44 written: 5.4 TB/s); 64 sequences of 16k to 32k positions in fp8
// 645 + 12 us (3.29 GB read: 5.2 TB/s).  One sequence of 700 positions takes 11.5 + 4 us: 2 us
// to find the share, 2 for tables and first loads, 1 for the tiles, 2 to combine; the launches the
// rest.  With the compensated product 86, 166, 646 and 11.6 us.
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

// Where a pair's partials are: slot `first` of the workgroup that holds its first macro tile, then
// the slots 2 b of the workgroups b up to `last`; last < 0: normalized where it was computed.
struct Split {
  int32_t first, last;
  int32_t row;  // of the slots' rows, the pair's first
};

constexpr int kWaves = 4;
constexpr int kPartRows = 32 * kWaves;  // rows of a partial, at most
constexpr int kTile = 32;          // key positions per LDS tile
constexpr int kGrid = 512;         // persistent workgroups, at most: two per CU
// (256 dims: the states of a workgroup take more than half of a CU's LDS and registers)
template <int D>
constexpr int per_cu() { return D == 256 ? 1 : 2; }
template <int D>
constexpr int grid_of() { return kGrid / 2 * per_cu<D>(); }
constexpr int kMaxNodes = 256;     // nodes of one sequence's tree
constexpr int kWords = kMaxNodes / 64;
constexpr int kRingBytes = 64 << 10;
constexpr int kBadWords = kMaxNodes / kTile + 3;  // tiles that a range of kMaxNodes meets
// Tiles per workgroup from which the kv groups take neighbouring heads apart: these share a
// position's cache lines (fp8, 8 heads of 128: 645 us, 710 together; 55 heads of 96: 163 and 197),
// but a pair's tiles then come one by one, which leaves short shares to few waves.
constexpr int kApartTiles = 8;
constexpr float kLazy = 8.f;       // log2 headroom before the running max moves
constexpr float kLowExp = -100.f;  // lowest exponent that weights times value scales are held over

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
  int32_t compensate;     // the product with the values also takes what rounding the weights dropped
  void* out;
  int64_t out_row_stride, out_head_stride;
  int32_t max_blocks;     // row blocks of the longest tree
  struct Split* splits;   // [num_seqs][hkv][max_blocks]
  float* part;            // [2 * kGrid][kPartRows * (head_dim + 2)]
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

// What the rounding of (a, b) to the packed pair `w` dropped, as a pair of the type (INF: nothing
// of a number that is infinite there).
template <int QT, bool INF>
__device__ __forceinline__ uint32_t dropped2(float a, float b, uint32_t w) {
  if constexpr (QT == RLT_BF16) {
    a -= __uint_as_float(w << 16);
    b -= __uint_as_float(w & 0xffff0000u);
  } else {
    a -= f16_bits_to_f32((uint16_t)w);
    b -= f16_bits_to_f32((uint16_t)(w >> 16));
  }
  if constexpr (INF) {
    a = fabsf(a) < INFINITY ? a : 0.f;
    b = fabsf(b) < INFINITY ? b : 0.f;
  }
  return pack2<QT>(a, b);
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

// Macro tiles [m0, m0 + count) of `macro` positions (a power of two of tiles) of one pair of
// the sequence, and its row blocks.
struct Span {
  int m0, count, blocks;
};
template <int RB>
__device__ __forceinline__ Span span_of(const Params& P, const Seq& v, int macro) {
  Span x;
  x.blocks = (v.nodes * P.group + RB - 1) / RB;
  x.m0 = first_position(P, v) / macro;
  x.count = x.blocks ? max(0, (v.len + macro - 1) / macro - x.m0) : 0;
  return x;
}
template <int RB>
__device__ __forceinline__ Span uniform_span(const Params& P, const Seq& v, int macro) {
  Span x = span_of<RB>(P, v, macro);
  x.m0 = uniform(x.m0);
  x.count = uniform(x.count);
  x.blocks = uniform(x.blocks);
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

template <int QT, int KVT, int D, int RW>
struct Geometry {
  static constexpr bool FP8 = KVT != QT;
  static constexpr int ELT = FP8 ? 1 : 2;
  static constexpr int KW = kWaves / RW;
  static constexpr int RB = 32 * RW;                 // rows per block
  static constexpr int ROW = (D == 96 ? 128 : D) * ELT;  // bytes of an LDS row
  static constexpr int SLOTS = ROW / 16;
  static constexpr int PIECES = D * ELT / 16;        // 16-byte pieces of a row in the pool
  static constexpr int RPL = 64 / SLOTS;             // rows filled by one wave-wide load
  static constexpr int LOADS = kTile / RPL;          // such loads per K (V) tile
  static constexpr int TILE = kTile * ROW;           // bytes of a K (V) tile
  static constexpr int FIT = kRingBytes / (KW * 2 * TILE);
  static constexpr int S = FIT > 4 ? 4 : FIT;        // stages
  static_assert(S >= (RW == 1 ? 1 : 2), "row waves that share tiles need a second stage");
  // a row wave's loads of a K (V) tile (of fewer loads than waves some are done twice)
  static constexpr int LV = LOADS >= RW ? LOADS / RW : 1;
  static_assert(LOADS % RW == 0 || RW % LOADS == 0, "the row waves share a tile's loads");
  static constexpr int RING = KW * S * 2 * TILE;
  static constexpr int OSTRIDE = D + 4;              // floats per row of the combine buffer
  static constexpr int COMBINE = KW * RB * OSTRIDE * 4;
  static constexpr int BODY = RING > COMBINE ? RING : COMBINE;
};

template <int QT, int KVT, int D, int RW>
struct Shared {
  using G = Geometry<QT, KVT, D, RW>;
  alignas(16) uint8_t body[G::BODY];                 // the ring, then the combine buffer
  // per kv group and stage, for each row wave: its positions' key scales, then value scales
  alignas(16) float scale[G::KW][G::S + 1][64];
  uint64_t words[G::RB][kWords];                     // mask words of the row block's nodes
  int lo[G::RB];
  float ml[G::KW][G::RB][2];
  uint32_t bad[2 * kBadWords];  // positions with a non-finite value in masked tiles
  int64_t totals[2][kWaves];
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

// CP: what the weights' rounding to q's type dropped is a second operand of the product with the
// values, which keeps ~16 bits of each weight (bf16; fp16 22) instead of 8 (11).
template <int QT, int KVT, int D, int SM, int RW, bool CP>
__global__ __launch_bounds__(64 * kWaves, per_cu<D>()) void rlt_tree_kernel(Params P) {
  using G = Geometry<QT, KVT, D, RW>;
  constexpr bool FP8 = G::FP8;
  constexpr int ELT = G::ELT, KW = G::KW, RB = G::RB, S = G::S;
  constexpr int SLOTS = G::SLOTS, PIECES = G::PIECES, RPL = G::RPL;
  constexpr int NQ = D / 16;  // contraction slices of S^T
  constexpr int ND = D / 32;  // dim tiles of O^T
  constexpr int LV = G::LV, LK = LV + (SM == 2 ? 1 : 0);  // a wave's loads per tile
  constexpr bool REFER = QT == RLT_F16 && SM == 2;
  constexpr float LIFT = QT == RLT_F16 ? 7.f : 0.f;
  __shared__ Shared<QT, KVT, D, RW> sh;
  const int t = threadIdx.x, lane = t & 63, l32 = lane & 31, h = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(t >> 6);
  const int kg = w / RW, rw = w % RW;  // kv group, row wave

  // ---- this workgroup's share of the macro tiles, in both forms: the kv groups on one head's
  // neighbouring tiles, or (`apart`) each on its own one of KW neighbouring heads
  const int per = (P.num_seqs + 64 * kWaves - 1) / (64 * kWaves);
  const int s_lo = min(t * per, P.num_seqs), s_hi = min(s_lo + per, P.num_seqs);
  const int head_groups = (P.hkv + KW - 1) / KW;
  int64_t run = 0, run_apart = 0;
  for (int s = s_lo; s < s_hi; ++s) {
    const Seq v = seq_of(P, s);
    const Span x = span_of<RB>(P, v, kTile * KW), y = span_of<RB>(P, v, kTile);
    run += (int64_t)x.count * x.blocks * P.hkv;
    run_apart += (int64_t)y.count * y.blocks * head_groups;
  }
  int64_t incl = run, incl_apart = run_apart;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(incl, o, RLT_WAVE), z = __shfl_up(incl_apart, o, RLT_WAVE);
    if (lane >= o) {
      incl += y;
      incl_apart += z;
    }
  }
  if (lane == 63) {
    sh.totals[0][w] = incl;
    sh.totals[1][w] = incl_apart;
  }
  __syncthreads();
  int64_t total_apart = 0;
  for (int i = 0; i < kWaves; ++i) total_apart += sh.totals[1][i];
  const bool apart = KW > 1 && P.hkv > 1 && uniform(total_apart) >= (int64_t)kApartTiles * grid_of<D>();
  const int macro = apart ? kTile : kTile * KW;
  const int units = apart ? head_groups : P.hkv;
  int64_t before = apart ? incl_apart - run_apart : incl - run, total = 0;
  if (apart) run = run_apart;
  for (int i = 0; i < kWaves; ++i) {
    const int64_t x = sh.totals[apart ? 1 : 0][i];
    if (i < w) before += x;
    total += x;
  }
  total = uniform(total);
  const int64_t share = (total + grid_of<D>() - 1) / grid_of<D>();
  const int64_t f_begin = (int64_t)blockIdx.x * share;
  const int64_t f_end = min(f_begin + share, total);
  if (f_begin >= f_end) return;  // uniform over the workgroup
  if (before <= f_begin && f_begin < before + run) {
    int64_t at = before;
    for (int s = s_lo; s < s_hi; ++s) {
      const Span x = span_of<RB>(P, seq_of(P, s), macro);
      const int64_t n = (int64_t)x.count * x.blocks * units;
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
  Span sp = uniform_span<RB>(P, sv, macro);

  // ---- lane constants of the loads: a wave's LV loads fill RPL rows each from row ld_first of a
  // tile on, lane L row L / SLOTS and slot L % SLOTS of them (of fewer loads than row waves
  // some are done twice); of the per-vector scales it takes positions SP rw .. SP rw + SP - 1
  constexpr int DUP = G::LOADS >= RW ? 1 : RW / G::LOADS;
  constexpr int NG = LV * RPL / 8;
  constexpr int SP = kTile / RW;
  const int ld_row = lane / SLOTS, ld_slot = lane % SLOTS;
  const int ld_first = rw / DUP * (LV * RPL);
  const int sc_first = SP * rw - ld_first;
  const uint32_t k_tok = (uint32_t)P.k_token_stride * ELT, v_tok = (uint32_t)P.v_token_stride * ELT;
  uint8_t* const ring = sh.body + kg * (S * 2 * G::TILE);  // the group's S key tiles, then S value tiles
  // (block, offset) of a tile's first position: advanced without a division
  const int step_q = uniform(macro / P.block_size), step_r = macro - step_q * P.block_size;

  // (the scale is not folded into qk_scale, which maxima and masked scores are multiplied by: it
  // may be 0 or negative)
  const float qk_scale = P.qk_scale_log2;
  float k_mul = 1.f, v_mul = 1.f;
  if (SM == 1) {
    k_mul = P.k_scale[0];
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
    while (f >= seq_start + (int64_t)sp.count * sp.blocks * units) {
      seq_start += (int64_t)sp.count * sp.blocks * units;
      ++seq;
      sv = uniform_seq(P, seq);
      sp = uniform_span<RB>(P, sv, macro);
    }
    const uint32_t in_seq = (uint32_t)(f - seq_start);
    const int pair = uniform((int)(in_seq / (uint32_t)sp.count));
    const int a = (int)(in_seq - (uint32_t)pair * sp.count);
    const int n = (int)min((int64_t)(sp.count - a), f_end - f);
    const int unit = uniform(pair / sp.blocks), rb = pair - unit * sp.blocks;
    const int head0 = apart ? unit * KW : unit, heads = apart ? min(KW, P.hkv - head0) : 1;
    const bool alive = !apart || kg < heads;  // (the last heads may be fewer than the kv groups)
    const int kvh = alive ? head0 + (apart ? kg : 0) : head0;
    const int rows = min(RB, sv.nodes * P.group - rb * RB);
    const int node0 = rb * RB / P.group;

    // ---- loads of the next tile of the group
    // (constant address space and scalar addresses: scalar loads, which the vector loads'
    // counter does not see -- a wait for a vector load would wait for all tiles in flight)
    const auto* table = (const __attribute__((address_space(4))) int32_t*)uniform(
        (int64_t)(P.tables + (int64_t)seq * P.table_stride));
    const uint8_t* const k_head = (const uint8_t*)P.k + (int64_t)kvh * P.k_head_stride * ELT;
    const uint8_t* const v_head = (const uint8_t*)P.v + (int64_t)kvh * P.v_head_stride * ELT;
    const int first_tb = (sp.m0 + a) * macro + (apart ? 0 : kg * kTile);
    // this wave's rows of a tile are whole 8-position groups, and so are the pool's blocks: a
    // scalar (block, offset) per group
    const int cur = first_tb + ld_first;
    int next_idx = uniform(cur / P.block_size), next_off = cur - next_idx * P.block_size;
    int blk[NG], off[NG];
    auto next_tile = [&]() {
      int idx = next_idx, o = next_off;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int32_t e = table[uniform(min(idx, P.table_width - 1))];
        blk[g] = e >= 0 && e < P.num_blocks ? e : 0;
        off[g] = o;
        o += 8;
        if (o >= P.block_size) {
          o = 0;
          ++idx;
        }
      }
      next_idx += step_q;
      next_off += step_r;
      if (next_off >= P.block_size) {
        next_off -= P.block_size;
        ++next_idx;
      }
    };
    auto load_rows = [&](const uint8_t* head, int64_t bs, uint32_t tok, uint8_t* dst, auto swz) {
      const uint8_t* base[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g)
        base[g] = head + uniform((int64_t)blk[g] * (bs * ELT) + (int64_t)((uint64_t)((uint32_t)off[g]) * tok));
      const uint32_t to = lds_offset(dst) + ld_first * G::ROW;
#pragma unroll
      for (int i = 0; i < LV; ++i) {
        const int piece = ld_slot ^ swz(ld_first + RPL * i + ld_row);
        if (PIECES == SLOTS || piece < PIECES) {
          const uint32_t lds = uniform((int)(to + RPL * i * G::ROW));
          if constexpr (RPL <= 8) {
            load_lds16(base[RPL * i >> 3], (uint32_t)((RPL * i & 7) + ld_row) * tok + piece * 16, lds);
          } else {
            // 16 rows per load: two groups
            const uint8_t* const at = ld_row >= 8 ? base[2 * i + 1] : base[2 * i];
            load_lds16(at + (uint32_t)(ld_row & 7) * tok + piece * 16, lds);
          }
        }
      }
    };
    auto load_k = [&](int stage, int scale_stage) {
      load_rows(k_head, P.k_block_stride, k_tok, ring + stage * G::TILE,
                [](int r) { return k_swz<SLOTS>(r); });
      if constexpr (SM == 2) {
        // the wave's share of the tile's scales: SP key scales, then SP value scales
        if (lane < 2 * SP) {
          const int at = sc_first + (lane & (SP - 1)), g = at >> 3;
          int64_t bk = blk[0];
          int og = off[0];
#pragma unroll
          for (int x = 1; x < NG; ++x) {
            bk = g == x ? blk[x] : bk;
            og = g == x ? off[x] : og;
          }
          load_lds4((lane >= SP ? P.v_scale : P.k_scale) + bk * P.s_block_stride +
                        (int64_t)(og + (at & 7)) * P.s_token_stride + (int64_t)kvh * P.s_head_stride,
                    uniform((int)lds_offset(&sh.scale[kg][scale_stage][2 * SP * rw])));
        }
      }
    };
    auto load_v = [&](int stage) {
      load_rows(v_head, P.v_block_stride, v_tok, ring + (S + stage) * G::TILE,
                [](int r) { return v_swz<SLOTS, FP8>(r); });
    };

    // this wave's tiles: a row wave's barriers are the workgroup's, so those of KW groups alike
    const int tiles = RW > 1 ? n : alive ? max(0, min(n, (sv.len - first_tb + macro - 1) / macro)) : 0;
    if constexpr (RW == 1) {
#pragma unroll
      for (int i = 0; i < S; ++i)
        if (i < tiles) {
          next_tile();
          load_k(i, i);
          load_v(i);
        }
    } else {
#pragma unroll 1
      for (int i = 0; i < S - 1 && i < tiles && alive; ++i) {
        next_tile();
        load_k(i, i);
        load_v(i);
      }
    }

    // ---- this wave's rows: B operands of S^T, and the masks of the block's nodes
    u32x4 qreg[NQ];
    int local;  // node within the block
    {
      const int r = rw * 32 + l32;
      const int rho = rb * RB + r;
      const int node = rho / P.group, head = kvh * P.group + rho % P.group;
      local = r < rows ? node - node0 : 0;
      const uint16_t* qp = (const uint16_t*)P.q + (int64_t)(sv.q_begin + node) * P.q_row_stride +
                           (int64_t)head * P.q_head_stride;
#pragma unroll
      for (int c = 0; c < NQ; ++c) {
        // (codes: slices 2 j and 2 j + 1 take a lane's 16 elements 32 j + 16 h ..)
        const int e = FP8 ? 32 * (c / 2) + 16 * h + 8 * (c % 2) : 16 * c + 8 * h;
        qreg[c] = r < rows ? *(const u32x4*)(qp + e) : u32x4{0, 0, 0, 0};
      }
      // (arrived here: a wait at their use would wait for every tile in flight, in every step)
#pragma unroll
      for (int c = 0; c < NQ; ++c) asm volatile("" : "+v"(qreg[c]));
    }
    const int nodes_here = min(sv.nodes - node0, (rows + rb * RB - node0 * P.group + P.group - 1) / P.group);
    if (t < nodes_here) sh.lo[t] = node_mask(P, sv, node0 + t, sh.words[t]);
    if (t < 2 * kBadWords) sh.bad[t] = 0;
    // the masked tiles: of the tree, and where a sliding window begins
    const int tree_tile = max(sv.base, 0) / kTile, first_tile = first_position(P, sv) / kTile;
    __syncthreads();

    f32x16 oacc[ND];
    float m_run = -INFINITY, m_use = 0.f, l_run = 0.f;
    float v_exp = kLowExp;  // REFER: oacc is the sum over 2^v_exp
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) oacc[dt][i] = 0.f;

    // no row hides any of the positions of the tile at tb
    auto is_full = [&](int tb) {
      return tb + kTile <= sv.base && (P.window <= 0 || tb >= sv.len - P.window);
    };
    // ---- S^T = K Q^T of the tile in stage `kt`; all operand reads in flight together
    auto scores = [&](f32x16& sc, const uint8_t* kt) {
      constexpr int NR = FP8 ? NQ / 2 : NQ;
      u32x4 raw[NR];
#pragma unroll
      for (int c = 0; c < NR; ++c) raw[c] = *(const u32x4*)(kt + k_lane + ((32 * c) ^ k_x));
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = 0.f;
      if constexpr (!FP8) {
#pragma unroll
        for (int c = 0; c < NQ; ++c) sc = mfma<QT>(raw[c], qreg[c], sc);
      } else {
#pragma unroll
        for (int c = 0; c < NQ; ++c) {
          const uint2 lo = widen<QT>(raw[c / 2][2 * (c % 2)]), hi = widen<QT>(raw[c / 2][2 * (c % 2) + 1]);
          sc = mfma<QT>(u32x4{lo.x, lo.y, hi.x, hi.y}, qreg[c], sc);
        }
      }
    };
    // ---- weights in the log2 domain, packed as the P^T operands.  The running maximum moves
    // only when a tile's exceeds it by kLazy (weights stay below 2^kLazy), so the accumulators
    // are rarely rescaled.  The product takes them in q's 16-bit type, as precise as the output.
    // fp16 has few exponents: there weights lie 2^LIFT above their place, below its largest
    // number, and weights times value scales, which may be of any size, are held over a power
    // of two that follows the row's largest such product (REFER).
    auto scale_at = [](int pos) { return pos / SP * (2 * SP) + pos % SP; };
    constexpr int NP = CP ? 16 : 8;  // packed weights, then what their rounding dropped
    auto weigh = [&](f32x16& sc, uint32_t (&p)[NP], int tb, bool full, const float* scale) {
      if constexpr (SM == 1) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] *= k_mul;
      }
      if constexpr (SM == 2) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 x = *(const f32x4*)(scale + scale_at(8 * g + 4 * h));
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[4 * g + i] *= x[i];
        }
      }
      if (!full) {
        // bit 8 g + i: position 8 g + 4 h + i of the tile
        const uint32_t sees = tile_bits(sh.words[local], sv.base, sh.lo[local], tb) >> (4 * h);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          sc[i] = (sees >> (8 * (i >> 2) + (i & 3))) & 1 ? sc[i] : -INFINITY;
      }
      float mx = sc[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, sc[i]);
      mx = half_max(mx) * qk_scale;
      const bool grow = mx > m_run + kLazy;
      if (__builtin_amdgcn_ballot_w64(grow) != 0) {
        const float m_new = grow ? mx : m_run;
        const float step = grow ? m_new - m_run : 0.f;
        l_run *= __builtin_amdgcn_exp2f(-step);
        float o_step = step;
        if constexpr (REFER) {
          const float down = fminf(floorf(step), v_exp - kLowExp);
          o_step -= down;
          v_exp -= down;
        }
        const float corr = __builtin_amdgcn_exp2f(-o_step);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) oacc[dt] *= corr;
        m_run = m_new;
        m_use = m_new == -INFINITY ? 0.f : m_new - LIFT;
      }
      float x[16];
#pragma unroll
      for (int i = 0; i < 16; ++i)
        x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], qk_scale, -m_use));
      float part[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) part[g] = (x[4 * g] + x[4 * g + 1]) + (x[4 * g + 2] + x[4 * g + 3]);
      l_run += (part[0] + part[1]) + (part[2] + part[3]);
      if constexpr (SM == 2) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 y = *(const f32x4*)(scale + scale_at(8 * g + 4 * h) + SP);
          // (a hidden position's scale may be anything, and its weight is 0)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[4 * g + i] = x[4 * g + i] == 0.f ? 0.f : x[4 * g + i] * y[i];
        }
      }
      if constexpr (REFER) {
        float top = fabsf(x[0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, fabsf(x[i]));
        top = half_max(top);
        const bool up = top > __builtin_amdgcn_ldexpf(32768.f, (int)v_exp);
        if (__builtin_amdgcn_ballot_w64(up) != 0) {
          // (the largest product becomes 2^7 .. 2^8; not finite: it stays so)
          const float e = up ? (float)(__builtin_amdgcn_frexp_expf(top) - 8) : v_exp;
          const float corr = __builtin_amdgcn_exp2f(v_exp - e);
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) oacc[dt] *= corr;
          v_exp = e;
        }
        const float down = __builtin_amdgcn_exp2f(-v_exp);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= down;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = pack2<QT>(x[2 * i], x[2 * i + 1]);
      if constexpr (CP) {
        // (weights times value scales may be infinite)
#pragma unroll
        for (int i = 0; i < 8; ++i) p[8 + i] = dropped2<QT, SM == 2>(x[2 * i], x[2 * i + 1], p[i]);
      }
    };
    // In masked tiles a value may be hidden from some rows, and 0 times a non-finite value would
    // spoil them: such values are cleared (idempotent: the row waves may all do it) and marked,
    // and rows that see them get them behind the stream.  Rows past the sequence belong to no row.
    auto clean = [&](uint8_t* vt, int tb) {
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
    };
    // ---- O^T += V^T P^T of the tile in stage `vt`: operand c ND + dt is dim tile dt of chunk c
    constexpr int VW = FP8 ? 2 : 4;  // words of an operand as read
    auto read_v = [&](uint32_t (&va)[2 * ND][VW], const uint8_t* vt) {
#pragma unroll
      for (int n = 0; n < 2 * ND; ++n) {
        const int c = n / ND, dt = n % ND;
        if constexpr (!FP8) {
          const int piece = 2 * ((lane >> 4) & 1) + ((i16 >> 1) & 1);  // within the dim tile
          const uint8_t* vr = vt + (16 * c + vr16) * G::ROW +
                              ((4 * dt + piece) ^ v_swz<SLOTS, false>(vr16)) * 16 + (i16 & 1) * 8;
          const s16x4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(lds_void*)vr);
          const s16x4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(lds_void*)(vr + 8 * G::ROW));
          __builtin_memcpy(&va[n][0], &x0, 8);
          __builtin_memcpy(&va[n][2], &x1, 8);
        } else {
          const int r = 16 * c + vr8;
          const uint8_t* vr = vt + r * G::ROW +
                              ((2 * dt + ((lane >> 4) & 1)) ^ v_swz<SLOTS, true>(r)) * 16 + (i16 & 1) * 8;
          const i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
              (__attribute__((address_space(3))) i32x2*)(lds_void*)vr);
          va[n][0] = (uint32_t)x[0];
          va[n][1] = (uint32_t)x[1];
        }
      }
    };
    auto product = [&](const uint32_t (&va)[2 * ND][VW], const uint32_t (&p)[NP]) {
#pragma unroll
      for (int n = 0; n < 2 * ND; ++n) {
        const int c = n / ND, dt = n % ND;
        u32x4 a4;
        if constexpr (!FP8) {
          a4 = u32x4{va[n][0], va[n][1], va[n][2], va[n][3]};
        } else {
          const uint2 lo = widen<QT>(va[n][0]), hi = widen<QT>(va[n][1]);
          a4 = u32x4{lo.x, lo.y, hi.x, hi.y};
        }
        oacc[dt] = mfma<QT>(a4, u32x4{p[4 * c], p[4 * c + 1], p[4 * c + 2], p[4 * c + 3]}, oacc[dt]);
        if constexpr (CP)
          oacc[dt] = mfma<QT>(a4, u32x4{p[8 + 4 * c], p[9 + 4 * c], p[10 + 4 * c], p[11 + 4 * c]}, oacc[dt]);
      }
    };

    int tb = first_tb;
    if constexpr (RW == 1) {
      int stage = 0, sstage = 0;
      for (int it = 0; it < tiles; ++it) {
        uint8_t* const kt = ring + stage * G::TILE;
        uint8_t* const vt = ring + (S + stage) * G::TILE;
        const float* const scale = sh.scale[kg][sstage];
        const bool more = it + S < tiles;
        const bool full = is_full(tb);
        // (ahead of this tile's keys: its values and the next S - 1 tiles)
        if (more) wait_loads<LV + (S - 1) * (LK + LV)>();
        else wait_loads<0>();
        f32x16 sc;
        scores(sc, kt);
        wait_lds();
        if (more) {
          next_tile();
          load_k(stage, sstage == 0 ? S : sstage - 1);
        }
        // with a second stage the values are here by now: their reads run beside the weights
        uint32_t p[NP], va[2 * ND][VW];
        if (S == 1) weigh(sc, p, tb, full, scale);
        if (more) wait_loads<S * LK + (S - 1) * LV>();
        if (!full) clean(vt, tb);
        read_v(va, vt);
        __builtin_amdgcn_sched_barrier(0);
        if (S > 1) weigh(sc, p, tb, full, scale);
        wait_lds();
        if (more) load_v(stage);
        product(va, p);
        tb += macro;
        stage = stage + 1 == S ? 0 : stage + 1;
        sstage = sstage == S ? 0 : sstage + 1;
      }
    } else {
      int stage = 0;
      for (int it = 0; it < tiles; ++it) {
        if (it + S - 1 < tiles) {
          wait_loads<(S - 2) * (LK + LV)>();
          stage_barrier();
          const int to = stage == 0 ? S - 1 : stage - 1;
          if (alive) {
            next_tile();
            load_k(to, to);
            load_v(to);
          }
        } else {
          wait_loads<0>();
          stage_barrier();
        }
        if (tb < sv.len && alive) {  // wave-uniform: not the last tiles of a macro tile
          uint8_t* const vt = ring + (S + stage) * G::TILE;
          const bool full = is_full(tb);
          f32x16 sc;
          scores(sc, ring + stage * G::TILE);
          uint32_t p[NP], va[2 * ND][VW];
          if (!full) clean(vt, tb);
          read_v(va, vt);
          __builtin_amdgcn_sched_barrier(0);
          weigh(sc, p, tb, full, sh.scale[kg][stage]);
          product(va, p);
        }
        tb += macro;
        stage = stage + 1 == S ? 0 : stage + 1;
      }
    }
    wait_loads<0>();
    __syncthreads();  // every wave is done with the ring: the combine buffer takes its place

    // ---- the kv groups' states side by side in LDS, then combined in order
    float* const ob = (float*)sh.body;
    {
      const int r = rw * 32 + l32;
      const float l = half_sum(l_run);
      if (h == 0) {
        sh.ml[kg][r][0] = m_run;
        sh.ml[kg][r][1] = l;
      }
      float* const row = ob + (kg * RB + r) * G::OSTRIDE + 4 * h;
      if constexpr (REFER) {
        const float back = __builtin_amdgcn_exp2f(v_exp);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) oacc[dt] *= back;
      }
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x16& o = oacc[dt];
          *(f32x4*)(row + 32 * dt + 8 * g) = f32x4{o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]};
        }
    }
    __syncthreads();
    // marked values, for the rows that see them
    uint32_t any_bad = 0;
    for (int i = 0; i < 2 * kBadWords; ++i) any_bad |= sh.bad[i];
    const bool whole = n == sp.count;
    const int slot = 2 * blockIdx.x + (f == f_begin ? 0 : 1);
    if (a == 0 && t < heads)
      P.splits[((int64_t)seq * P.hkv + head0 + t) * P.max_blocks + rb] =
          Split{slot, whole ? -1 : (int)((f + sp.count - 1) / share), t * RB};
    float* const part = P.part + (int64_t)slot * kPartRows * (D + 2);
    for (int e = t; e < heads * rows * (D / 4); e += 64 * kWaves) {
      const int hr = e / (D / 4), d = 4 * (e % (D / 4));
      const int hx = hr / rows, r = hr - hx * rows;  // head of the unit, row of the block
      float m = -INFINITY, l = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      if (apart) {
        m = sh.ml[hx][r][0];
        l = sh.ml[hx][r][1];
        o = *(const f32x4*)(ob + (hx * RB + r) * G::OSTRIDE + d);
      } else {
#pragma unroll
        for (int g = 0; g < KW; ++g) m = fmaxf(m, sh.ml[g][r][0]);
#pragma unroll
        for (int g = 0; g < KW; ++g) {
          const float mg = sh.ml[g][r][0], lg = sh.ml[g][r][1];
          // (a group that saw no key adds nothing; one whose sum is NaN spoils the row)
          const float x = mg == -INFINITY ? (lg == 0.f ? 0.f : lg) : __builtin_amdgcn_exp2f(mg - m);
          const f32x4 og = *(const f32x4*)(ob + (g * RB + r) * G::OSTRIDE + d);
          l += lg * x;
          o += og * x;
        }
      }
      const int rho = rb * RB + r;
      if (any_bad) {
        const int local_node = rho / P.group - node0;
        for (int i = 0; i < 2 * kBadWords; ++i) {
          const int at_tile = (i < kBadWords ? tree_tile + i : first_tile + i - kBadWords) * kTile;
          uint32_t left = sh.bad[i];
          if (left) left &= tile_bits(sh.words[local_node], sv.base, sh.lo[local_node], at_tile);
          for (; left; left &= left - 1) {
            const int pos = at_tile + __builtin_ctz(left);
            const int32_t e2 = table[min(pos / P.block_size, P.table_width - 1)];
            const int64_t at = (int64_t)(e2 >= 0 && e2 < P.num_blocks ? e2 : 0) * P.v_block_stride +
                               (int64_t)(pos % P.block_size) * P.v_token_stride +
                               (int64_t)(head0 + hx) * P.v_head_stride + d;
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
                             (int64_t)((head0 + hx) * P.group + rho % P.group) * P.out_head_stride + d;
        *(uint2*)op = make_uint2(pack2<QT>(o[0] * inv, o[1] * inv), pack2<QT>(o[2] * inv, o[3] * inv));
      } else {
        *(f32x4*)(part + (hx * RB + r) * D + d) = o;
        if (d == 0) *(float2*)(part + kPartRows * D + 2 * (hx * RB + r)) = make_float2(m, l);
      }
    }
    __syncthreads();  // the ring, the masks and the sums are reused by the next pair
    f += n;
  }
}

// The partials of a pair that crosses shares, combined in order: workgroup (pair, y) takes the
// rows y R .. of it, R rows at a time over lanes of 4 dims, with CG groups of threads that
// take a run of the contributions each.  Rows of sequences without a key are cleared here.
constexpr int kMergeThreads = 1024;
template <int D, int CG>
constexpr int merge_rows() { return kMergeThreads / CG / (D == 64 ? 16 : D == 256 ? 64 : 32); }
template <int QT, int D, int RB, int CG>
__global__ __launch_bounds__(kMergeThreads) void rlt_tree_merge_kernel(Params P) {
  constexpr int R = merge_rows<D, CG>(), LPR = kMergeThreads / CG / R;
  __shared__ float sh[CG > 1 ? CG - 1 : 1][kMergeThreads / CG][6];
  const int t = threadIdx.x, cg = t / (kMergeThreads / CG), u = t % (kMergeThreads / CG);
  const int r = blockIdx.y * R + u / LPR, d = 4 * (u % LPR);
  const int rb = blockIdx.x % P.max_blocks, sh_id = blockIdx.x / P.max_blocks;
  const int kvh = sh_id % P.hkv, seq = sh_id / P.hkv;
  const Split x = P.splits[blockIdx.x];
  const Seq sv = seq_of(P, seq);
  const Span sp = span_of<RB>(P, sv, kTile);
  const int rows = min(RB, sv.nodes * P.group - rb * RB);
  if (rows <= 0 || (sp.count > 0 && x.last < 0)) return;  // uniform over the workgroup
  const bool live = r < rows && d < D;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  const int rho = rb * RB + r;
  uint16_t* const op = (uint16_t*)P.out + (int64_t)(sv.q_begin + rho / P.group) * P.out_row_stride +
                       (int64_t)(kvh * P.group + rho % P.group) * P.out_head_stride + d;
  if (sp.count == 0) {
    if (live && cg == 0) *(uint2*)op = make_uint2(0, 0);
    return;
  }
  // state (m, l, o) joined with another one; a state without a key has m = -inf, l = 0
  auto join = [&](float m2, float l2, const f32x4& o2) {
    const float mo = fmaxf(m, m2);
    const float a = m == -INFINITY ? (l == 0.f ? 0.f : l) : __builtin_amdgcn_exp2f(m - mo);
    const float b = m2 == -INFINITY ? (l2 == 0.f ? 0.f : l2) : __builtin_amdgcn_exp2f(m2 - mo);
    l = l * a + l2 * b;
    o = o * a + o2 * b;
    m = mo;
  };
  constexpr int64_t stride = (int64_t)kPartRows * (D + 2);
  const int b0 = x.first >> 1, count = x.last - b0 + 1, per = (count + CG - 1) / CG;
  const int i0 = cg * per, i1 = min(i0 + per, count);
  if (live) {
    constexpr int AHEAD = 4;
    for (int i = i0; i < i1; i += AHEAD) {
      float2 ml[AHEAD];
      f32x4 oo[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) {
        const int at = min(i + k, i1 - 1);
        const float* const part =
            P.part + (at == 0 ? (int64_t)x.first : 2 * (int64_t)(b0 + at)) * stride;
        ml[k] = *(const float2*)(part + kPartRows * D + 2 * (x.row + r));
        oo[k] = *(const f32x4*)(part + (x.row + r) * D + d);
      }
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (i + k < i1) join(ml[k].x, ml[k].y, oo[k]);
    }
  }
  if constexpr (CG > 1) {
    if (cg > 0) {
      float* const s = sh[cg - 1][u];
      s[0] = m;
      s[1] = l;
#pragma unroll
      for (int c = 0; c < 4; ++c) s[2 + c] = o[c];
    }
    __syncthreads();
    if (cg > 0) return;
#pragma unroll
    for (int g = 0; g < CG - 1; ++g) {
      const float* const s = sh[g][u];
      join(s[0], s[1], f32x4{s[2], s[3], s[4], s[5]});
    }
  }
  if (!live) return;
  const float v_mul = P.scale_mode == 1 ? P.v_scale[0] : 1.f;
  const float inv = l == 0.f ? 0.f : v_mul / l;
  *(uint2*)op = make_uint2(pack2<QT>(o[0] * inv, o[1] * inv), pack2<QT>(o[2] * inv, o[3] * inv));
}

}  // namespace tree
