// Rotary positions on MI355X (gfx950): queries and keys turned by their positions, on their own
// (rlt_rotary) or on the way into the paged KV cache (rlt_kv_append); and the cache read back
// as numbers (rlt_kv_load).
//
// Pair p of a head's first `rotary_dim` dims, (a, b) = (x[2p], x[2p + 1]) in the interleaved
// layout or (x[p], x[p + rotary_dim / 2]) in the other, becomes
//   (a c - b s, a s + b c),  (c, s) = amplitude (cos, sin)(2 pi position turns[p]),
// and the inverse takes -s, which is the transpose and so the gradient.  position * turns[p]
// and its reduction to an eighth of a turn are float64 (at position 2^20 a float32 angle is off
// by 0.06), the sine and cosine of the rest float32 series; products and sums float32, rounded
// once to the rows' type.
//
// 8-bit pools take x over its scale: per tensor, per vector (amax / 448, as rlt_kv_store_fp8), or one
// scale per block of tokens and kv head, amax / M of the call's rows in the block (M = 448 for
// e4m3, 127 for int8).  A block that the sequence's earlier tokens had begun keeps the larger of
// its scale and that, and where it grew its earlier codes are held over the new one: the values
// they stand for are quantized again, each time off by half a step of that scale at most.  (N(0, 1)
// tokens one by one into blocks of 16: 2.4 growths in the mean, rms error 1.25 times that of quantizing
// the block once in int8, where values are off by up to 2.9 steps, and 1.34 times in e4m3.)
//
// Work: a workgroup takes 8 rows of a sequence (with block scales: one block of it, 16 rows at
// a time), makes their sines and cosines once in LDS, and its four waves take the heads of q, k
// and v in turn.  A lane holds both halves of its pairs (2 x 16 bytes), a group of LP lanes one
// head vector, so that maxima are lane exchanges and a block's rows stay in registers between
// its maximum and its codes.  What bounds it: each row is read and written once, at the rate of
// a large copy (16384 rows of 20 heads of 128 in bf16, 168 MB: 34.8 us, 4.8 TB/s; 8 prompts of
// 2048 into an int8 cache 45 us), and at a few rows the chain lengths -> table -> rows -> scale
// -> codes of one launch (1 row: 3.4 us in a replayed graph, 6.3 into block scales).

#include "common.h"
#include "fp8_codec.h"
#include "rlt_mi355x.h"

#include <math.h>

#include <type_traits>

namespace {

constexpr int kThreads = 256;
constexpr int kWavesPerGroup = kThreads / 64;
constexpr int kMaxPairs = 128;   // head_dim <= 256
constexpr int kMaxKvItems = 512; // k and v heads, whose maxima over long blocks are kept in LDS
// Workgroups of one launch: a grid holds fewer than 2^32 threads, and a call may ask for more (its
// windows are padded to the longest); those behind go into further launches.
constexpr int64_t kGridGroups = (int64_t)1 << 23;

// What the rows are written to.
enum Mode {
  kApply = 0,       // q_out and k_out
  kSame = 1,        // a pool of the rows' type
  kTensorFp8 = 2,   // e4m3, one scale for the pool (read)
  kVectorFp8 = 3,   // e4m3, a scale per token and head (written)
  kBlockFp8 = 4,    // e4m3, a scale per block and head (written)
  kBlockInt8 = 5,   // int8, a scale per block and head (written)
};
constexpr bool in_blocks(int mode) { return mode == kBlockFp8 || mode == kBlockInt8; }
// Rows that a workgroup works on at a time, whose sines are in LDS: fewer are more workgroups of
// fewer registers (16384 rows of 20 heads 40.8 us by 16, 34.7 by 8); a block of 16 is held whole.
constexpr int rows_of(int mode) { return in_blocks(mode) ? 16 : 8; }

struct Side {
  const void* src;
  int64_t src_row, src_head;
  void* dst;  // rows (kApply, and q), or the pool
  int64_t dst_block, dst_row, dst_head;
  float* scale;
};

struct Params {
  Side q, k, v;
  int32_t hq, hkv, head_dim;
  int64_t rows;
  const int64_t* positions;  // of every row (nullptr: its place in the sequence)
  const double* turns;       // turns per position of every pair
  float amplitude;
  int32_t rotary_dim, interleaved;
  float sign;                // of the sine: -1 turns back
  int64_t s_block, s_token, s_head;
  const int32_t* tables;
  int64_t table_stride;
  int32_t table_width, num_blocks, block_size;
  const int32_t* lengths;
  const int32_t* cu;
  int32_t num_seqs, max_rows, tiles;
  uint32_t first_group;  // of the launch
};

// ---------------------------------------------------------------- sines

// (cos, sin) of 2 pi t, |error| < 2^-23: t less its nearest eighth-turn multiple of 1/4 in float64,
// then the Taylor series on [-pi/4, pi/4] (the terms left out are below 2e-9).
__device__ __forceinline__ float2 turn(double t) {
  const double quarter = rint(4.0 * t);
  const float x = (float)((t - 0.25 * quarter) * 6.283185307179586);
  const int n = (int)(quarter - 4.0 * rint(0.25 * quarter)) & 3;
  const float y = x * x;
  float s = fmaf(y, 2.7557319e-6f, -1.9841270e-4f);
  s = fmaf(y, s, 8.3333333e-3f);
  s = fmaf(y, s, -1.6666667e-1f);
  s = fmaf(x * y, s, x);
  float c = fmaf(y, -2.7557319e-7f, 2.4801587e-5f);
  c = fmaf(y, c, -1.3888889e-3f);
  c = fmaf(y, c, 4.1666667e-2f);
  c = fmaf(y, c, -0.5f);
  c = fmaf(y, c, 1.f);
  const float a = n & 1 ? s : c, b = n & 1 ? c : s;
  return make_float2((n == 1 || n == 2) ? -a : a, n >= 2 ? -b : b);
}

// ---------------------------------------------------------------- pieces of W elements

// as loaded: 16 bytes, or one element
template <int DT, int W>
struct Piece {
  static_assert(W == 1 || W == (DT == RLT_F32 ? 4 : 8), "16-byte pieces");
  typedef typename std::conditional<W == 1, float, uint4>::type T;
  T raw;

  __device__ __forceinline__ void load(const void* base, int64_t at) {
    if constexpr (W == 1) raw = load_as_f32<DT>(base, at);
    else if constexpr (DT == RLT_F32) raw = *(const uint4*)((const float*)base + at);
    else raw = *(const uint4*)((const uint16_t*)base + at);
  }
  __device__ __forceinline__ void clear() {
    if constexpr (W == 1) raw = 0.f;
    else raw = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void floats(float (&x)[W]) const {
    if constexpr (W == 1) {
      x[0] = raw;
    } else {
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == RLT_F32) {
          x[i] = __uint_as_float(w[i]);
        } else if constexpr (DT == RLT_BF16) {
          x[2 * i] = bf16_bits_to_f32((uint16_t)w[i]);
          x[2 * i + 1] = bf16_bits_to_f32((uint16_t)(w[i] >> 16));
        } else {
          x[2 * i] = f16_bits_to_f32((uint16_t)w[i]);
          x[2 * i + 1] = f16_bits_to_f32((uint16_t)(w[i] >> 16));
        }
      }
    }
  }
};

template <int DT, int W>
__device__ __forceinline__ void load_piece(const void* base, int64_t at, float (&x)[W]) {
  Piece<DT, W> p;
  p.load(base, at);
  p.floats(x);
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == RLT_BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
}

template <int DT, int W>
__device__ __forceinline__ void store_piece(void* base, int64_t at, const float (&x)[W]) {
  if constexpr (W == 1) {
    store_from_f32<DT>(base, at, x[0]);
  } else if constexpr (DT == RLT_F32) {
    *(float4*)((float*)base + at) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
    *(uint4*)((uint16_t*)base + at) = make_uint4(pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3]),
                                                 pack2<DT>(x[4], x[5]), pack2<DT>(x[6], x[7]));
  }
}

// ---------------------------------------------------------------- codes

template <int MODE>
constexpr float top_of() { return MODE == kBlockInt8 ? 127.f : rlt_fp8::kMax; }

// A scale and its reciprocal; 0 where quotient() is not for it: a scale that is no positive number,
// or at the ends of float32, where the reciprocal or the remainder would be subnormal.  (Scales
// of blocks are positive, 2^122 at most; below kSmallScale they and their rows are taken kRaise
// times, which moves no bit of a quotient.)
constexpr float kSmallScale = 0x1p-90f, kRaise = 0x1p64f;
struct Divisor {
  float by, inverse;
};
template <int MODE>
__device__ __forceinline__ Divisor divisor(float scale) {
  const bool fits = in_blocks(MODE) || (scale >= kSmallScale && scale <= 0x1p120f);
  return Divisor{scale, fits ? 1.f / scale : 0.f};
}

// x / scale, correctly rounded: the reciprocal is, the first quotient is off by an ulp at most and
// the remainder exact (where the code is not 0: multiples of 2^-33 2^-113), so that one more step
// rounds as the division does, in 3 instructions for its 10.
__device__ __forceinline__ float quotient(float x, const Divisor& d) {
  const float q = x * d.inverse;
  return copysignf(fmaf(fmaf(-q, d.by, x), d.inverse, q), x);  // (the step turns -0 into 0)
}

// x / scale within +-M; e4m3 keeps NaN, int8 takes it as 0.  (Infinities would make the remainder NaN, and so would the
// quotient of a scale that is given, far below x / M.)
template <int MODE>
__device__ __forceinline__ float clamped(float x, const Divisor& d) {
  constexpr float M = MODE == kBlockInt8 ? 127.f : rlt_fp8::kMax;
  float y;
  if constexpr (MODE == kTensorFp8) {
    const float q = x * d.inverse;
    y = fabsf(q) < 2.f * M ? quotient(x, d) : q;
  } else {
    y = fabsf(x) < INFINITY ? quotient(x, d) : x;
  }
  const float c = fminf(fmaxf(y, -M), M);
  return y != y ? (MODE == kBlockInt8 ? 0.f : y) : c;
}

// four codes, round to nearest even
template <int MODE>
__device__ __forceinline__ uint32_t codes4(const float (&x)[4], const Divisor& d) {
  if constexpr (MODE == kBlockInt8) {
    uint32_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = (uint32_t)(int)rintf(clamped<MODE>(x[i], d)) & 0xffu;
    return b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
  } else {
    bool plain = in_blocks(MODE) || d.inverse != 0.f;
    // (a NaN's sign stays, as store_fp8's; a vector that holds one has a scale of NaN)
    if constexpr (MODE == kTensorFp8) plain &= x[0] == x[0] && x[1] == x[1] && x[2] == x[2] && x[3] == x[3];
    if (plain) {
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(clamped<MODE>(x[0], d), clamped<MODE>(x[1], d), 0, false);
      return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(clamped<MODE>(x[2], d), clamped<MODE>(x[3], d), w, true);
    }
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= rlt_fp8::encode(x[i], d.by) << (8 * i);
    return w;
  }
}
template <int MODE>
__device__ __forceinline__ float value_of(uint32_t code) {
  if constexpr (MODE == kBlockInt8) return (float)(int8_t)code;
  else return fp8x2_to_f32<false>(code).x;
}

template <int MODE, int W>
__device__ __forceinline__ void store_codes(void* pool, int64_t at, const float (&x)[W], const Divisor& d) {
  uint8_t* const p = (uint8_t*)pool + at;
  if constexpr (W == 1) {
    const float y[4] = {x[0], 0.f, 0.f, 0.f};
    *p = (uint8_t)codes4<MODE>(y, d);
  } else {
    uint32_t w[W / 4];
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const float y[4] = {x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]};
      w[i] = codes4<MODE>(y, d);
    }
    if constexpr (W == 8) *(uint2*)p = make_uint2(w[0], w[1]);
    else *(uint32_t*)p = w[0];
  }
}

// |x| as a block's maximum takes it: what is not finite does not move a scale.
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}

// ---------------------------------------------------------------- the kernel

// One head's rows of a chunk: lane group g of LP lanes holds row RPW st + g in step st, a lane NS
// slots of two W-element pieces (a and b).
template <int W, int NS, int NSTEP>
struct Held {
  float x[NSTEP][NS][2][W];
};

template <int DT, int W, int NS, int NSTEP>
struct Raw {
  Piece<DT, W> x[NSTEP][NS][2];
};

// (four waves a SIMD: left to itself the compiler takes up to 165 registers for the addresses of
// a block's rows, and 8 prompts of 2048 into int8 56 us for 45)
template <int DT, int W, int LP, int MODE>
__global__ __launch_bounds__(kThreads, 4) void rlt_rotary_kernel(Params P) {
  constexpr int kRows = rows_of(MODE);
  constexpr int NS = W == 1 ? 2 : 1;
  constexpr int RPW = 64 / LP;
  constexpr int NSTEP = kRows < RPW ? 1 : kRows / RPW;
  constexpr bool BLOCKS = in_blocks(MODE);
  __shared__ float2 table[kRows * kMaxPairs];
  __shared__ float tops[BLOCKS ? kMaxKvItems : 1];
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int pairs = P.rotary_dim / 2;
  // (before the chain of loads that finds the rows)
  const double turns0 = pairs ? P.turns[t % pairs] : 0.0;

  // ---- the tile's rows [i0, i1) of its sequence
  const uint32_t tile_index = P.first_group + blockIdx.x;
  int64_t begin = 0;    // packed row of the sequence's first
  int count, start = 0; // its rows, and the position of the first
  int seq = 0, i0, i1, page = 0;
  if constexpr (MODE == kApply) {
    begin = (int64_t)tile_index * kRows;
    count = (int)min((int64_t)kRows, P.rows - begin);
    i0 = 0;
    i1 = count;
  } else {
    seq = (int)(tile_index / (uint32_t)P.tiles);
    const int tile = (int)(tile_index - (uint32_t)seq * P.tiles);
    const int64_t b = P.cu[seq], e = P.cu[seq + 1];
    begin = b < 0 ? 0 : b > P.rows ? P.rows : b;
    // (all n rows end at the sequence's last position; the first max_rows of them are worked on)
    const int64_t n = max((e > P.rows ? P.rows : e) - begin, (int64_t)0);
    count = (int)min(n, (int64_t)P.max_rows);
    start = (int)(P.lengths[seq] - n);
    if constexpr (BLOCKS) {
      const int first = start >= 0 ? start / P.block_size
                                   : -(int)(((int64_t)P.block_size - 1 - start) / P.block_size);
      page = first + tile;
      const int64_t from = (int64_t)page * P.block_size - start;
      i0 = (int)(from < 0 ? 0 : from);
      i1 = (int)(from + P.block_size < count ? from + P.block_size : count);
    } else {
      i0 = tile * kRows;
      i1 = min(count, i0 + kRows);
    }
  }
  if (i0 >= i1) return;  // uniform over the workgroup

  // the pool block of page `idx` of the sequence (-1: not in the pool, nothing is written)
  auto block_at = [&](int idx) {
    const int32_t e = idx >= 0 && idx < P.table_width ? P.tables[(int64_t)seq * P.table_stride + idx] : -1;
    return e >= 0 && e < P.num_blocks ? e : -1;
  };
  const int entry = BLOCKS ? block_at(page) : 0;
  const int o0 = BLOCKS ? start + i0 - page * P.block_size : 0;  // offset of row i0 in its block

  auto sines = [&](int c0, int c1) {
    for (int e = t; e < (c1 - c0) * pairs; e += kThreads) {
      const int r = e / pairs, p = e - r * pairs;
      const int64_t row = begin + c0 + r;
      const int64_t pos = P.positions ? P.positions[row] : (int64_t)start + c0 + r;
      const float2 cs = turn((double)pos * (e == t || kThreads % pairs == 0 ? turns0 : P.turns[p]));
      table[r * pairs + p] = make_float2(cs.x * P.amplitude, cs.y * P.amplitude * P.sign);
    }
  };

  // ---- lane constants: slots of pieces (a, b)
  const int in_group = lane % LP, group = lane / LP;
  const int turning = P.interleaved || W == 1 ? P.rotary_dim / (2 * W) : pairs / W;
  const int pieces = (P.head_dim + 2 * W - 1) / (2 * W);
  int at_a[NS], at_b[NS];  // element of each piece, -1: none
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const int i = in_group + LP * n;
    at_a[n] = at_b[n] = -1;
    if (i < pieces) {
      if (i < turning && !P.interleaved) {
        at_a[n] = W * i;
        at_b[n] = pairs + W * i;
      } else {
        at_a[n] = 2 * W * i;
        at_b[n] = 2 * W * i + W < P.head_dim ? 2 * W * i + W : -1;
      }
    }
  }

  // rows [c0, c1) of one head, as loaded
  auto fetch = [&](Raw<DT, W, NS, NSTEP>& raw, const Side& s, int head, int c0, int c1) {
#pragma unroll
    for (int st = 0; st < NSTEP; ++st) {
      if (st * RPW >= c1 - c0) continue;  // uniform
      const int r = st * RPW + group;
      const int64_t at = (begin + c0 + r) * s.src_row + (int64_t)head * s.src_head;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        raw.x[st][n][0].clear();
        raw.x[st][n][1].clear();
        if (r < c1 - c0) {
          if (at_a[n] >= 0) raw.x[st][n][0].load(s.src, at + at_a[n]);
          if (at_b[n] >= 0) raw.x[st][n][1].load(s.src, at + at_b[n]);
        }
      }
    }
  };
  // as float32, turned if `turns`
  auto expand = [&](Held<W, NS, NSTEP>& held, const Raw<DT, W, NS, NSTEP>& raw, bool turns, int c0, int c1) {
#pragma unroll
    for (int st = 0; st < NSTEP; ++st) {
      if (st * RPW >= c1 - c0) continue;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        raw.x[st][n][0].floats(held.x[st][n][0]);
        raw.x[st][n][1].floats(held.x[st][n][1]);
      }
    }
    if (!turns) return;
#pragma unroll
    for (int st = 0; st < NSTEP; ++st) {
      if (st * RPW >= c1 - c0) continue;
      const int r = st * RPW + group;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        const int i = in_group + LP * n;
        if (i >= turning || r >= c1 - c0) continue;
        float(&a)[W] = held.x[st][n][0];
        float(&b)[W] = held.x[st][n][1];
        const float2* const cs = table + r * pairs + W * i;
        if (W == 1 || !P.interleaved) {
#pragma unroll
          for (int e = 0; e < W; ++e) {
            const float2 z = cs[e];
            const float u = a[e] * z.x - b[e] * z.y, v = a[e] * z.y + b[e] * z.x;
            a[e] = u;
            b[e] = v;
          }
        } else {
#pragma unroll
          for (int e = 0; e + 1 < W; e += 2) {
            const float2 y = cs[e / 2], z = cs[W / 2 + e / 2];
            const float ua = a[e] * y.x - a[e + 1] * y.y, va = a[e] * y.y + a[e + 1] * y.x;
            const float ub = b[e] * z.x - b[e + 1] * z.y, vb = b[e] * z.y + b[e + 1] * z.x;
            a[e] = ua;
            a[e + 1] = va;
            b[e] = ub;
            b[e + 1] = vb;
          }
        }
      }
    }
  };
  // the largest finite |x| of the held rows, in every lane
  auto top = [&](const Held<W, NS, NSTEP>& held, int rows) {
    float m = 0.f;
#pragma unroll
    for (int st = 0; st < NSTEP; ++st) {
      if (st * RPW >= rows) continue;
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int e = 0; e < W; ++e)
          m = fmaxf(m, fmaxf(finite_abs(held.x[st][n][0][e]), finite_abs(held.x[st][n][1][e])));
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, RLT_WAVE));
    return m;
  };

  // k and v first (their scales are a longer chain), then q
  const int kv_items = MODE == kApply ? P.hkv : 2 * P.hkv;
  const int items = kv_items + P.hq;
  const int first_item = wave + kWavesPerGroup * blockIdx.y, step = kWavesPerGroup * gridDim.y;
  auto side = [&](int item) -> const Side& { return item >= kv_items ? P.q : item < P.hkv ? P.k : P.v; };
  auto head_of = [&](int item) { return item >= kv_items ? item - kv_items : item < P.hkv ? item : item - P.hkv; };
  auto scale_at = [&](int item) {
    return side(item).scale + (int64_t)entry * P.s_block + (int64_t)head_of(item) * P.s_head;
  };
  const bool several = BLOCKS && i1 - i0 > kRows;
  Raw<DT, W, NS, NSTEP> raw;
  if constexpr (BLOCKS) {
    if (several) {
      // a block of more rows than are held: its maxima first
      for (int i = t; i < kv_items; i += kThreads) tops[i] = 0.f;
      for (int c0 = i0; c0 < i1; c0 += kRows) {
        const int c1 = min(c0 + kRows, i1);
        __syncthreads();
        sines(c0, c1);
        __syncthreads();
        for (int item = first_item; item < kv_items; item += step) {
          Held<W, NS, NSTEP> held;
          fetch(raw, side(item), head_of(item), c0, c1);
          expand(held, raw, item < P.hkv, c0, c1);
          const float m = top(held, c1 - c0);
          if (lane == 0) tops[item] = fmaxf(tops[item], m);
        }
      }
    }
  }
  for (int c0 = i0; c0 < i1; c0 += kRows) {
    const int c1 = min(c0 + kRows, i1);
    // an item's rows and its block's scale are loaded while the one before it is worked on, the
    // first one's while the sines are made
    float old_next = 0.f;
    auto ahead = [&](int item) {
      if (item >= items) return;
      fetch(raw, side(item), head_of(item), c0, c1);
      if (BLOCKS && item < kv_items && entry >= 0) old_next = *scale_at(item);
    };
    ahead(first_item);
    if (several) __syncthreads();
    sines(c0, c1);
    __syncthreads();
    for (int item = first_item; item < items; item += step) {
      const bool is_q = item >= kv_items;
      const int head = head_of(item);
      const Side& s = side(item);
      Held<W, NS, NSTEP> held;
      expand(held, raw, is_q || item < P.hkv, c0, c1);
      const float old = old_next;
      ahead(item + step);

      if (MODE == kApply || is_q) {
#pragma unroll
        for (int st = 0; st < NSTEP; ++st) {
          const int r = st * RPW + group;
          if (r >= c1 - c0) continue;
          const int64_t at = (begin + c0 + r) * s.dst_row + (int64_t)head * s.dst_head;
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            if (at_a[n] >= 0) store_piece<DT, W>(s.dst, at + at_a[n], held.x[st][n][0]);
            if (at_b[n] >= 0) store_piece<DT, W>(s.dst, at + at_b[n], held.x[st][n][1]);
          }
        }
        continue;
      }
      if constexpr (BLOCKS) {
        if (entry < 0) continue;
        const float m = several ? tops[item] : top(held, c1 - c0);
        const float fresh = fmaxf(m * (1.f / top_of<MODE>()), rlt_fp8::kTiny);
        const float scale = o0 > 0 && old > fresh ? old : fresh;
        const float raise =
            __builtin_amdgcn_readfirstlane(__float_as_int(scale)) < __float_as_int(kSmallScale) ? kRaise : 1.f;
        const Divisor by = divisor<MODE>(scale * raise);
        const int64_t base = (int64_t)entry * s.dst_block + (int64_t)head * s.dst_head;
        if (c0 == i0 && o0 > 0 && scale > old) {
          // the block's earlier codes, over the new scale
          const int per_row = P.head_dim / W, n = o0 * per_row;
          for (int e = lane; e < n; e += 64) {
            const int r = e / per_row;
            const int64_t at = base + (int64_t)r * s.dst_row + (e - r * per_row) * W;
            float x[W];
#pragma unroll
            for (int u = 0; u < W; ++u) x[u] = value_of<MODE>(((const uint8_t*)s.dst)[at + u]) * old * raise;
            store_codes<MODE, W>(s.dst, at, x, by);
          }
        }
        if (lane == 0 && c1 == i1) *scale_at(item) = scale;  // (the last chunk: all read the old one)
#pragma unroll
        for (int st = 0; st < NSTEP; ++st) {
          const int r = st * RPW + group;
          if (r >= c1 - c0) continue;
          const int64_t at = base + (int64_t)(o0 + (c0 - i0) + r) * s.dst_row;
#pragma unroll
          for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int el = half ? at_b[n] : at_a[n];
              if (el < 0) continue;
              float x[W];
#pragma unroll
              for (int u = 0; u < W; ++u) x[u] = held.x[st][n][half][u] * raise;
              store_codes<MODE, W>(s.dst, at + el, x, by);
            }
          }
        }
      } else if constexpr (MODE != kApply) {
#pragma unroll
        for (int st = 0; st < NSTEP; ++st) {
          if (st * RPW >= c1 - c0) continue;  // uniform
          const int r = st * RPW + group;
          const int pos = start + c0 + r;
          const int e = r < c1 - c0 && pos >= 0 ? block_at(pos / P.block_size) : -1;
          const int off = pos % P.block_size;
          float scale = 1.f;
          if constexpr (MODE == kTensorFp8) scale = s.scale[0];
          if constexpr (MODE == kVectorFp8) {
            // (NaN-propagating, as rlt_kv_store_fp8's)
            float m = 0.f;
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
              for (int u = 0; u < W; ++u)
                m = rlt_fp8::nan_max(m, rlt_fp8::nan_max(fabsf(held.x[st][n][0][u]), fabsf(held.x[st][n][1][u])));
#pragma unroll
            for (int o = LP / 2; o >= 1; o >>= 1) m = rlt_fp8::nan_max(m, __shfl_xor(m, o, RLT_WAVE));
            scale = rlt_fp8::dynamic_scale(m);
          }
          if (e < 0) continue;
          const Divisor by = divisor<MODE>(scale);
          const int64_t at = (int64_t)e * s.dst_block + (int64_t)off * s.dst_row + (int64_t)head * s.dst_head;
          if (MODE == kVectorFp8 && in_group == 0)
            s.scale[(int64_t)e * P.s_block + (int64_t)off * P.s_token + (int64_t)head * P.s_head] = scale;
#pragma unroll
          for (int n = 0; n < NS; ++n) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int el = half ? at_b[n] : at_a[n];
              if (el < 0) continue;
              if constexpr (MODE == kSame) store_piece<DT, W>(s.dst, at + el, held.x[st][n][half]);
              else store_codes<MODE, W>(s.dst, at + el, held.x[st][n][half], by);
            }
          }
        }
      }
    }
  }
}

// ---------------------------------------------------------------- reading back

struct LoadParams {
  const void* k;
  const void* v;
  int64_t k_block, k_token, k_head, v_block, v_token, v_head;
  const float* ks;
  const float* vs;
  int64_t s_block, s_token, s_head;  // 0 where the scales have no such axis
  const int32_t* tables;
  int64_t table_stride;
  int32_t table_width, num_blocks, block_size;
  const int32_t* lengths;
  const int32_t* cu;
  int64_t rows;
  int32_t num_seqs, max_rows, tiles, tile_rows, hkv, head_dim;
  uint32_t first_group;  // of the launch
  void* k_out;
  void* v_out;
};

// W consecutive elements of a pool as float32, in one load where W is more than 1.
template <int CT, int W>
__device__ __forceinline__ void load_elements(const void* pool, int64_t at, float (&x)[W]) {
  if constexpr (W == 1) {
    x[0] = load_as_f32<CT>(pool, at);
  } else if constexpr (CT == RLT_FP8_E4M3 || CT == RLT_INT8) {
    static_assert(W == 16, "16-byte pieces");
    const uint4 v = *(const uint4*)((const uint8_t*)pool + at);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (CT == RLT_INT8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * i + j] = (float)(int8_t)(w[i] >> (8 * j));
      } else {
        const float2 lo = fp8x2_to_f32<false>(w[i]), hi = fp8x2_to_f32<true>(w[i]);
        x[4 * i] = lo.x; x[4 * i + 1] = lo.y; x[4 * i + 2] = hi.x; x[4 * i + 3] = hi.y;
      }
    }
  } else {
    load_piece<CT, W>(pool, at, x);
  }
}

// W consecutive floats to an output, 16 bytes a store.
template <int OT, int W>
__device__ __forceinline__ void store_elements(void* out, int64_t at, const float (&x)[W]) {
  if constexpr (W == 1) {
    store_from_f32<OT>(out, at, x[0]);
  } else {
    constexpr int P = OT == RLT_F32 ? 4 : 8;
    static_assert(W % P == 0 || W < P, "whole stores");
    if constexpr (W < P) {
      // (float32 pools read as 16 bits: 8 bytes)
      *(uint2*)((uint16_t*)out + at) = make_uint2(pack2<OT>(x[0], x[1]), pack2<OT>(x[2], x[3]));
    } else {
#pragma unroll
      for (int i = 0; i < W / P; ++i) {
        float y[P];
#pragma unroll
        for (int j = 0; j < P; ++j) y[j] = x[P * i + j];
        store_piece<OT, P>(out, at + P * i, y);
      }
    }
  }
}

// A workgroup takes `tile_rows` rows of a sequence, whose blocks it looks up once; a thread a
// column of W elements over the rows, so that its loads are in flight together.  HBM bounds it
// (16 sequences of up to 8192 positions of 8 heads in int8: 122 us, 4.5 TB/s).
constexpr int kLoadRows = 8;
template <int CT, int OT, int W>
__global__ __launch_bounds__(kThreads) void rlt_kv_load_kernel(LoadParams P) {
  __shared__ int entries[kLoadRows], offsets[kLoadRows];
  const uint32_t tile_index = P.first_group + blockIdx.x;
  const int seq = (int)(tile_index / (uint32_t)P.tiles);
  const int tile = (int)(tile_index - (uint32_t)seq * P.tiles);
  const int64_t b = P.cu[seq], e = P.cu[seq + 1];
  const int64_t begin = b < 0 ? 0 : b > P.rows ? P.rows : b;
  const int64_t n = max((e > P.rows ? P.rows : e) - begin, (int64_t)0);
  const int count = (int)min(n, (int64_t)P.max_rows), start = (int)(P.lengths[seq] - n);
  const int i0 = tile * P.tile_rows, rows = min(count - i0, P.tile_rows);
  if (rows <= 0) return;  // uniform over the workgroup
  const int t = threadIdx.x;
  if (t < rows) {
    const int pos = start + i0 + t;
    const int idx = pos >= 0 ? pos / P.block_size : -1;
    const int32_t x = idx >= 0 && idx < P.table_width ? P.tables[(int64_t)seq * P.table_stride + idx] : -1;
    entries[t] = x >= 0 && x < P.num_blocks ? x : -1;
    offsets[t] = pos - idx * P.block_size;
  }
  __syncthreads();
  // columns of a row (k, then v); where they are fewer than the threads these take several rows
  const int per_vec = (P.head_dim + W - 1) / W, columns = 2 * P.hkv * per_vec;
  const int together = columns < kThreads ? kThreads / columns : 1;
  const int first = columns < kThreads ? t / columns : 0;
  if (first >= together) return;
  for (int c = t - first * columns; c < columns; c += kThreads) {
    const int vec = c / per_vec, d = (c - vec * per_vec) * W;
    const bool value = vec >= P.hkv;
    const int head = value ? vec - P.hkv : vec;
    const void* const pool = value ? P.v : P.k;
    const float* const scales = value ? P.vs : P.ks;
    const int64_t block = value ? P.v_block : P.k_block, token = value ? P.v_token : P.k_token;
    const int64_t from = (int64_t)head * (value ? P.v_head : P.k_head) + d;
    void* const out = value ? P.v_out : P.k_out;
    const int64_t to = ((begin + i0) * P.hkv + head) * P.head_dim + d, row = (int64_t)P.hkv * P.head_dim;
#pragma unroll 4
    for (int r = first; r < rows; r += together) {
      const int entry = entries[r], off = offsets[r];
      float x[W];
#pragma unroll
      for (int u = 0; u < W; ++u) x[u] = 0.f;
      if (entry >= 0) {
        const float scale = scales ? scales[(int64_t)entry * P.s_block + (int64_t)off * P.s_token +
                                            (int64_t)head * P.s_head] : 1.f;
        load_elements<CT, W>(pool, (int64_t)entry * block + (int64_t)off * token + from, x);
#pragma unroll
        for (int u = 0; u < W; ++u) x[u] *= scale;
      }
      store_elements<OT, W>(out, to + r * row, x);
    }
  }
}

// ---------------------------------------------------------------- dispatch

constexpr int kGroupsWanted = 1024;  // workgroups from which the chip is filled

// The heads go to several workgroups where those with rows are few: rows / rows_of, and one more
// for each sequence (6 ragged windows of up to 700 rows, of whose 528 tiles 330 have some, into
// fp8 with a scale per vector: 21.6 -> 19.4 us)
template <int DT, int MODE>
int launch_rotary(Params P, bool vec, int64_t gx, hipStream_t stream) {
  const int items = P.hq + (MODE == kApply ? 1 : 2) * P.hkv;
  const int64_t some = P.rows / rows_of(MODE) + (MODE == kApply ? 1 : P.num_seqs), filled = some < gx ? some : gx;
  const int64_t most = (items + kWavesPerGroup - 1) / kWavesPerGroup, want = (kGroupsWanted + filled - 1) / filled;
  constexpr int W = DT == RLT_F32 ? 4 : 8;
  const int lanes = P.head_dim / (2 * W);  // that hold a vector
  for (int64_t at = 0; at < gx; at += kGridGroups) {
    const dim3 grid((unsigned)(gx - at < kGridGroups ? gx - at : kGridGroups), (unsigned)(want < most ? want : most));
    P.first_group = (uint32_t)at;
    if (!vec) rlt_rotary_kernel<DT, 1, 64, MODE><<<grid, kThreads, 0, stream>>>(P);
    else if (lanes <= 4) rlt_rotary_kernel<DT, W, 4, MODE><<<grid, kThreads, 0, stream>>>(P);
    else if (lanes <= 8) rlt_rotary_kernel<DT, W, 8, MODE><<<grid, kThreads, 0, stream>>>(P);
    else if (lanes <= 16) rlt_rotary_kernel<DT, W, 16, MODE><<<grid, kThreads, 0, stream>>>(P);
    else if constexpr (DT == RLT_F32) rlt_rotary_kernel<DT, W, 32, MODE><<<grid, kThreads, 0, stream>>>(P);
  }
  return rlt_launch_status();
}

template <int MODE>
int launch_rotary_dt(const Params& P, int dtype, bool vec, int64_t gx, hipStream_t stream) {
  switch (dtype) {
    case RLT_F32: return launch_rotary<RLT_F32, MODE>(P, vec, gx, stream);
    case RLT_F16: return launch_rotary<RLT_F16, MODE>(P, vec, gx, stream);
    case RLT_BF16: return launch_rotary<RLT_BF16, MODE>(P, vec, gx, stream);
    default: return RLT_ERR_ARGUMENT;
  }
}

// 16-byte pieces: every address a multiple of `bytes`, given strides in elements of `elt` bytes
bool aligned(const void* p, int64_t a, int64_t b, int64_t c, int elt, int bytes) {
  return (uintptr_t)p % bytes == 0 && a * elt % bytes == 0 && b * elt % bytes == 0 && c * elt % bytes == 0;
}

// the rotation's part of the arguments
int set_turns(Params& P, const double* turns, int32_t rotary_dim, float amplitude, int32_t interleaved,
              int32_t inverse) {
  if (rotary_dim < 0 || rotary_dim % 2 || rotary_dim > P.head_dim || (rotary_dim && !turns))
    return RLT_ERR_ARGUMENT;
  P.turns = turns;
  P.rotary_dim = rotary_dim;
  P.amplitude = amplitude;
  P.interleaved = interleaved ? 1 : 0;
  P.sign = inverse ? -1.f : 1.f;
  return RLT_OK;
}

}  // namespace

extern "C" {

int rlt_rotary(const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k,
               int64_t k_row_stride, int64_t k_head_stride, const int64_t* positions, int64_t rows,
               const double* turns, int32_t rotary_dim, float amplitude, int32_t interleaved,
               int32_t inverse, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
               int32_t dtype, void* q_out, int64_t qo_row_stride, int64_t qo_head_stride,
               void* k_out, int64_t ko_row_stride, int64_t ko_head_stride, hipStream_t stream) {
  if (rows < 0 || num_q_heads < 0 || num_kv_heads < 0 || head_dim <= 0 || head_dim > 2 * kMaxPairs)
    return RLT_ERR_ARGUMENT;
  if (dtype != RLT_F32 && dtype != RLT_F16 && dtype != RLT_BF16) return RLT_ERR_ARGUMENT;
  Params P = {};
  P.q = Side{q, q_row_stride, q_head_stride, q_out, 0, qo_row_stride, qo_head_stride, nullptr};
  P.k = Side{k, k_row_stride, k_head_stride, k_out, 0, ko_row_stride, ko_head_stride, nullptr};
  P.hq = num_q_heads;
  P.hkv = num_kv_heads;
  P.head_dim = head_dim;
  P.rows = rows;
  P.positions = positions;
  if (const int st = set_turns(P, turns, rotary_dim, amplitude, interleaved, inverse)) return st;
  if (rows == 0 || num_q_heads + num_kv_heads == 0) return RLT_OK;
  if (!positions || (num_q_heads && (!q || !q_out)) || (num_kv_heads && (!k || !k_out)))
    return RLT_ERR_ARGUMENT;
  const int elt = dtype == RLT_F32 ? 4 : 2, pair = 32 / elt;
  const bool vec = head_dim % pair == 0 && rotary_dim % pair == 0 &&
                   aligned(q, q_row_stride, q_head_stride, 0, elt, 16) &&
                   aligned(k, k_row_stride, k_head_stride, 0, elt, 16) &&
                   aligned(q_out, qo_row_stride, qo_head_stride, 0, elt, 16) &&
                   aligned(k_out, ko_row_stride, ko_head_stride, 0, elt, 16);
  const int64_t gx = (rows + rows_of(kApply) - 1) / rows_of(kApply);
  if (gx >= ((int64_t)1 << 31)) return RLT_ERR_UNSUPPORTED;
  return launch_rotary_dt<kApply>(P, dtype, vec, gx, stream);
}

int rlt_kv_append(const void* k, int64_t k_row_stride, int64_t k_head_stride, const void* v,
                  int64_t v_row_stride, int64_t v_head_stride, int32_t dtype, void* key_cache,
                  void* value_cache, int64_t k_block_stride, int64_t k_token_stride,
                  int64_t kc_head_stride, int64_t v_block_stride, int64_t v_token_stride,
                  int64_t vc_head_stride, int32_t num_blocks, int32_t block_size, int32_t kv_dtype,
                  float* key_scale, float* value_scale, int32_t scale_mode, int64_t s_block_stride,
                  int64_t s_token_stride, int64_t s_head_stride, const int32_t* block_tables,
                  int64_t table_stride, int32_t table_width, const int32_t* context_lengths,
                  const int32_t* cu_seqlens_q, int32_t num_seqs, int32_t max_q_len, int64_t rows,
                  int32_t num_kv_heads, int32_t head_dim, const int64_t* positions,
                  const double* turns, int32_t rotary_dim, float amplitude, int32_t interleaved,
                  const void* q, int64_t q_row_stride, int64_t q_head_stride, int32_t num_q_heads,
                  void* q_out, int64_t qo_row_stride, int64_t qo_head_stride, hipStream_t stream) {
  if (rows < 0 || num_seqs < 0 || max_q_len < 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      head_dim > 2 * kMaxPairs || num_blocks <= 0 || block_size <= 0 || table_width < 0)
    return RLT_ERR_ARGUMENT;
  if (2 * num_kv_heads > kMaxKvItems) return RLT_ERR_UNSUPPORTED;
  if (dtype != RLT_F32 && dtype != RLT_F16 && dtype != RLT_BF16) return RLT_ERR_ARGUMENT;
  int mode;
  if (kv_dtype == dtype && scale_mode == 0) mode = kSame;
  else if (kv_dtype == RLT_FP8_E4M3 && scale_mode == 1) mode = kTensorFp8;
  else if (kv_dtype == RLT_FP8_E4M3 && scale_mode == 2) mode = kVectorFp8;
  else if (kv_dtype == RLT_FP8_E4M3 && scale_mode == 3) mode = kBlockFp8;
  else if (kv_dtype == RLT_INT8 && scale_mode == 3) mode = kBlockInt8;
  else return RLT_ERR_ARGUMENT;
  if (scale_mode && (!key_scale || !value_scale)) return RLT_ERR_ARGUMENT;
  Params P = {};
  P.hkv = num_kv_heads;
  P.hq = q ? num_q_heads : 0;
  P.head_dim = head_dim;
  P.rows = rows;
  P.positions = positions;
  if (const int st = set_turns(P, turns, rotary_dim, amplitude, interleaved, 0)) return st;
  if (rows == 0 || num_seqs == 0 || max_q_len == 0) return RLT_OK;
  if (!k || !v || !key_cache || !value_cache || !context_lengths || !cu_seqlens_q ||
      (table_width && !block_tables) || P.hq < 0 || (P.hq && !q_out))
    return RLT_ERR_ARGUMENT;
  P.q = Side{q, q_row_stride, q_head_stride, q_out, 0, qo_row_stride, qo_head_stride, nullptr};
  P.k = Side{k, k_row_stride, k_head_stride, key_cache, k_block_stride, k_token_stride, kc_head_stride, key_scale};
  P.v = Side{v, v_row_stride, v_head_stride, value_cache, v_block_stride, v_token_stride, vc_head_stride, value_scale};
  P.s_block = s_block_stride;
  P.s_token = s_token_stride;
  P.s_head = s_head_stride;
  P.tables = block_tables;
  P.table_stride = table_stride;
  P.table_width = table_width;
  P.num_blocks = num_blocks;
  P.block_size = block_size;
  P.lengths = context_lengths;
  P.cu = cu_seqlens_q;
  P.num_seqs = num_seqs;
  if (max_q_len > rows) max_q_len = (int32_t)rows;  // (a longest window known by its bound only)
  // blocks that a window of max_q_len rows meets, or its groups of rows
  const int64_t tiles = in_blocks(mode) ? ((int64_t)max_q_len + block_size - 2) / block_size + 1
                                        : ((int64_t)max_q_len + rows_of(mode) - 1) / rows_of(mode);
  const int64_t gx = tiles * num_seqs;
  if (gx >= ((int64_t)1 << 31)) return RLT_ERR_UNSUPPORTED;
  P.max_rows = max_q_len;
  P.tiles = (int32_t)tiles;
  const int elt = dtype == RLT_F32 ? 4 : 2, pair = 32 / elt;
  const int code = mode == kSame ? elt : 1, piece = 16 / elt * code;  // bytes of a piece in the pool
  const bool vec = head_dim % pair == 0 && rotary_dim % pair == 0 &&
                   aligned(k, k_row_stride, k_head_stride, 0, elt, 16) &&
                   aligned(v, v_row_stride, v_head_stride, 0, elt, 16) &&
                   aligned(key_cache, k_block_stride, k_token_stride, kc_head_stride, code, piece) &&
                   aligned(value_cache, v_block_stride, v_token_stride, vc_head_stride, code, piece) &&
                   (!P.hq || (aligned(q, q_row_stride, q_head_stride, 0, elt, 16) &&
                              aligned(q_out, qo_row_stride, qo_head_stride, 0, elt, 16)));
  switch (mode) {
    case kSame: return launch_rotary_dt<kSame>(P, dtype, vec, gx, stream);
    case kTensorFp8: return launch_rotary_dt<kTensorFp8>(P, dtype, vec, gx, stream);
    case kVectorFp8: return launch_rotary_dt<kVectorFp8>(P, dtype, vec, gx, stream);
    case kBlockFp8: return launch_rotary_dt<kBlockFp8>(P, dtype, vec, gx, stream);
    default: return launch_rotary_dt<kBlockInt8>(P, dtype, vec, gx, stream);
  }
}

}  // extern "C"

namespace {

template <int CT, int OT>
int launch_load(LoadParams P, bool vec, int64_t gx, hipStream_t stream) {
  constexpr int W = CT == RLT_F32 ? 4 : CT == RLT_FP8_E4M3 || CT == RLT_INT8 ? 16 : 8;
  for (int64_t at = 0; at < gx; at += kGridGroups) {
    const unsigned grid = (unsigned)(gx - at < kGridGroups ? gx - at : kGridGroups);
    P.first_group = (uint32_t)at;
    if (vec) rlt_kv_load_kernel<CT, OT, W><<<grid, kThreads, 0, stream>>>(P);
    else rlt_kv_load_kernel<CT, OT, 1><<<grid, kThreads, 0, stream>>>(P);
  }
  return rlt_launch_status();
}

template <int CT>
int launch_load_ot(const LoadParams& P, int out_dtype, bool vec, int64_t gx, hipStream_t stream) {
  switch (out_dtype) {
    case RLT_F32: return launch_load<CT, RLT_F32>(P, vec, gx, stream);
    case RLT_F16: return launch_load<CT, RLT_F16>(P, vec, gx, stream);
    case RLT_BF16: return launch_load<CT, RLT_BF16>(P, vec, gx, stream);
    default: return RLT_ERR_ARGUMENT;
  }
}

}  // namespace

extern "C" int rlt_kv_load(const void* key_cache, const void* value_cache, int64_t k_block_stride,
                           int64_t k_token_stride, int64_t k_head_stride, int64_t v_block_stride,
                           int64_t v_token_stride, int64_t v_head_stride, int32_t num_blocks,
                           int32_t block_size, int32_t kv_dtype, const float* key_scale,
                           const float* value_scale, int32_t scale_mode, int64_t s_block_stride,
                           int64_t s_token_stride, int64_t s_head_stride,
                           const int32_t* block_tables, int64_t table_stride, int32_t table_width,
                           const int32_t* context_lengths, const int32_t* cu_seqlens,
                           int32_t num_seqs, int32_t max_len, int64_t rows, int32_t num_kv_heads,
                           int32_t head_dim, int32_t out_dtype, void* k_out, void* v_out,
                           hipStream_t stream) {
  if (rows < 0 || num_seqs < 0 || max_len < 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      num_blocks <= 0 || block_size <= 0 || table_width < 0 || scale_mode < 0 || scale_mode > 3)
    return RLT_ERR_ARGUMENT;
  const bool codes = kv_dtype == RLT_FP8_E4M3 || kv_dtype == RLT_INT8;
  if (codes != (scale_mode != 0) || (kv_dtype == RLT_INT8 && scale_mode != 3)) return RLT_ERR_ARGUMENT;
  if (scale_mode && (!key_scale || !value_scale)) return RLT_ERR_ARGUMENT;
  if (rows == 0 || num_seqs == 0 || max_len == 0) return RLT_OK;
  if (!key_cache || !value_cache || !context_lengths || !cu_seqlens || !k_out || !v_out ||
      (table_width && !block_tables))
    return RLT_ERR_ARGUMENT;
  if (max_len > rows) max_len = (int32_t)rows;
  LoadParams P = {};
  P.k = key_cache;
  P.v = value_cache;
  P.k_block = k_block_stride;
  P.k_token = k_token_stride;
  P.k_head = k_head_stride;
  P.v_block = v_block_stride;
  P.v_token = v_token_stride;
  P.v_head = v_head_stride;
  P.ks = scale_mode ? key_scale : nullptr;
  P.vs = scale_mode ? value_scale : nullptr;
  P.s_block = scale_mode >= 2 ? s_block_stride : 0;
  P.s_token = scale_mode == 2 ? s_token_stride : 0;
  P.s_head = scale_mode >= 2 ? s_head_stride : 0;
  P.tables = block_tables;
  P.table_stride = table_stride;
  P.table_width = table_width;
  P.num_blocks = num_blocks;
  P.block_size = block_size;
  P.lengths = context_lengths;
  P.cu = cu_seqlens;
  P.rows = rows;
  P.num_seqs = num_seqs;
  P.max_rows = max_len;
  P.hkv = num_kv_heads;
  P.head_dim = head_dim;
  P.k_out = k_out;
  P.v_out = v_out;
  // (few rows: shorter tiles, whose threads wait for fewer loads in turn)
  P.tile_rows = kLoadRows;
  auto groups = [&]() { return ((int64_t)max_len + P.tile_rows - 1) / P.tile_rows * num_seqs; };
  while (P.tile_rows > 4 && groups() < kGroupsWanted) P.tile_rows /= 2;
  const int64_t gx = groups();
  if (gx >= ((int64_t)1 << 31)) return RLT_ERR_UNSUPPORTED;
  P.tiles = (int32_t)(gx / num_seqs);
  const int elt = kv_dtype == RLT_F32 ? 4 : codes ? 1 : 2;
  const bool vec = head_dim % (16 / elt) == 0 &&
                   aligned(key_cache, k_block_stride, k_token_stride, k_head_stride, elt, 16) &&
                   aligned(value_cache, v_block_stride, v_token_stride, v_head_stride, elt, 16) &&
                   ((uintptr_t)k_out | (uintptr_t)v_out) % 16 == 0;
  switch (kv_dtype) {
    case RLT_F32: return launch_load_ot<RLT_F32>(P, out_dtype, vec, gx, stream);
    case RLT_F16: return launch_load_ot<RLT_F16>(P, out_dtype, vec, gx, stream);
    case RLT_BF16: return launch_load_ot<RLT_BF16>(P, out_dtype, vec, gx, stream);
    case RLT_FP8_E4M3: return launch_load_ot<RLT_FP8_E4M3>(P, out_dtype, vec, gx, stream);
    case RLT_INT8: return launch_load_ot<RLT_INT8>(P, out_dtype, vec, gx, stream);
    default: return RLT_ERR_ARGUMENT;
  }
}
