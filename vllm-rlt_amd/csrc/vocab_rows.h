// Rows of a vocabulary split over workgroups: loads, and the order of a row's columns
// (descending value, NaN first, equal values by ascending column).
#pragma once

#include "common.h"

namespace vocab {

constexpr int kThreads = 256;

// Monotone 32-bit key of a logit: larger keys are larger values, NaN the largest, the two
// zeros equal; no value has key 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  if (x != x) return 0xffffffffu;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// Larger composites come first in the row's order; 0 is no column.
__device__ __forceinline__ unsigned long long composite(uint32_t key, uint32_t col) {
  return ((unsigned long long)key << 32) | (uint32_t)~col;
}
__device__ __forceinline__ uint32_t composite_col(unsigned long long c) { return ~(uint32_t)c; }

template <int DT>
__host__ __device__ constexpr int elements() { return DT == RLT_F32 ? 4 : 8; }  // in 16 bytes

// 16 bytes of a row at any element's alignment
template <int DT>
struct Piece;
template <>
struct Piece<RLT_F32> {
  struct __attribute__((packed, aligned(4))) T { uint32_t w[4]; };
};
template <>
struct Piece<RLT_BF16> {
  struct __attribute__((packed, aligned(2))) T { uint32_t w[4]; };
};
template <>
struct Piece<RLT_F16> {
  struct __attribute__((packed, aligned(2))) T { uint32_t w[4]; };
};

template <int DT>
__device__ __forceinline__ float piece_at(const typename Piece<DT>::T& p, int e) {
  if constexpr (DT == RLT_F32) return __uint_as_float(p.w[e]);
  else {
    const uint16_t b = (uint16_t)(e & 1 ? p.w[e >> 1] >> 16 : p.w[e >> 1]);
    return DT == RLT_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
  }
}

// A slice of EPT * kThreads columns from `begin`: element e of piece i of thread t is column
// begin + (i kThreads + t) elements() + e.
template <int DT, int EPT>
struct Slice {
  static constexpr int VE = elements<DT>();
  static constexpr int NP = EPT / VE;
  static_assert(NP * VE == EPT, "whole pieces");
  typename Piece<DT>::T p[NP];
  __device__ static __forceinline__ int64_t column(int64_t begin, int i) {
    return begin + (int64_t)(i * kThreads + (int)threadIdx.x) * VE;
  }
  // all loads in flight together; columns past the row are not read
  __device__ __forceinline__ void load(const void* row, int64_t begin, int64_t vocab) {
    using T = typename Piece<DT>::T;
    constexpr int ELT = DT == RLT_F32 ? 4 : 2;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int64_t c = column(begin, i);
      if (c + VE <= vocab) {
        p[i] = *(const T*)((const uint8_t*)row + c * ELT);
      } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) p[i].w[w] = 0;
        for (int e = 0; e < VE; ++e) {
          if (c + e < vocab) {
            if constexpr (DT == RLT_F32) p[i].w[e] = ((const uint32_t*)row)[c + e];
            else p[i].w[e >> 1] |= (uint32_t)((const uint16_t*)row)[c + e] << (16 * (e & 1));
          }
        }
      }
    }
  }
  __device__ __forceinline__ float at(int i, int e) const { return piece_at<DT>(p[i], e); }
  // (a value that the type holds)
  __device__ __forceinline__ void set(int i, int e, float v) {
    if constexpr (DT == RLT_F32) {
      p[i].w[e] = __float_as_uint(v);
    } else {
      const uint32_t b = DT == RLT_BF16 ? f32_to_bf16_bits(v) : f32_to_f16_bits(v);
      p[i].w[e >> 1] = e & 1 ? (p[i].w[e >> 1] & 0xffffu) | b << 16 : (p[i].w[e >> 1] & 0xffff0000u) | b;
    }
  }
};

__device__ __forceinline__ unsigned long long wave_max(unsigned long long x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const unsigned long long y = __shfl_xor(x, o, RLT_WAVE);
    x = x > y ? x : y;
  }
  return x;
}

}  // namespace vocab
