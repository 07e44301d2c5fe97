// Rows of a vocabulary split over workgroups: loads, and the order of a row's columns
// (descending value, NaN first, equal values by ascending column).
#pragma once

#include "common.h"

#include <type_traits>

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

// A value combined over the wave by lane exchanges of the vector unit (quads, halves, rows of
// 16, then the row pairs): the same exchanges through LDS took a large part of these kernels.
template <class F>
__device__ __forceinline__ uint32_t wave_join(uint32_t x, F f) {
  auto step = [&](auto ctrl) {
    x = f(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, true));
  };
  step(std::integral_constant<int, 0xB1>{});   // quad_perm: lane ^ 1
  step(std::integral_constant<int, 0x4E>{});   // quad_perm: lane ^ 2
  step(std::integral_constant<int, 0x141>{});  // row_half_mirror: the other quad of eight
  step(std::integral_constant<int, 0x140>{});  // row_mirror: the other eight of the row
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = f(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return f(b[0], b[1]);
}
__device__ __forceinline__ float wave_max(float x) {
  return __uint_as_float(wave_join(__float_as_uint(x), [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t x) {
  return wave_join(x, [](uint32_t a, uint32_t b) { return a + b; });
}
// the same of 64-bit values, as (low, high) halves
template <class F>
__device__ __forceinline__ uint64_t wave_join(uint64_t x, F f) {
  auto step = [&](auto ctrl) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(x >> 32), decltype(ctrl)::value, 0xf, 0xf, true);
    x = f(x, (uint64_t)hi << 32 | lo);
  };
  step(std::integral_constant<int, 0xB1>{});
  step(std::integral_constant<int, 0x4E>{});
  step(std::integral_constant<int, 0x141>{});
  step(std::integral_constant<int, 0x140>{});
  auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
  auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(x >> 32), (uint32_t)(x >> 32), false, false);
  x = f((uint64_t)hi[0] << 32 | lo[0], (uint64_t)hi[1] << 32 | lo[1]);
  lo = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
  hi = __builtin_amdgcn_permlane32_swap((uint32_t)(x >> 32), (uint32_t)(x >> 32), false, false);
  return f((uint64_t)hi[0] << 32 | lo[0], (uint64_t)hi[1] << 32 | lo[1]);
}
__device__ __forceinline__ double wave_sum(double x) {
  return __longlong_as_double((long long)wave_join((uint64_t)__double_as_longlong(x), [](uint64_t a, uint64_t b) {
    return (uint64_t)__double_as_longlong(__longlong_as_double((long long)a) + __longlong_as_double((long long)b));
  }));
}
__device__ __forceinline__ unsigned long long wave_max(unsigned long long x) {
  return wave_join((uint64_t)x, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
}

}  // namespace vocab
