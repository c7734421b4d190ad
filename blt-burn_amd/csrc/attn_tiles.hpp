// What the attention kernels over key tiles share: operand layouts, row arithmetic
// and the handling of values that are not finite.
#pragma once
#include "common.hpp"

namespace blt {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
#define LDS_PTR(p) ((__attribute__((address_space(3))) s16x4_t*)(p))

// x / d for 0 <= x < 2^31 by one product: m = floor(2^s / d) + 1 with s = 31 + ceil(log2 d)
// is at most 2^s / d + 1, so x m / 2^s passes x / d by less than 1 / d.
struct Divisor {
  uint32_t m;
  int s;
};
inline Divisor divisor_of(int d) {
  int l = 0;
  while (((int64_t)1 << l) < d) ++l;
  return Divisor{(uint32_t)(((uint64_t)1 << (31 + l)) / (uint64_t)d + 1), 31 + l};
}
__device__ inline int over(int x, const Divisor& d) {
  return (int)(((uint64_t)(uint32_t)x * d.m) >> d.s);
}

__device__ inline float uniform(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}

// Words of two bf16 values: the largest exponents seen so far; whether one of them is an
// infinite value's or a NaN's; a word with such values zeroed.
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
__device__ inline uint32_t exponents2(uint32_t seen, uint32_t x) {
  return __builtin_bit_cast(
      uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, seen),
                                          __builtin_bit_cast(u16x2_t, x & 0x7f807f80u)));
}
__device__ inline bool not_finite2(uint32_t seen) {
  return (seen & 0xffffu) == 0x7f80u || (seen >> 16) == 0x7f80u;
}
__device__ inline uint32_t finite2(uint32_t x) {
  x = (x & 0x7f800000u) == 0x7f800000u ? x & 0xffffu : x;
  return (x & 0x7f80u) == 0x7f80u ? x & 0xffff0000u : x;
}

// p = 2^(s c - m c) is one fma with m c rounded, which is off by 2^-24 |m c| in the exponent: much
// where scores are large (beyond 2^31 the largest key's p would overflow or vanish).  From here
// on m is taken from s first, which is exact.  Only looked at where a wave's offsets move.
constexpr float kFar = 1024.f;

}  // namespace blt
