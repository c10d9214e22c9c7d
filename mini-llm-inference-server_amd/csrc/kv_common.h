// What the kernels that write the pools share: conversions of 16-bit values, the rotation of a pair as torch evaluates it,
// quantised rows of fp8 and 4-bit pools.
#pragma once

#include <type_traits>

#include "common.h"

namespace mllm {
namespace {

template <typename T>
__device__ __forceinline__ float to_f32(uint16_t b) {
  if constexpr (std::is_same<T, BF16>::value)
    return bf16_bits_to_f32(b);
  else
    return f16_bits_to_f32(b);
}
template <typename T>
__device__ __forceinline__ uint16_t from_f32(float f) {
  if constexpr (std::is_same<T, BF16>::value)
    return f32_to_bf16_bits(f);
  else
    return f32_to_f16_bits(f);
}

// Four 16-bit values (two dwords) -> four e4m3fn bytes of x * inv.
template <typename T>
__device__ __forceinline__ uint32_t quant4(uint32_t w0, uint32_t w1, float inv) {
  return f32_to_e4m3fn_bits(to_f32<T>((uint16_t)w0) * inv) |
         (f32_to_e4m3fn_bits(to_f32<T>((uint16_t)(w0 >> 16)) * inv) << 8) |
         (f32_to_e4m3fn_bits(to_f32<T>((uint16_t)w1) * inv) << 16) |
         (f32_to_e4m3fn_bits(to_f32<T>((uint16_t)(w1 >> 16)) * inv) << 24);
}
// Eight 16-bit values (16 bytes) -> eight e4m3fn bytes.
template <typename T>
__device__ __forceinline__ u32x2 quant8(u32x4 x, float inv) {
  return u32x2{quant4<T>(x[0], x[1], inv), quant4<T>(x[2], x[3], inv)};
}

// round(round(x c) + round(r s)) in the 16-bit type.  The rounded products pass through an empty asm:
// for fp16 the compiler narrows these float ops to native half arithmetic and would otherwise fuse the
// first product into the sum's fma, skipping that product's own rounding.
template <typename T>
__device__ __forceinline__ uint16_t rot1(uint16_t x, uint16_t c, float r, uint16_t s) {
  float a = to_f32<T>(from_f32<T>(to_f32<T>(x) * to_f32<T>(c)));
  float b = to_f32<T>(from_f32<T>(r * to_f32<T>(s)));
  asm volatile("" : "+v"(a), "+v"(b));
  return from_f32<T>(a + b);
}

union Chunk {
  u32x4 v;
  uint16_t e[8];
};

// ---------------------------------------------------------------- 4-bit pools

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

// The scale exponent of the 32 dims that lanes 4 i .. 4 i + 3 hold, eight each.
template <typename T>
__device__ __forceinline__ uint32_t block_exp(u32x4 x) {
  uint32_t m = max_u16x2(max_u16x2(x[0] & 0x7fff7fffu, x[1] & 0x7fff7fffu), max_u16x2(x[2] & 0x7fff7fffu, x[3] & 0x7fff7fffu));
  uint32_t a = max(m & 0xffffu, m >> 16);
  a = max(a, (uint32_t)__shfl_xor((int)a, 1, 64));
  a = max(a, (uint32_t)__shfl_xor((int)a, 2, 64));
  if constexpr (std::is_same<T, BF16>::value)
    return fp4_scale_exp<T>(bf16_bits_to_f32((uint16_t)a));
  else
    return fp4_scale_exp<T>(f16_bits_to_f32((uint16_t)a));
}

struct Fp4Pool {
  char* codes;
  uint8_t* scales;
};

// Byte of `scales` of (slot, head, dim block).
__device__ __forceinline__ int64_t k_scale_at(int64_t slot, int h, int blk, int hkv, int nblk) {
  return (slot * nblk + blk) * hkv + h;
}
__device__ __forceinline__ int64_t v_scale_at(int64_t slot, int h, int blk, int hkv, int nblk, int bs) {
  const int64_t page = slot / bs;
  return ((page * hkv + h) * nblk + blk) * bs + (slot - page * bs);
}

}  // namespace
}  // namespace mllm
