// Packed fp32 arithmetic: two neighbouring values in one 64-bit register, one instruction for both, each
// rounded as its scalar form is.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace bt {

__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  return (uint64_t)__float_as_uint(hi) << 32 | __float_as_uint(lo);
}
__device__ __forceinline__ float low(uint64_t a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float high(uint64_t a) { return __uint_as_float((uint32_t)(a >> 32)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t sub2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// Two bf16 (the lower half first) as a pair, and back.
__device__ __forceinline__ uint64_t pair_of_bf16(uint32_t w) {
  return (uint64_t)(w & 0xffff0000u) << 32 | (w << 16);
}
__device__ __forceinline__ uint32_t bf16_of_pair(uint64_t a) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(low(a), high(a));
  return *reinterpret_cast<const uint32_t*>(&p);
}

}  // namespace bt
