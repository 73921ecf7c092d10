// The 8-bit KV cache's number format, shared by the kernels that write, read and attend it.
//
// A pool element is an e4m3 code c and stands for c * s, with one fp32 scale s for each
// (layer, block, KV head) of K and of V. Scales are powers of two: e4m3 is a floating
// format, so the mantissa of a scale buys no precision, while a power of two makes
// x / s exact (codes are rounded once), makes the change of a block's scale a shift of
// exponents (older codes are only rounded where they fall below the normal range, 2^-6),
// and lets the attention kernels move s between factors without a rounding.
#pragma once

#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace b2p {

// Smallest block exponent. Blocks of smaller values (all-zero ones among them) use it: 448 *
// 2^-110 is still a normal fp32 number and so are the products with it.
constexpr int kFp8MinExp = -110;

// The exponent e of a block's scale 2^e: the smallest e >= kFp8MinExp with amax <= 448 * 2^e.
// 448 = 1.75 * 2^8, so e is amax's own exponent less 8, plus one where its mantissa is above
// 1.75. amax must be finite and not negative.
__device__ __forceinline__ int fp8_block_exp(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < kFp8MinExp ? kFp8MinExp : e;
}

__device__ __forceinline__ float exp2_int(int e) {  // 2^e for -126 <= e <= 127
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// The largest magnitude a value may round to in 4 significant bits without leaving fp32
// (fp32 and bf16 rows above it, the last 6 % below 2^128, are stored as this value).
constexpr float kFp8Saturate = 0x1.ep127f;

// x * inv (inv = 2^-e of the value's block, |x * inv| <= 448) as an e4m3 code, ties to even.
__device__ __forceinline__ uint8_t fp8_code(float x, float inv) {
  return (uint8_t)__nv_cvt_float_to_fp8(fminf(fmaxf(x, -kFp8Saturate), kFp8Saturate) * inv,
                                        __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float fp8_value(uint8_t code) {  // without its scale
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3)));
}

// Two codes (bits 0..7 and 8..15 of `two`) as a pair of f16 values, exactly (NaN stays NaN).
__device__ __forceinline__ uint32_t fp8x2_to_f16x2(uint16_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(two));
  return r;
}

// Two values of the cache (codes times scales, or means of them) as a pair of T. f16 rows from 63,488 up are stored as
// 65,536 (half a step of their code up), which is past f16's largest finite value: 65,504 stands
// for it, and for everything above it in a pool that other types' rows went into. NaN stays NaN.
template <typename T>
__device__ __forceinline__ uint32_t pack_values(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  } else {
    return pack2<T>(lo, hi);
  }
}

template <typename T>
__device__ __forceinline__ T value_as(float x) {  // the same for one value
  return std::is_same<T, __half>::value ? from_f32<T>(x > 65504.f ? 65504.f : x < -65504.f ? -65504.f : x)
                                        : from_f32<T>(x);
}

}  // namespace b2p
