// act8.cuh — activations in 8 bits: 32 values share a scale 2^e and are e4m3 codes of x 2^-e.
//
// e is the least integer >= -126 for which the largest finite |x| of the block is at most 448 2^e, so no value
// saturates, scaling is exact and the only error is the code's own rounding (half a step, 2^-4 of a normal value;
// values below 2^-6 2^e are rounded to multiples of 2^-9 2^e). A value that is not finite becomes NaN. Stored: a byte a
// value, and e + 127 in a byte a block.
#pragma once
#include <cuda_fp8.h>
#include <stdint.h>

namespace bd {

constexpr int kAct8Block = 32;

__device__ __forceinline__ float act8_size(float x) {  // |x|, 0 where x is not finite
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}

__device__ __forceinline__ int act8_exponent(float largest) {
  const uint32_t bits = __float_as_uint(largest);
  // largest = 1.m 2^k <= 1.75 2^(8 + e)
  return max((int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0), -126);
}

__device__ __forceinline__ float act8_power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Two codes (x in the low byte). `inverse` is 2^-e.
__device__ __forceinline__ uint32_t act8_code2(float x, float y, float inverse) {
  const float nan = __int_as_float(0x7FC00000);
  float2 v;
  v.x = fabsf(x) <= 3.402823466e38f ? x * inverse : nan;
  v.y = fabsf(y) <= 3.402823466e38f ? y * inverse : nan;
  return __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ uint32_t act8_code4(const float* x, float inverse) {
  return act8_code2(x[0], x[1], inverse) | (act8_code2(x[2], x[3], inverse) << 16);
}

// What two codes stand for. Rounding up may carry the largest values past a type's range: they stand for its limit.
__device__ __forceinline__ float2 act8_value2(uint32_t codes, float scale, float limit) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
  float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
  v.x *= scale, v.y *= scale;
  if (fabsf(v.x) > limit) v.x = copysignf(limit, v.x);
  if (fabsf(v.y) > limit) v.y = copysignf(limit, v.y);
  return v;
}

constexpr float kAct8LimitF32 = 3.402823466e38f, kAct8LimitBF16 = 3.3895313892515355e38f, kAct8LimitF16 = 65504.f;

}  // namespace bd
