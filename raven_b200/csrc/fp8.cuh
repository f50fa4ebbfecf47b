// Rounding a block of 128 values to FP8 (include/raven_gpu.h, raven_fp8_encode_device).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

namespace raven_fp8 {

__device__ inline float load_value(const float* p) { return *p; }
__device__ inline float load_value(const __half* p) { return __half2float(*p); }
__device__ inline float load_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// The least e >= -127 with `top` <= 448 * 2^e, for a finite magnitude given as
// bits; 0 for zero. 448 = 1.75 * 2^8: one exponent more when the mantissa is above 1.75.
__device__ inline int exponent_of(uint32_t top) {
  const int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return top == 0 ? 0 : max(e, -127);
}
// 2^-e
__device__ inline float inverse_of(int e) {
  return e == -127 ? 1.7014118346046923e38f : __uint_as_float((uint32_t)(127 - e) << 23);
}
__device__ inline bool odd_value(float x) { return (__float_as_uint(x) & 0x7fffffffu) >= 0x7f800000u; }  // infinite or NaN
// Four codes, the first lowest, rounded to nearest even.
__device__ inline uint32_t codes_of(const float* x, float inv) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0] * inv, x[1] * inv), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2] * inv, x[3] * inv), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// The same with the NaN code for what is not finite (the conversion saturates infinities).
__device__ inline uint32_t with_nan(uint32_t w, const float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (odd_value(x[i])) w = (w & ~(0xffu << (8 * i))) | (0x7fu << (8 * i));
  return w;
}

}  // namespace raven_fp8
