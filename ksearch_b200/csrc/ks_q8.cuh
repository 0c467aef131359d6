// Device helpers of the paged 8-bit cache: codes of one byte (int8, or e4m3 floats: sign, 4 exponent bits, 3 mantissa bits, bias 7) and
// their scales.  Every code is a number of f16 (int8 exactly, e4m3's 2^-9 .. 448 too), so products of codes can run on f16 tensor cores.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

namespace {

__device__ __forceinline__ uint32_t q8_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 q8_h2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

__device__ __forceinline__ float q8_warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Two codes in the low halfword, from values that are over their scale already: nearest, ties to even, the largest code beyond it.
// (NaN has been replaced.)
template <bool FP8>
__device__ __forceinline__ uint32_t q8_encode2(float a, float b) {
  if constexpr (FP8) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
  } else {
    const int x = __float2int_rn(fminf(fmaxf(a, -127.0f), 127.0f)), y = __float2int_rn(fminf(fmaxf(b, -127.0f), 127.0f));
    return ((uint32_t)x & 0xFFu) | ((uint32_t)y & 0xFFu) << 8;
  }
}
// The low two bytes' codes as f16.  e4m3's NaN patterns come out as 448: no code of a cache is NaN, so 0 times a masked one stays 0.
template <bool FP8>
__device__ __forceinline__ __half2 q8_decode2h(uint32_t w) {
  if constexpr (FP8) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((unsigned short)w));
    return __hmin2(q8_h2(r), __float2half2_rn(448.0f));
  } else {
    // 1024 + (code + 128) has the biased code in its low mantissa bits
    return __hsub2(q8_h2(__byte_perm(w ^ 0x8080u, 0x64646464u, 0x4140)), __float2half2_rn(1152.0f));
  }
}
template <bool FP8>
__device__ __forceinline__ float2 q8_decode2f(uint32_t w) {
  return __half22float2(q8_decode2h<FP8>(w));
}

// Scales are used inside 2^-100 .. 2^100: their reciprocals and logarithms are finite then (NaN and what is not positive count as 2^-100).
__device__ __forceinline__ float q8_scale(float s) { return fminf(fmaxf(s, 0x1p-100f), 0x1p100f); }
// The least power of two 2^e, e >= -100, with amax <= qmax 2^e: 127 = 1.984375 x 2^6, 448 = 1.75 x 2^8.
template <bool FP8>
__device__ __forceinline__ float q8_scale_for(float amax) {
  const uint32_t b = __float_as_uint(amax), top = FP8 ? 0x600000u : 0x7E0000u;
  int e = (int)(b >> 23) - 127 - (FP8 ? 8 : 6) + ((b & 0x7FFFFFu) > top ? 1 : 0);
  e = min(max(e, -100), 100);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
// The least power of two that s (0, or inside the range above) does not exceed.
__device__ __forceinline__ float q8_power_above(float s) {
  const uint32_t b = __float_as_uint(s);
  return fminf(__uint_as_float((b & 0x7FFFFFu) ? (b & 0x7F800000u) + 0x800000u : b), 0x1p100f);
}

}  // namespace
