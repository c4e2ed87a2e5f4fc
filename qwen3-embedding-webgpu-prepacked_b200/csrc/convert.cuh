// Conversions between the stored types (f16, bf16, E4M3, INT8) and f32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace qwa {

__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __half from_float<__half>(float x) {
  return __float2half_rn(x);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// Two 16-bit values of a register <-> f32.
template <bool kBf16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (kBf16)  // a bf16 is the upper half of an f32
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (kBf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two E4M3 codes (low byte first) -> f16x2, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(codes)));
  return r;
}
// f32 pair -> two E4M3 codes, round to nearest even, saturating; NaN stays NaN.
__device__ __forceinline__ uint32_t float2_to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t half2_to_e4m3x2(uint32_t pair) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(pair));
  return r;
}
// 2^e for -126 <= e <= 127 (0 for -127, infinity for 128).
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((e + 127) << 23); }


// 2^e as two equal 16-bit values. f16: 0 below 2^-24, infinity above 2^15.
template <bool kBf16>
__device__ __forceinline__ uint32_t pair_pow2(int e) {
  uint32_t h;
  if constexpr (kBf16) {
    h = static_cast<uint32_t>(e + 127) << 7;
  } else {
    if (e > 15) h = 0x7c00u;
    else if (e >= -14) h = static_cast<uint32_t>(e + 15) << 10;
    else if (e >= -24) h = 1u << (e + 24);
    else h = 0u;
  }
  return h | (h << 16);
}

// Two 8-bit codes (the low 16 bits) -> the pair of 16-bit values code * 2^e,
// scale2 = pair_pow2(e). Exact for what the cache's rule writes: a code has at most
// 7 significant bits, and e keeps code * 2^e in range.
template <bool kBf16, bool kE4M3>
__device__ __forceinline__ uint32_t code_pair(uint32_t codes, uint32_t scale2) {
  uint32_t h;
  if constexpr (kE4M3) {
    h = e4m3x2_to_half2(codes);
  } else {
    // 1024 + (code + 128) has the code's bits in an f16's low byte
    const uint32_t u = __byte_perm(codes ^ 0x8080u, 0x64646464u, 0x4140);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u),
                              __floats2half2_rn(1152.f, 1152.f));
    h = *reinterpret_cast<const uint32_t*>(&v);
  }
  if constexpr (kBf16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    const uint32_t b = pack2<true>(f.x, f.y);
    const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&b),
                                     *reinterpret_cast<const __nv_bfloat162*>(&scale2));
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&h),
                              *reinterpret_cast<const __half2*>(&scale2));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

}  // namespace qwa
