// 8-bit floats (e4m3) with power-of-two scales, as the 8-bit cache holds them.
//
// A page's scale is 2^e, -15 <= e <= 7, the least that brings the page's largest
// absolute value under the type's 448. A power of two moves a value without
// rounding it (but for those that become subnormal), so the mantissa's three bits
// are all the cache loses, a page can move to a larger scale when larger tokens
// join it, and the bounds make every stored value an f16 and a bf16 number exactly:
// 448 * 2^7 = 57344 is below f16's largest, 2^-9 * 2^-15 its smallest.
#pragma once

#include <cuda_fp8.h>

#include "cvsa_common.cuh"

namespace cvsa {

constexpr int kScaleMin = -15, kScaleMax = 7;

// Four codes (low byte first) as f16, two a word; exact.
__device__ __forceinline__ void e4m3x4_to_f16x4(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}
// Four codes as floats; exact.
__device__ __forceinline__ void e4m3x4_to_f4(uint32_t four, float* f) {
  uint32_t lo, hi;
  e4m3x4_to_f16x4(four, lo, hi);
  f16x2_to_f2(lo, f[0], f[1]);
  f16x2_to_f2(hi, f[2], f[3]);
}
// Four floats as codes: nearest, halves to even, beyond 448 saturated, NaN kept.
__device__ __forceinline__ uint32_t f4_to_e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126..127

// The exponent of a page's scale for largest absolute value `amax` (finite, >= 0):
// the least e with amax <= 1.75 * 2^(8 + e), in the scale's range.
__device__ __forceinline__ int scale_exponent(float amax) {
  const int bits = __float_as_int(amax);
  const int e = (bits >> 23) - 127 - ((bits & 0x7fffff) > 0x600000 ? 7 : 8);
  return max(kScaleMin, min(kScaleMax, e));
}
// The exponent that a stored scale stands for, in range whatever the word holds.
__device__ __forceinline__ int scale_exponent_of(float scale) {
  const int e = ((__float_as_int(scale) >> 23) & 0xff) - 127;
  return max(kScaleMin, min(kScaleMax, e));
}

// A page's factor as two f16, for widen16, from its scale.
__device__ __forceinline__ uint32_t widen_factor(float scale) {
  const uint32_t h = __half_as_ushort(__float2half_rn(pow2(scale_exponent_of(scale))));  // exact
  return h | h << 16;
}

// Whether one of 16 codes is NaN.
__device__ __forceinline__ bool any_nan8(const uint4& c) {
  auto top = [](uint32_t w) { return (w & 0x7f7f7f7fu) + 0x01010101u; };
  return ((top(c.x) | top(c.y) | top(c.z) | top(c.w)) & 0x80808080u) != 0;
}

// 16 codes times their page's factor, as f16; exact.
__device__ __forceinline__ void widen16(const uint4& codes, uint32_t factor, uint4* out) {
  const uint32_t* c = reinterpret_cast<const uint32_t*>(&codes);
  uint32_t* o = reinterpret_cast<uint32_t*>(out);
  const __half2 f = *reinterpret_cast<const __half2*>(&factor);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t two[2];
    e4m3x4_to_f16x4(c[i], two[0], two[1]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&two[j]), f);
      o[2 * i + j] = *reinterpret_cast<const uint32_t*>(&x);
    }
  }
}

}  // namespace cvsa
