// The 8-bit form of a cached key or value row (the d values of one sequence, head and
// position), shared by the kernels that write it and those that read it.
//
// A row is d e4m3 codes and one power of two 2^e, the least e >= -127 with
// max|row| <= 448 * 2^e (448 = largest e4m3 value), kept as one byte e + 127 (E8M0).
// A power of two because scaling by it is exact: a value is rounded once, when its
// code is made, and code * 2^e has at most four significant bits, so reading the row
// back as bf16 rounds nothing and every reader sees the same numbers.  (Where bf16 has them: with e
// of -125 to -127 the smallest codes stand for less than its smallest step, 2^-133, and are rounded to it, and
// a code of 256 or more under 2^120, which the writer does not make, is infinite.)  A free fp32
// scale would use the last half binade below 448 too, but e4m3 is a floating type:
// its relative step is the same there, only values 2^-15 below the largest gain.
// (A row with values above 1.9375 * 2^127 stops at code 240: 256 would stand for 2^128.)
// Byte 255 is E8M0's NaN: a row that holds an infinity or a NaN reads back as NaN.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "sb_common.cuh"

namespace sb {

constexpr uint32_t kScaleNan = 255;
constexpr uint32_t kScaleTop = 247;      // 2^120, the largest that a finite row has
constexpr float kCodeTop = 240.f;        // the largest code value that stands for a float under it

// byte -> 2^(byte - 127); 0 is the fp32 subnormal 2^-127, 255 NaN
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == kScaleNan ? 0x7fc00000u : byte << 23);
}

// The scale byte of a row whose largest magnitude has these fp32 bits:
// 1.m * 2^(x-127) <= 448 * 2^e = 1.75 * 2^(e+8)  <=>  e + 127 >= x - 8 (+ 1 where 1.m > 1.75).
__device__ __forceinline__ uint32_t e8m0_of_amax(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return kScaleNan;
  const int byte = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return byte < 0 ? 0u : (uint32_t)byte;
}

// 2^-(byte - 127), by which a row is multiplied before its values become codes (0 for a NaN row)
__device__ __forceinline__ float e8m0_inverse(uint32_t byte) {
  return byte == kScaleNan ? 0.f : __uint_as_float((254u - byte) << 23);
}

// four fp32 values -> four e4m3 codes (nearest, ties to even), the first in the low byte
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// two e4m3 codes (the low 16 bits) -> two fp16 values, exact
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ float2 f16x2_to_float2(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

}  // namespace sb
