// The 4-bit cache format: E2M1 values, two a byte (the even dim in the low half),
// with one power of two (E8M0) per token, kv head and 32 dims.
//
// A block's exponent is the smallest e >= -126 with amax <= 7 * 2^e: the largest
// E2M1 value is 6 and its neighbour below 4, so that a value up to 7 is off by half
// a step like any other (with 6 as the limit half of the blocks whose largest
// value lies between 6 and 7 would lose a bit).  A block with an infinity or a NaN
// gets exponent byte 255 (NaN) and zeros.
#pragma once

#include "common.h"
#include "kv_quant.h"

namespace prism {

constexpr int kFp4Block = 32;

// The exponent byte of a block whose largest magnitude has the bits `amax`: its
// own exponent less 2 (6 is 1.5 * 2^2), one more where the mantissa is above 1.75.
__device__ __forceinline__ uint32_t fp4_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = static_cast<int>((bits + 0x1FFFFFu) >> 23) - 2;
  return bits >= 0x7F800000u ? 255u : static_cast<uint32_t>(max(e, 1));
}

// What an exponent byte stands for.
__device__ __forceinline__ float e8m0_value(uint32_t e) {
  return e == 255u ? __uint_as_float(0x7FC00000u) : e == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(e << 23);
}

// Eight values over a power of two -> eight codes, to nearest, ties to the even
// code, magnitudes above 6 to 6 (the native conversion).
__device__ __forceinline__ uint32_t fp4_encode8(const float (&x)[8], uint32_t exponent) {
  if (exponent == 255u) return 0u;
  const float scale = __uint_as_float(exponent << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
  return w;
}

// A row of eight values a lane, a block in each four lanes -> the lane's codes and
// its block's exponent.
__device__ __forceinline__ uint32_t fp4_quantize8(const float (&x)[8], uint32_t& exponent) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = nan_max(amax, fabsf(x[i]));
  amax = group_max<4>(amax);
  exponent = fp4_exponent(amax);
  return fp4_encode8(x, exponent);
}

// Two fp32 values -> two bf16 ones, to nearest even.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float up) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(floatx2{lo, up}, bf16x2));
}

// Eight float16 queries times a power of two -> the sum of two bf16 numbers, exact (11
// bits are in 8 and 3), to meet bf16 keys, which hold every code times every power of
// two.  Infinities and NaN are the first's alone.
__device__ __forceinline__ void split_float16(const u32x4& q, float unit, u32x4& first, u32x4& second) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float lo = f16_bits_to_f32(q[j] & 0xFFFFu) * unit, up = f16_bits_to_f32(q[j] >> 16) * unit;
    first[j] = pack_bf16(lo, up);
    second[j] = pack_bf16(fabsf(lo) < INFINITY ? lo - __uint_as_float(first[j] << 16) : 0.f,
                          fabsf(up) < INFINITY ? up - __uint_as_float(first[j] & 0xFFFF0000u) : 0.f);
  }
}

// Eight codes times a scale.
__device__ __forceinline__ void fp4_decode8(uint32_t w, float scale, float (&x)[8]) {
  const floatx2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0);
  const floatx2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
  const floatx2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2);
  const floatx2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
  x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1], x[4] = c[0], x[5] = c[1], x[6] = d[0], x[7] = d[1];
}

}  // namespace prism
