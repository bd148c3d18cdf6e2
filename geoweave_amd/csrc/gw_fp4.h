// The 4-bit format of a paged cache: e2m1 values (0, 1/2, 1, 3/2, 2, 3, 4, 6 and a sign; two to a byte, the first in the
// low half) with one power of two for each 32 of a row (a biased exponent in a byte, 255: not a number). It is
// the matrix cores' own block format: two values become 16-bit ones by one instruction.
//
// The power of two is the one that brings the largest of the 32 to (3.5, 7]: then no value is off by more than one
// unit, half the widest step (4 to 6; a largest of up to 7 becomes 6). Over normal rows the rms error is 0.112 of
// the rms value; with (4, 8] it is 0.115 and values near 8 are off by two units, with (3, 6] it is 0.117. The power is
// exact and so is the quotient: an element's code does not depend on how a kernel rounds.
#pragma once

#include "gw_common.h"

namespace gw {
namespace {

constexpr uint32_t kFp4NaN = 255u;
constexpr uint32_t kFp4Beyond = 253u;  // the least scale of values that 16 bits have no finite number for: 4 * 2^126 is 2^128

// Of the eight codes of a word: all bits of those whose values, under a scale from kFp4Beyond on, are no finite number: magnitudes from
// 4 on under 2^126, from 2 on under 2^127, all under NaN.
__device__ __forceinline__ uint32_t fp4_beyond(uint32_t w, uint32_t scale) {
  if (scale < kFp4Beyond) return 0u;
  uint32_t hit = 0x11111111u;
  if (scale != kFp4NaN) hit &= scale == kFp4Beyond ? (w >> 1) & (w >> 2) : w >> 2;
  return hit * 15u;
}

// Byte of the power of two for 32 values, from the bits of the largest magnitude (inf and NaN have the largest bits).
__device__ __forceinline__ uint32_t fp4_scale(uint32_t top) {
  if (top >= 0x7f800000u) return kFp4NaN;
  const int e = (int)((top + 0x1FFFFFu) >> 23) - 2;  // one more where the mantissa is above 1.75
  return (uint32_t)(e > 0 ? e : 0);
}
__device__ __forceinline__ float fp4_unit(uint32_t scale) { return __uint_as_float(scale << 23); }  // its exponent is what the conversions read

// Codes of eight values, nearest (of two as near the even code), for a power of two that is a number.
__device__ __forceinline__ uint32_t fp4_pack8(const float* x, uint32_t scale) {
  const float u = fp4_unit(scale);
  uint32_t w = 0u;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], u, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], u, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], u, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], u, 3);
  return w;
}

// Values of the two codes in byte B of w. bf16 holds each exactly (2^128 and above is inf).
template <int B>
__device__ __forceinline__ uint32_t fp4_pair(BF16, uint32_t w, float unit) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, unit, B));
}
template <int B>
__device__ __forceinline__ uint32_t fp4_pair(FP16, uint32_t w, float unit) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, unit, B));
}
// The eight values of a word.
template <typename E>
__device__ __forceinline__ uint4 fp4_operand(uint32_t w, float unit) {
  return make_uint4(fp4_pair<0>(E{}, w, unit), fp4_pair<1>(E{}, w, unit), fp4_pair<2>(E{}, w, unit), fp4_pair<3>(E{}, w, unit));
}

}  // namespace
}  // namespace gw
