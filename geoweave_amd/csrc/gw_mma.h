// Pieces shared by the matrix-core passes: the 32x32x16 products, the XOR swizzle of 64-row LDS
// tiles, lane-pair exchanges, and fp16/bf16 packing.
#pragma once

#include <math.h>

#include "gw_common.h"

namespace gw {
namespace {

constexpr float kDLog2e = 1.4426950408889634f;
constexpr float kDLn2 = 0.6931471805599453f;

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// D = A B + C for a 32x32 tile with a k-step of 16. Lane l supplies A[l % 32][8 (l / 32) + i]
// and B[8 (l / 32) + i][l % 32] (i < 8, one 16-byte register quad each); accumulator entry r
// of lane l is D[8 (r / 4) + 4 (l / 32) + r % 4][l % 32].
__device__ __forceinline__ f32x16 mma(BF16, uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                 __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(FP16, uint4 a, uint4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// Keeps the compiler from moving LDS accesses across this point; within one wave the LDS
// performs them in issue order, so no barrier is needed between a wave's own write and read.
__device__ __forceinline__ void lds_fence() { asm volatile("" ::: "memory"); }

__device__ __forceinline__ uint16_t to_half_bits(BF16, float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
__device__ __forceinline__ uint16_t to_half_bits(FP16, float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }

typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_v __attribute__((ext_vector_type(2)));
// Two floats to two 16-bit floats of the tag's type, round to nearest even, in one word
// (v_cvt_pk_f16_f32 / v_cvt_pk_bf16_f32).
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, f16x2_v));
}
__device__ __forceinline__ uint32_t pack_pair(FP16, float a, float b) { return pack_f16(a, b); }
__device__ __forceinline__ uint32_t pack_pair(BF16, float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){a, b}, bf16x2_v));
}
// Eight consecutive floats as one 16-byte operand quad.
template <typename E>
__device__ __forceinline__ uint4 pack_quad(const float* v) {
  return make_uint4(pack_pair(E{}, v[0], v[1]), pack_pair(E{}, v[2], v[3]), pack_pair(E{}, v[4], v[5]),
                    pack_pair(E{}, v[6], v[7]));
}

// 0 where sel is all ones, neg where it is zero (v_bfi_b32: (sel & 0) | (~sel & neg)).
__device__ __forceinline__ float select_bias(int sel, float neg) {
  float r;
  asm("v_bfi_b32 %0, %1, 0, %2" : "=v"(r) : "v"(sel), "v"(neg));
  return r;
}
// Lanes l and l ^ 32 exchange (v_permlane32_swap); both get op(own, partner).
__device__ __forceinline__ float pair_max(float x) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}

// LDS tiles of 64 rows of 128 bytes: the 16-byte chunk c of row R sits at c ^ swz(R). Operand
// reads (consecutive rows, one chunk) and tile stores (8 lanes per row) then touch distinct
// banks in every group of 8 and of 16 lanes.
__device__ __forceinline__ int swz(int R) { return (R & 7) ^ ((R >> 3) & 1); }

__device__ __forceinline__ float in_to_float(int in_fp16, uint32_t u) {
  return in_fp16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)u) : __uint_as_float(u << 16);
}

// Non-zero when either 16-bit half of w has its exponent field e all ones (inf or nan).
__device__ __forceinline__ uint32_t nonfinite2(uint32_t w, uint32_t e) {
  return (uint32_t)((w & e) == e) | (uint32_t)(((w >> 16) & e) == e);
}

// 32x32 bit-matrix transpose across the lanes of each half-wave: lane i holds row i (bit c =
// element (i, c)); afterwards lane c holds column c (bit i = element (i, c)). Five rounds of
// exchanging bit blocks with the lane 16, 8, 4, 2, 1 apart.
__device__ __forceinline__ uint32_t lane_bit_transpose32(uint32_t x, int lane) {
  const uint32_t masks[5] = {0x0000FFFFu, 0x00FF00FFu, 0x0F0F0F0Fu, 0x33333333u, 0x55555555u};
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    const int j = 16 >> i;
    const uint32_t m = masks[i];
    const uint32_t y = (uint32_t)__shfl_xor((int)x, j);
    x = (lane & j) ? ((x & ~m) | ((y >> j) & m)) : ((x & m) | ((y << j) & ~m));
  }
  return x;
}

}  // namespace
}  // namespace gw
