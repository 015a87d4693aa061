// MXFP4 helpers shared by its kernels: the place of a scale, the scale of a block, E2M1 conversion.
#pragma once

#include "common.cuh"

namespace b2 {
namespace mx4 {

constexpr int kBlk = 32;  // columns per scale

// Byte of the scale of (row, block of 32 columns) in the tiled scale array (see b2_mx4_args).
__host__ __device__ __forceinline__ int64_t scale_at(int64_t row, int64_t blk, int64_t nkb) {
  return ((row >> 7) * nkb + (blk >> 2)) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4 + (blk & 3);
}

// The E8M0 code of a block, from the largest of its elements' bits without the sign (NaN and infinity are the largest):
// 2^(floor(log2 amax) - 2) is the fp32 exponent field less two; a block with an infinity or a NaN gets the NaN scale.
__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t scale_code(uint32_t top) {
  return top >= 0x7f800000u ? 255u : (uint32_t)max((int)(top >> 23) - 2, 0);
}
// 2^(127 - code), by which the elements are divided (exactly).
__device__ __forceinline__ float inverse_scale(uint32_t code) {
  return code == 255u ? 0.f : __uint_as_float((254u - code) << 23);
}
__device__ __forceinline__ float e8m0_to_f32(uint32_t code) {
  if (code == 255u) return __uint_as_float(0x7FC00000u);
  return code ? __uint_as_float(code << 23) : __uint_as_float(0x00400000u);  // code 0: 2^-127
}

// Eight floats -> eight E2M1 codes, element 0 in the lowest nibble.
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// Eight codes -> four half2 (exact: every E2M1 value is a half).
__device__ __forceinline__ void e2m1x8_to_half2(uint32_t c, __half2* h) {
  uint32_t o[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(c));
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = *reinterpret_cast<__half2*>(&o[i]);
}

}  // namespace mx4
}  // namespace b2
