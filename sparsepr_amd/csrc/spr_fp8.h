// The 8-bit format of the projections: e4m3 codes (a sign, four bits of exponent, three of fraction,
// 448 at most) and one scale byte b, 2^(b - 127), for a group of 128 values of a row or of 128 x 128.
// A power of two, since the scaled matrix instruction takes it as an operand: the products need no
// arithmetic between two blocks, and scaling a value to its code is exact but for the one rounding.
#pragma once

#include "spr_elem.h"

namespace spr {

constexpr int FP8_GROUP = 128;
constexpr uint32_t FP8_NAN_SCALE = 255;

// The scale byte of a group from the bits of its largest magnitude (bits order as magnitudes do, with
// infinities and NaNs on top): the smallest power of two e with magnitude <= 448 e = 1.75 * 2^8 e, so
// the fraction's part above .75 carries into the exponent.  2^-126 at least, so that its inverse is
// a normal number too; NaN where the group has an infinity or a NaN.
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t top) {
  if (top >= 0x7f800000u) return FP8_NAN_SCALE;
  const int b = static_cast<int>((top + 0x1FFFFFu) >> 23) - 8;
  return static_cast<uint32_t>(b < 1 ? 1 : b);
}
// 2^(127 - b): what values are multiplied by (0 for a NaN group, whose codes do not matter)
__device__ __forceinline__ float fp8_inverse_scale(uint32_t b) {
  return b == FP8_NAN_SCALE ? 0.0f : __uint_as_float((254u - b) << 23);
}
// 2^(b - 127); byte 0 is 2^-127, a subnormal
__device__ __forceinline__ float fp8_scale(uint32_t b) {
  return b == FP8_NAN_SCALE ? __uint_as_float(0x7fc00000u) : __uint_as_float(b == 0 ? 0x00400000u : b << 23);
}

__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t magnitude_bits8(const float (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, magnitude_bits(x[e]));
  return m;
}

// Eight values times `inv` as codes, to nearest even.  (inf * 0 of a NaN group gives NaN codes there.)
__device__ __forceinline__ uint64_t fp8_codes8(const float (&x)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    int32_t c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, 0, false);
    w[i] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, c, true));
  }
  return w[0] | (static_cast<uint64_t>(w[1]) << 32);
}

__host__ __device__ __forceinline__ int64_t fp8_width(int64_t n) { return (n + 15) & ~int64_t(15); }
__host__ __device__ __forceinline__ int64_t fp8_groups(int64_t n) { return (n + FP8_GROUP - 1) / FP8_GROUP; }

}  // namespace spr
