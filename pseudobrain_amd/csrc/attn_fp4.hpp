// The 4-bit cache's format (gfx950): 32 consecutive values of a head share a scale,
// a power of two; each is one of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} of it.
//
// Largest |x| of the 32 rounds to 2^e or 1.5 2^e by its two leading mantissa bits;
// the scale is 2^(e - 2), so that it becomes 4 or 6 of them (1.75 2^e and more would
// round to 8, half a step past the largest: the scale is doubled, and no value is off
// by more than half of its step). The byte is the scale's float32 exponent, 2 to 252:
// with it every value that a code stands for is a normal float32 and bfloat16 number.
// 255 stands for 32 values among which one is infinite or NaN.
//
// Conversions are the hardware's (a scale enters by its exponent bits): they round to
// nearest, ties to the even code, and saturate; both directions are exact otherwise,
// and scale 255 gives NaN.
#pragma once

#include "attn_tile.hpp"

namespace pbgdn {

constexpr int FP4_BLOCK = 32;  // values that share a scale
constexpr uint32_t FP4_MIN_SCALE = 2, FP4_MAX_SCALE = 252, FP4_NAN_SCALE = 255;

// The scale byte of 32 values whose largest magnitude has these bits (0x7f800000 and
// above where one is not finite).
__device__ __forceinline__ uint32_t fp4_scale_of(uint32_t top) {
  const int e = static_cast<int>((top + 0x200000u) >> 23) - 2;
  const uint32_t s = e < static_cast<int>(FP4_MIN_SCALE) ? FP4_MIN_SCALE
                     : e > static_cast<int>(FP4_MAX_SCALE) ? FP4_MAX_SCALE : static_cast<uint32_t>(e);
  return top >= 0x7f800000u ? FP4_NAN_SCALE : s;
}
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Eight values as a word of codes, the first in its lowest bits.
__device__ __forceinline__ uint32_t fp4_pack8(const float *x, float scale) {
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
  return w;
}
// Values 2 BYTE and 2 BYTE + 1 of a word as a pair of bfloat16 (which holds them exactly).
template <int BYTE>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, BYTE));
}
// Eight values of a word as four such pairs: an operand of the 16-bit matrix products.
__device__ __forceinline__ v4u32_t fp4_unpack8(uint32_t w, float scale) {
  return v4u32_t{fp4_pair<0>(w, scale), fp4_pair<1>(w, scale), fp4_pair<2>(w, scale), fp4_pair<3>(w, scale)};
}

}  // namespace pbgdn
