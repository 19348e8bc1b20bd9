// Device helpers of the 4-bit cache: E2M1 codes with a power-of-two scale (E8M0 byte) for 32
// channels, by the conversion instructions of gfx950.
#pragma once
#include "ci8_device.h"

namespace ci8 {

constexpr int kFp4Block = 32;  // channels that share a scale

// Scale operand of the conversions: the E8M0 byte as an FP32 exponent. 255 converts to NaN.
__device__ __forceinline__ float fp4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// The same for byte i of a word of scales: the word turned so that the byte is the exponent, one
// instruction. The conversion to BF16 reads nothing else of it (65536 random words gave what their
// exponents alone do).
__device__ __forceinline__ uint32_t fp4_scale_turn(uint32_t i) { return (8 * i + 9) & 31; }
__device__ __forceinline__ float fp4_scale_in(uint32_t word, uint32_t turn) {
  return __uint_as_float(__builtin_amdgcn_alignbit(word, word, turn));
}

// Eight codes (channel 0 in the lowest bits) times the scale, in BF16: exact, since a code has
// two significant bits.
__device__ __forceinline__ u32x4 fp4_to_bf16x8(uint32_t codes, float scale) {
  return u32x4{
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3))};
}

// E8M0 byte of a block whose largest |x| has the bits amax: 127 + e for the smallest e with
// amax <= 7 * 2^e, held in -125 .. 125, 255 for an infinity or NaN. With amax = m * 2^E, 1 <= m
// < 2, e is E - 2 up to m = 1.75 and E - 1 beyond: adding 0x1FFFFF carries into the exponent
// exactly when the fraction passes 0x600000. e >= -125 keeps half a unit a normal BF16 number,
// e <= 125 keeps 4 units finite.
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t amax) {
  const uint32_t exponent = (amax + 0x1FFFFFu) >> 23;
  const uint32_t byte = min(max(exponent, 4u) - 2, 252u);
  return amax >= 0x7F800000u ? 255 : byte;
}

// Eight values as codes for that scale: nearest, ties to the even code, at most 6.
__device__ __forceinline__ uint32_t fp4_codes8(const float (&x)[8], uint32_t scale_byte) {
  const float s = fp4_scale(scale_byte);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], s, 3);
  return scale_byte == 255 ? 0 : c;
}

}  // namespace ci8
