// The 4-bit K/V cache (gfx950): its layout and the conversions to and from it.
//
// A head's row of 128 channels is four groups of 32 channels, each 4-bit floats (a sign and one of
// 0 .5 1 1.5 2 3 4 6) times a power of two: the number format of CDNA4's scaled MFMAs and of its
// 4-bit converters: the importance feeds K to the matrix cores as stored, the attention converts two values
// an instruction to bf16, exactly. 4.25 bits per value.
//
// Cell = 16 consecutive slots of one K/V head, kCellBytes bytes; the cells of a slot group's heads lie
// side by side: cache[slot / 16][kv_head][kCellBytes]. In a cell, slot s (0..15):
//   K codes   byte 64 s + c / 2, channel c in its low (even c) or high half
//   V codes   kCellV + 256 (s / 4) + 16 w + 4 (s % 4): the 4-byte word of channels 8 w .. 8 w + 7
//   K scales  kCellKs + 16 (c / 32) + s: byte b stands for 2^(b - 127), 255 for NaN
//   V scales  kCellVs + 16 (c / 32) + s
// A 16-byte load of V brings four keys' words of the same channels: the operand of P V holds several
// keys of one channel per lane, and a row is still written in whole words of its own.
#pragma once

#include "fdl_device.h"

namespace fdl {

constexpr int kCellSlots = 16;
constexpr int kCellV = 1024, kCellKs = 2048, kCellVs = 2112;
constexpr int kCellBytes = 2176;
constexpr int kKv4HeadDim = 128;

// Scale byte of a group whose largest magnitude is `top`: the smallest e with top <= 7 * 2^e (a
// cut-off at 6 then costs at most the 1 * 2^e that rounding between 4 and 6 costs), clamped to
// [-127, 125], where 6 * 2^125 is still finite; 255 for a NaN or infinite top.
__device__ __forceinline__ uint32_t kv4_scale_byte(float top) {
  const uint32_t b = __float_as_uint(top);
  const int expo = static_cast<int>(b >> 23);               // top >= 0
  if (expo == 255) return 255;
  const int e = expo - ((b & 0x7fffffu) <= 0x600000u ? 2 : 1);  // biased by 127
  return static_cast<uint32_t>(min(max(e, 0), 252));
}

// Codes of 8 channels with scale byte `b`, channel i in bits 4 i .. 4 i + 3: round to nearest, ties to
// the even code, cut off at 6. A NaN group's codes are 0.
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], uint32_t b) {
  const float scale = __uint_as_float(b << 23);
  uint32_t w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
  return b == 255 ? 0u : w;
}

// Channels 2 i and 2 i + 1 of a word as two bf16 (exact: a code has two significant bits), times the
// scale whose byte is bits 23..30 of `scale` (255: NaN).
template <int i>
__device__ __forceinline__ uint32_t kv4_bf16x2(uint32_t word, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, i));
}

}  // namespace fdl
