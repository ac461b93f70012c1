// Rows in 8 bits: e4m3 values with one power-of-two scale (e8m0) for each block of 128 consecutive elements of a row.
//
// The scale of a block is the least 2^e, e >= -126, with max |x| <= 448 * 2^e (448: the largest e4m3).  x / 2^e is exact in
// fp32 apart from numbers far below the block's largest, so the one rounding is that to e4m3, to the nearest, ties to even; no
// value reaches past 448.  A block that holds an infinity or NaN has a NaN for its scale and for all its values.
#pragma once

#include "ccq_tile.h"

namespace ccq {

constexpr int kFp8Block = 128;
constexpr unsigned kFp8Nan = 255;  // the scale's byte e + 127; this one is its NaN

// |x| as bits: the maximum of such words passes on infinities and NaN, which fmaxf does not
__device__ __forceinline__ unsigned magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// byte of the scale of a block whose largest magnitude is m: 448 is 1.75 * 2^8, so a significand above 1.75 carries
__device__ __forceinline__ unsigned scale_byte(unsigned m) {
  const int e = (int)((m + 0x1fffffu) >> 23) - 8;
  return m >= 0x7f800000u ? kFp8Nan : (unsigned)max(e, 1);
}
// 1 / scale, of a byte in 1 .. 247 (the NaN's is not used)
__device__ __forceinline__ float scale_inverse(unsigned byte) { return __uint_as_float((254u - (byte & 0xffu)) << 23); }

// four values of a block as a word of e4m3
__device__ __forceinline__ unsigned fp8_word(float a, float b, float c, float d, unsigned byte) {
  const float s = scale_inverse(byte);
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * s, b * s, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c * s, d * s, w, true);
  return byte == kFp8Nan ? 0x7f7f7f7fu : (unsigned)w;
}

// maximum over 16 consecutive lanes, by rotations within them
__device__ __forceinline__ unsigned lanes_max16(unsigned x) {
  x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, true));  // row_ror:8, 4, 2, 1
  x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, true));
  x = max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, true));
  return max(x, (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, true));
}
// over groups of L consecutive lanes (L a power of two <= 64)
__device__ __forceinline__ unsigned lanes_max(unsigned x, int L) {
  if (L >= 16) {
    x = lanes_max16(x);
    for (int o = 16; o < L; o <<= 1) x = max(x, (unsigned)__shfl_xor((int)x, o));
    return x;
  }
  for (int o = L >> 1; o > 0; o >>= 1) x = max(x, (unsigned)__shfl_xor((int)x, o));
  return x;
}

}  // namespace ccq
