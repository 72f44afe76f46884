// Microscaled 4-bit floating point (OCP MXFP4): the layout the quantisation and the product share.
//
// A row of K values is padded with zeros to Kp = a multiple of MX_GROUP (256) and cut into
// blocks of 32.  A block has one power of two 2^(s - 127), s a byte (255: not a number), and
// 32 e2m1 codes (sign, two exponent bits, one mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6).
//   codes   [rows, Kp / 2]       two codes a byte, the even k in the low nibble
//   scales  [Kp / 256, rows, 8]  the 8 blocks of a row's group side by side, rows next to each
//                                other: the scales of a product tile are one run of memory
// A group of codes is one 128-byte line of its row.
#pragma once

#include "icsa_common.h"

#define MX_BLOCK 32
#define MX_GROUP 256                       // k values of one 128-byte line of codes
#define MX_GROUP_BLOCKS (MX_GROUP / MX_BLOCK)

__host__ __device__ __forceinline__ int mx_padded(int k) { return (k + MX_GROUP - 1) / MX_GROUP * MX_GROUP; }

// Scale byte of a block whose largest magnitude has the f32 bits `amax` (sign bit clear):
// 2^e with e = floor(log2 amax) - 2, so that amax 2^-e lies in [4, 8) (6 is the largest code),
// kept within [-127, 127] (f32 exponents are at most 127, so only below).  Bits from the
// exponent of infinity on: 255.
__device__ __forceinline__ unsigned mx_scale_byte(unsigned amax) {
  const int e = (int)(amax >> 23);
  return e == 255 ? 255u : (unsigned)max(e - 2, 0);
}
// 2^-(s - 127): s is at most 252 where it is not 255, so the factor is a normal number.
__device__ __forceinline__ float mx_inv_scale(unsigned s) { return __uint_as_float((254u - s) << 23); }
// 2^(s - 127); s = 0 is the subnormal 2^-127
__device__ __forceinline__ float mx_scale(unsigned s) {
  return s == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(s == 0 ? 0x00400000u : s << 23);
}

// 8 values, already divided by their block's scale, as 8 codes (round to nearest, ties to the
// even code, magnitudes over 6 to 6)
__device__ __forceinline__ unsigned mx_pack8(const float v[8]) {
  unsigned r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], 1.f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], 1.f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], 1.f, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], 1.f, 3);
  return r;
}
