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

// Rows may start at any element: vectors of the element's alignment (global memory takes them)
typedef bf16x8 bf16x8_a2 __attribute__((aligned(2)));
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef bf16x4 bf16x4_a2 __attribute__((aligned(2)));
typedef floatx4 floatx4_a4 __attribute__((aligned(4)));

// 8 values of a row from k on, zeros from K on; where K cuts them, value by value, so that nothing past the
// row is touched.
template <typename T>
__device__ __forceinline__ void load8_row(const T* row, int k, int K, float v[8]) {
  if (k + 8 <= K) {
    if constexpr (sizeof(T) == 2) {
      const bf16x8 x = *reinterpret_cast<const bf16x8_a2*>(row + k);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
    } else {
      const floatx4 a = *reinterpret_cast<const floatx4_a4*>(row + k), b = *reinterpret_cast<const floatx4_a4*>(row + k + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = k + i < K ? (float)row[k + i] : 0.f;
}

// Scale byte of a block whose 32 values four neighbouring lanes hold, 8 each; the magnitudes are
// compared as f32 bit patterns without their sign, where NaN and infinity come out on top.
__device__ __forceinline__ unsigned mx_quantize8(const float v[8]) {
  unsigned amax = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = max(amax, __float_as_uint(v[e]) & 0x7fffffffu);
  amax = max(amax, (unsigned)__shfl_xor((int)amax, 1, 64));
  amax = max(amax, (unsigned)__shfl_xor((int)amax, 2, 64));
  return mx_scale_byte(amax);
}
// Their codes under that scale
__device__ __forceinline__ unsigned mx_codes8(const float v[8], unsigned s) {
  const float f = mx_inv_scale(s);
  float t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = v[e] * f;
  return s == 255 ? 0u : mx_pack8(t);
}
