// What the products in microscaled 4-bit floating point share: the matrix instruction, and a tile's way to the output.
//
// v_mfma_scale_f32_32x32x64_f8f6f4 takes one block of 32 codes (16 bytes) and its scale byte from
// each lane: lane l holds row l % 32, and k block l / 32 of the two that a step covers.  Which two blocks
// of a row's group of eight go together is free as long as both operands agree: step s takes
// blocks s (lanes 0-31) and 4 + s (lanes 32-63), so that a lane's four scale bytes of a group are
// one aligned dword of the scale layout, picked by the instruction's own byte select.
//
// The weights are the A operand: a lane then holds one token (accumulator column) and, of every 32
// outputs, 4 groups of 4 consecutive ones (outputs 8 (i / 4) + 4 (l / 32) + i % 4).
#pragma once

#include "attn_tile.h"
#include "icsa_kernels.h"
#include "mx_common.h"

#define MXG_LINE 128                                   // bytes of codes of one row and group

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// byte `kSel` of each scale register, both operands e2m1 (format 4)
template <int kSel>
__device__ __forceinline__ floatx16 mx_mfma(i32x4 a, i32x4 b, floatx16 c, int sa, int sb) {
  const i32x8 a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, kSel, sa, kSel, sb);
}

// gelu(t) = t / (1 + exp(-2 sqrt(2 / pi) (t + 0.044715 t^3))): no difference of near values on
// either side of zero.  exp2 of a large argument is infinity and the factor 0.
__device__ __forceinline__ float gelu_tanh(float t) {
  const float u = t * fmaf(0.044715f * t, t, 1.f);
  return t * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u * (-2.f * 0.7978845608028654f * 1.4426950408889634f)));
}

// Outputs of a row that are written: in 4 bits its padding too
__host__ __device__ __forceinline__ int out_columns(const MxGemmParams& p) {
  return p.out_kind == MX_OUT_MXFP4 ? mx_padded(p.N) : p.N;
}

__device__ __forceinline__ float bias_at(const MxGemmParams& p, int n) {
  if (p.bias == nullptr || n >= p.N) return 0.f;
  return p.bias_dtype == ICSA_DT_F32 ? reinterpret_cast<const float*>(p.bias)[n]
                                     : (float)reinterpret_cast<const bf16*>(p.bias)[n];
}

// activation of one 32 (n) x 32 (m) accumulator tile
__device__ __forceinline__ void tile_values(const MxGemmParams& p, const floatx16& acc, float v[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = acc[i];
  if (p.gelu) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = gelu_tanh(v[i]);
  }
}

// The tile's outputs n0 .. n0 + 31 of token m (this lane's) in 4 bits
__device__ __forceinline__ void store_mx(const MxGemmParams& p, float v[16], int n0, int m) {
  const int hl = (threadIdx.x & 63) >> 5, Np = mx_padded(p.N);
  unsigned amax = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (n0 + 8 * (i >> 2) + 4 * hl + (i & 3) >= p.N) v[i] = 0.f;         // the padding: zeros
    amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
  }
  const auto w = __builtin_amdgcn_permlane32_swap(amax, amax, false, false);
  const unsigned s = mx_scale_byte(max(w[0], w[1]));
  const float f = mx_inv_scale(s);
  unsigned q[2];                                       // 4 groups of 4 codes: 16 bits each
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = v[8 * h + e] * f;
    q[h] = s == 255 ? 0u : mx_pack8(t);
  }
  // lanes l and l ^ 32 hold alternating groups of 4 codes (hl = 0 first): lower lanes gather the
  // block's first 16 codes, upper lanes the last 16
  const auto x = __builtin_amdgcn_permlane32_swap(q[0], q[1], false, false);
  const unsigned lo = x[0], hi = x[1];                 // this half's codes of groups 2 hl, 2 hl + 1: from hl = 0, 1
  const u32x2 c = {(lo & 0xffffu) | hi << 16, lo >> 16 | (hi & 0xffff0000u)};
  if (m < p.m_last && n0 < Np) {
    *reinterpret_cast<u32x2*>(reinterpret_cast<unsigned char*>(p.out) + (int64_t)m * p.o_ss + n0 / 2 + 8 * hl) = c;
    if (hl == 0)
      p.out_scales[((int64_t)(n0 / MX_GROUP) * p.M + m) * MX_GROUP_BLOCKS + n0 / MX_BLOCK % MX_GROUP_BLOCKS] = (unsigned char)s;
  }
}

__device__ __forceinline__ void store_f32(const MxGemmParams& p, const float v[16], int n0, int m) {
  const int hl = (threadIdx.x & 63) >> 5;
  if (m >= p.m_last) return;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int n = n0 + 8 * g + 4 * hl;
    float* dst = reinterpret_cast<float*>(p.out) + (int64_t)m * p.o_ss + n;
    if (n + 4 <= p.N) *reinterpret_cast<floatx4_a4*>(dst) = floatx4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
    else
#pragma unroll
      for (int e = 0; e < 4; ++e) if (n + e < p.N) dst[e] = v[4 * g + e];
  }
}

// bf16 rows pass through 2 KB of the wave's LDS, 32 outputs of 32 tokens at a time, so that a store
// instruction writes 16 segments of 64 bytes.  16-byte chunk c of row r at c ^ (r / 4 % 4).
__device__ __forceinline__ void store_bf16(const MxGemmParams& p, unsigned char* stage, const float v[16], int n0, int m0) {
  const int lane = threadIdx.x & 63, li = lane & 31, hl = lane >> 5;
#pragma unroll
  for (int pr = 0; pr < 2; ++pr) {                     // lane halves swap: outputs 8 (2 pr + hl) .. + 7
    bf16x4 lo, hi;
#pragma unroll
    for (int e = 0; e < 4; ++e) { lo[e] = (bf16)v[8 * pr + e]; hi[e] = (bf16)v[8 * pr + 4 + e]; }
    const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
    const auto w0 = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false);
    const auto w1 = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
    *reinterpret_cast<u32x4*>(stage + li * 64 + (((2 * pr + hl) ^ ((li >> 2) & 3)) << 4)) = u32x4{w0[0], w1[0], w0[1], w1[1]};
  }
  const int n = n0 + 8 * (lane & 3);
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int r = 16 * x + (lane >> 2), m = m0 + r;
    const u32x4 c = *reinterpret_cast<const u32x4*>(stage + r * 64 + (((lane & 3) ^ ((r >> 2) & 3)) << 4));
    bf16* dst = reinterpret_cast<bf16*>(p.out) + (int64_t)m * p.o_ss + n;
    if (m < p.m_last && n + 8 <= p.N) *reinterpret_cast<u32x4_a2*>(dst) = c;
    else if (m < p.m_last) {
      const bf16x8 b = __builtin_bit_cast(bf16x8, c);
#pragma unroll
      for (int e = 0; e < 8; ++e) if (n + e < p.N) dst[e] = b[e];
    }
  }
}
