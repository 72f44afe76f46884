// Quantisation of rows to microscaled 4-bit floating point, and back.
//
// Both are one pass over memory: bf16 in 2 bytes a value, out 17/32 of a byte.  The quantisation is bound by them (14,040 x 5,120:
// 42 us, 4.3 TB/s); the way back, 41 us there, keeps the vector pipe 94 % busy with unpacking eight codes a lane.  Four lanes
// share a block of 32 values (8 each, one 16-byte load in bf16), so that a wave's loads and its
// code stores are contiguous; the block's largest magnitude is the maximum of the f32 bit patterns
// without their sign (integers: NaN and infinity come out on top), two exchanges between lanes.
#include "icsa_kernels.h"
#include "mx_common.h"

#define MXQ_THREADS 256
#define MXQ_WAVE_K 512                     // values of one row that a wave takes at a time
#define MXQ_AHEAD 4                        // such pieces requested together by a wave, one where there are few
// Up to so many pieces a wave takes one.  One against four, in us, quantisation of bf16 | dequantisation: 15,600 pieces (1,560 x
// 5,120) 6.8 to 7.6 | 8.8 to 9.9; 31,200 11.7 to 12.8 | 14.9 to 16.2; 46,800 16.2 to 18.4 | 20.5 to 20.3; 93,600 27.6 to 30.4 |
// 36.7 to 34.5; 140,400 39.6 to 42.3 | 53.9 to 49.0; 655,200 171 to 159 | 233 to 203.  (The quantisation alone would go over later.)
#define MXQ_FEW 32768

template <typename T, int kAhead>
__global__ void __launch_bounds__(MXQ_THREADS) icsa_mx_quantize_kernel(MxQuantParams p) {
  const int lane = threadIdx.x & 63;
  const int Kp = mx_padded(p.K), per_row = (Kp + MXQ_WAVE_K - 1) / MXQ_WAVE_K;
  const int64_t pieces = p.M * per_row;
  const int64_t wave = (int64_t)blockIdx.x * (MXQ_THREADS / 64) + (threadIdx.x >> 6);
  const int64_t first = wave * kAhead;
  float v[kAhead][8];
  int64_t row[kAhead];
  int k[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int64_t u = first + i;
    row[i] = u / per_row;
    k[i] = (int)(u % per_row) * MXQ_WAVE_K + 8 * lane;
    if (u < pieces) load8_row<T>(reinterpret_cast<const T*>(p.x) + row[i] * p.x_ss, k[i], p.K, v[i]);
  }
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    if (first + i >= pieces) return;                     // uniform for the wave
    const unsigned s = mx_quantize8(v[i]), codes = mx_codes8(v[i], s);
    if (k[i] < Kp) {
      *reinterpret_cast<unsigned*>(p.codes + row[i] * (Kp / 2) + k[i] / 2) = codes;
      if ((lane & 3) == 0)
        p.scales[((int64_t)(k[i] / MX_GROUP) * p.M + row[i]) * MX_GROUP_BLOCKS + k[i] / MX_BLOCK % MX_GROUP_BLOCKS] =
            (unsigned char)s;
    }
  }
}

hipError_t launch_mx_quantize(const MxQuantParams& p, hipStream_t stream) {
  if (p.M == 0) return hipSuccess;
  const int64_t pieces = p.M * ((mx_padded(p.K) + MXQ_WAVE_K - 1) / MXQ_WAVE_K);
  const bool few = pieces < MXQ_FEW;
  const int64_t per_wg = (MXQ_THREADS / 64) * (few ? 1 : MXQ_AHEAD);
  const int64_t grid = (pieces + per_wg - 1) / per_wg;
  if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
  const dim3 g((unsigned)grid), b(MXQ_THREADS);
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, b, 0, stream, p); };
  if (p.x_dtype == ICSA_DT_F32) {
    if (few) run(icsa_mx_quantize_kernel<float, 1>); else run(icsa_mx_quantize_kernel<float, MXQ_AHEAD>);
  } else {
    if (few) run(icsa_mx_quantize_kernel<bf16, 1>); else run(icsa_mx_quantize_kernel<bf16, MXQ_AHEAD>);
  }
  return hipGetLastError();
}

// Values of 8 codes a lane.  A code's value times a power of two has at most two significant
// bits, so bf16 holds every value below 2^128 (2^-128, the least, is a bf16 subnormal; from 2^128 on, under
// bytes that the quantisation does not write, both types have infinities); the product with a
// subnormal scale is exact in f32, and its upper half is the bf16.
template <typename T, int kAhead>
__global__ void __launch_bounds__(MXQ_THREADS) icsa_mx_dequantize_kernel(MxDequantParams p) {
  const int lane = threadIdx.x & 63;
  const int Kp = mx_padded(p.K), per_row = (p.K + MXQ_WAVE_K - 1) / MXQ_WAVE_K;
  const int64_t pieces = p.M * per_row;
  const int64_t wave = (int64_t)blockIdx.x * (MXQ_THREADS / 64) + (threadIdx.x >> 6);
  const int64_t first = wave * kAhead;
  unsigned code[kAhead];
  unsigned s[kAhead];
  int64_t row[kAhead];
  int k[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    const int64_t u = first + i;
    row[i] = u / per_row;
    k[i] = (int)(u % per_row) * MXQ_WAVE_K + 8 * lane;
    if (u < pieces && k[i] < p.K) {
      code[i] = *reinterpret_cast<const unsigned*>(p.codes + row[i] * (Kp / 2) + k[i] / 2);
      s[i] = p.scales[((int64_t)(k[i] / MX_GROUP) * p.M + row[i]) * MX_GROUP_BLOCKS + k[i] / MX_BLOCK % MX_GROUP_BLOCKS];
    }
  }
#pragma unroll
  for (int i = 0; i < kAhead; ++i) {
    if (first + i >= pieces || k[i] >= p.K) continue;
    const float f = mx_scale(s[i]);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const unsigned c = (code[i] >> (4 * e)) & 15u, m = c & 7u;
      // exponent field 0: m / 2; else (1 + mantissa / 2) 2^(exponent - 1)
      const float a = m < 2 ? 0.5f * (float)m : __uint_as_float(((m >> 1) + 126u) << 23 | (m & 1u) << 22);
      v[e] = (c & 8u ? -a : a) * f;
    }
    T* dst = reinterpret_cast<T*>(p.out) + row[i] * p.o_ss + k[i];
    if constexpr (sizeof(T) == 2) {
      unsigned short h[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = (unsigned short)(__float_as_uint(v[e]) >> 16);
      if (k[i] + 8 <= p.K) {
        *reinterpret_cast<u32x4_a2*>(dst) = u32x4{h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16,
                                               h[4] | (unsigned)h[5] << 16, h[6] | (unsigned)h[7] << 16};
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k[i] + e < p.K) reinterpret_cast<unsigned short*>(dst)[e] = h[e];
      }
    } else if (k[i] + 8 <= p.K) {
      *reinterpret_cast<floatx4_a4*>(dst) = floatx4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<floatx4_a4*>(dst + 4) = floatx4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k[i] + e < p.K) dst[e] = v[e];
    }
  }
}

hipError_t launch_mx_dequantize(const MxDequantParams& p, hipStream_t stream) {
  if (p.M == 0) return hipSuccess;
  const int64_t pieces = p.M * ((p.K + MXQ_WAVE_K - 1) / MXQ_WAVE_K);
  const bool few = pieces < MXQ_FEW;
  const int64_t per_wg = (MXQ_THREADS / 64) * (few ? 1 : MXQ_AHEAD);
  const int64_t grid = (pieces + per_wg - 1) / per_wg;
  if (grid > 0x7fffffffLL) return hipErrorInvalidValue;
  const dim3 g((unsigned)grid), b(MXQ_THREADS);
  auto run = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, b, 0, stream, p); };
  if (p.out_dtype == ICSA_DT_F32) {
    if (few) run(icsa_mx_dequantize_kernel<float, 1>); else run(icsa_mx_dequantize_kernel<float, MXQ_AHEAD>);
  } else {
    if (few) run(icsa_mx_dequantize_kernel<bf16, 1>); else run(icsa_mx_dequantize_kernel<bf16, MXQ_AHEAD>);
  }
  return hipGetLastError();
}
