// Rotary positions: the pair j of a head's first R dims is turned by its token's angle,
//   (x0, x1) -> (x0 c - x1 s, x0 s + x1 c),  c = cos[pos][j], s = sin[pos][j],
// and back (the transposed matrix, s -> -s) for gradients.  Pair j is dims 2 j, 2 j + 1 (interleaved) or j, j + R / 2 (halves); dims from R on
// are copied.  Up to four axes: consecutive runs of pairs turn by positions of their own (frames, rows, columns).  Pairs whose position
// is outside the table are copied, whatever they hold.  Tables are f32 from angles in 64 bits, the products f32, rounded once.
//
// A wave takes one token, or part of its heads where tokens are few: a lane keeps its pairs' cos and sin over the heads, so that
// tables are read once a token, and what bounds the kernel is x in and y out: q and k of 65,520 tokens, 40 heads of 128 each, take 496 us
// for 2.7 GB (5.4 TB/s).  Two tensors (q and k) go in one launch; 8 tokens of 40 and 8 heads take 4.6 us, most of it launch.
#include "icsa_kernels.h"

#define RO_THREADS 256
#define RO_WAVES 4
#define RO_UNROLL 4

namespace {

// position of pair j's axis, or -1 for one outside the table
__device__ __forceinline__ int pair_pos(const RotaryParams& p, const int* pos, int j) {
  int a = 0;
#pragma unroll
  for (int x = 0; x < RO_MAX_AXES - 1; ++x) a += x + 1 < p.axes && j >= p.ends[x];
  const int at = pos[a];
  return at >= 0 && at < p.rows ? at : -1;
}

template <typename T, int N> struct Vec;
template <> struct Vec<bf16, 8> {
  bf16x8 v;
  __device__ __forceinline__ void load(const bf16* p) { v = *reinterpret_cast<const bf16x8*>(p); }
  __device__ __forceinline__ void store(bf16* p) const { *reinterpret_cast<bf16x8*>(p) = v; }
  __device__ __forceinline__ float at(int e) const { return (float)v[e]; }
  __device__ __forceinline__ void set(int e, float x) { v[e] = (bf16)x; }
};
template <> struct Vec<float, 8> {
  floatx4 v[2];
  __device__ __forceinline__ void load(const float* p) { v[0] = reinterpret_cast<const floatx4*>(p)[0]; v[1] = reinterpret_cast<const floatx4*>(p)[1]; }
  __device__ __forceinline__ void store(float* p) const { reinterpret_cast<floatx4*>(p)[0] = v[0]; reinterpret_cast<floatx4*>(p)[1] = v[1]; }
  __device__ __forceinline__ float at(int e) const { return v[e >> 2][e & 3]; }
  __device__ __forceinline__ void set(int e, float x) { v[e >> 2][e & 3] = x; }
};

}  // namespace

// Whole 8-element chunks.  A lane has one unit of a head: interleaved, a chunk (4 pairs); halves, chunk c of either half (8 pairs);
// or a chunk past R.
template <typename T, bool HALF>
__global__ void __launch_bounds__(RO_THREADS) icsa_rotary_kernel(RotaryParams p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t item = (int64_t)blockIdx.x * RO_WAVES + wave;
  if (item >= p.tokens * p.shares) return;
  const int64_t tok = item / p.shares;
  const int share = (int)(item - tok * p.shares), b = (int)(tok / p.S), s = (int)(tok - (int64_t)b * p.S);
  constexpr int kPairs = HALF ? 8 : 4;
  const int turned = HALF ? p.R / 16 : p.R / 8, units = turned + (p.D - p.R) / 8, heads = 64 / units;   // heads a pass
  const int u = lane % units, h0 = lane / units;
  const bool on = h0 < heads, turn = u < turned;
  const int first = HALF ? (turn ? 8 * u : p.R + 8 * (u - turned)) : 8 * u;    // the unit's first dim
  const int half = HALF && turn ? p.R / 2 : 0;
  float c[kPairs] = {}, sn[kPairs] = {};
  unsigned still = 0u;                                // pairs that are copied: 0 times an infinity would not be
  if (on && turn) {
    const int* pos = p.pos + (int64_t)b * p.pos_sb + (int64_t)s * p.axes;
    const int np = p.R / 2, j0 = kPairs * u;
    const int at0 = pair_pos(p, pos, j0);
    bool alike = true;
#pragma unroll
    for (int x = 0; x < RO_MAX_AXES - 1; ++x) alike = alike && !(x + 1 < p.axes && j0 < p.ends[x] && j0 + kPairs > p.ends[x]);
    if (alike) {
      if (at0 >= 0) {
#pragma unroll
        for (int e = 0; e < kPairs; e += 4) {
          const floatx4 c4 = *reinterpret_cast<const floatx4*>(p.cos + (int64_t)at0 * np + j0 + e);
          const floatx4 s4 = *reinterpret_cast<const floatx4*>(p.sin + (int64_t)at0 * np + j0 + e);
#pragma unroll
          for (int x = 0; x < 4; ++x) { c[e + x] = c4[x]; sn[e + x] = s4[x]; }
        }
      } else {
        still = ~0u;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kPairs; ++e) {
        const int at = pair_pos(p, pos, j0 + e);
        if (at >= 0) { c[e] = p.cos[(int64_t)at * np + j0 + e]; sn[e] = p.sin[(int64_t)at * np + j0 + e]; }
        else still |= 1u << e;
      }
    }
    if (p.back) {
#pragma unroll
      for (int e = 0; e < kPairs; ++e) sn[e] = -sn[e];
    }
  }
  if (!on) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int H = p.H[i];
    if (H == 0) continue;
    // this share's heads, whole passes: 2^20 passes by 2^11 shares at most, without a sign in 32 bits
    const unsigned passes = (unsigned)(H + heads - 1) / heads;
    const int h_lo = (int)(passes * share / p.shares) * heads, h_hi = min(H, (int)(passes * (share + 1) / p.shares) * heads);
    const T* x = reinterpret_cast<const T*>(p.x[i]) + (int64_t)b * p.sb[i] + (int64_t)s * p.ss[i] + first;
    T* y = reinterpret_cast<T*>(p.y[i]) + (tok * H) * p.D + first;
    for (int hh = h_lo + h0; hh < h_hi; hh += RO_UNROLL * heads) {
      Vec<T, 8> v[RO_UNROLL], w[HALF ? RO_UNROLL : 1];
#pragma unroll
      for (int k = 0; k < RO_UNROLL; ++k) {
        const int h = hh + k * heads;
        if (h < h_hi) {
          v[k].load(x + (int64_t)h * p.sh[i]);
          if (HALF && turn) w[k].load(x + (int64_t)h * p.sh[i] + half);
        }
      }
#pragma unroll
      for (int k = 0; k < RO_UNROLL; ++k) {
        const int h = hh + k * heads;
        if (h >= h_hi) continue;
        if (turn) {
          if constexpr (HALF) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float a = v[k].at(e), d = w[k].at(e);
              if (still >> e & 1u) continue;
              v[k].set(e, fmaf(a, c[e], -d * sn[e]));
              w[k].set(e, fmaf(a, sn[e], d * c[e]));
            }
            w[k].store(y + (int64_t)h * p.D + half);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float a = v[k].at(2 * e), d = v[k].at(2 * e + 1);
              if (still >> e & 1u) continue;
              v[k].set(2 * e, fmaf(a, c[e], -d * sn[e]));
              v[k].set(2 * e + 1, fmaf(a, sn[e], d * c[e]));
            }
          }
        }
        v[k].store(y + (int64_t)h * p.D);
      }
    }
  }
}

// Any sizes, strides and alignment: a lane takes a pair, or a dim past R, at a time, in elements: 65,520 tokens, 12 + 12 heads of 80 with 20 dims
// turned 365 us, 40 in halves 323 (105 by their bytes; the kernel above, 40 interleaved, 92).
template <typename T>
__global__ void __launch_bounds__(RO_THREADS) icsa_rotary_any_kernel(RotaryParams p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t item = (int64_t)blockIdx.x * RO_WAVES + wave;
  if (item >= p.tokens * p.shares) return;
  const int64_t tok = item / p.shares;
  const int share = (int)(item - tok * p.shares), b = (int)(tok / p.S), s = (int)(tok - (int64_t)b * p.S);
  const int np = p.R / 2, units = np + p.D - p.R;
  const int* pos = p.pos + (int64_t)b * p.pos_sb + (int64_t)s * p.axes;
  for (int i = 0; i < 2; ++i) {
    const int H = p.H[i], h_lo = (int)((int64_t)H * share / p.shares), h_hi = (int)((int64_t)H * (share + 1) / p.shares);
    const T* x = reinterpret_cast<const T*>(p.x[i]) + (int64_t)b * p.sb[i] + (int64_t)s * p.ss[i];
    T* y = reinterpret_cast<T*>(p.y[i]) + (tok * H) * p.D;
    for (int at = lane; at < (h_hi - h_lo) * units; at += 64) {
      const int h = h_lo + at / units, u = at % units;
      const T* xh = x + (int64_t)h * p.sh[i];
      T* yh = y + (int64_t)h * p.D;
      if (u >= np) {
        yh[p.R + u - np] = xh[p.R + u - np];
        continue;
      }
      const int ps = pair_pos(p, pos, u), d0 = p.halves ? u : 2 * u, d1 = p.halves ? u + np : 2 * u + 1;
      if (ps < 0) {                                   // copied
        yh[d0] = xh[d0];
        yh[d1] = xh[d1];
        continue;
      }
      const float c = p.cos[(int64_t)ps * np + u], sn = p.back ? -p.sin[(int64_t)ps * np + u] : p.sin[(int64_t)ps * np + u];
      const float a = (float)xh[d0], d = (float)xh[d1];
      yh[d0] = (T)fmaf(a, c, -d * sn);
      yh[d1] = (T)fmaf(a, sn, d * c);
    }
  }
}

hipError_t launch_rotary(RotaryParams p, bool vec, hipStream_t stream) {
  // waves to fill the chip with: a token's heads are shared where tokens are few
  const int most = p.H[0] > p.H[1] ? p.H[0] : p.H[1];
  const int units = vec ? (p.halves ? p.R / 16 + (p.D - p.R) / 8 : p.D / 8) : 1;
  const int passes = vec ? (most + 64 / units - 1) / (64 / units) : most;
  int64_t shares = 2048 / p.tokens;
  shares = shares < 1 ? 1 : shares > passes ? passes : shares;
  p.shares = (int)shares;
  const int64_t wg = (p.tokens * shares + RO_WAVES - 1) / RO_WAVES;
  if (wg > 0x7fffffffLL) return hipErrorInvalidValue;
  const dim3 grid((unsigned)wg), threads(RO_THREADS);
  const bool f32 = p.dtype == ICSA_DT_F32;
  if (!vec) {
    if (f32) hipLaunchKernelGGL(icsa_rotary_any_kernel<float>, grid, threads, 0, stream, p);
    else hipLaunchKernelGGL(icsa_rotary_any_kernel<bf16>, grid, threads, 0, stream, p);
  } else if (p.halves) {
    if (f32) hipLaunchKernelGGL((icsa_rotary_kernel<float, true>), grid, threads, 0, stream, p);
    else hipLaunchKernelGGL((icsa_rotary_kernel<bf16, true>), grid, threads, 0, stream, p);
  } else {
    if (f32) hipLaunchKernelGGL((icsa_rotary_kernel<float, false>), grid, threads, 0, stream, p);
    else hipLaunchKernelGGL((icsa_rotary_kernel<bf16, false>), grid, threads, 0, stream, p);
  }
  return hipGetLastError();
}
