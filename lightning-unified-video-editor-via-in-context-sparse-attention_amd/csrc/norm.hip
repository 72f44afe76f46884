// Layer norm and RMS norm with their backward, f32 inside whatever the rows' types.
//   xh = (x - mean) r, r = 1 / sqrt(mean((x - mean)^2) + eps)   (RMS norm: mean = 0)
//   y  = xh a + b        a, b [dim] of a group of rows: a weight, or 1 + scale of a batch row
//   u  = dy a;  dx = r (u - mean(u) - xh mean(u xh))            (RMS norm: without mean(u))
//   da = sum over the group's rows of dy xh;  db = sum of dy
//
// A row is held by a quarter wave up to 256 elements, a wave up to 1,024, a workgroup up to 8,192, 8 elements a lane or twice
// as many.  Workgroups walk their group's rows with a stride and keep a, b and their partial da, db in registers; the next
// rows are requested before the present ones' sums are taken.  The forward takes the variance of the centred row from the registers
// (two reductions); the backward's two sums are one.  da and db: every workgroup's partial sums go to memory, and a second
// kernel adds them in a fixed order (the same inputs give the same bits).
//
// What bounds it: the bytes.  65,520 f32 rows of 5,120 into bf16 take 380 us (2.0 GB, 5.3 TB/s) and back 597 (3.4 GB, 5.6; a large copy
// reaches 4.9, its half of reads less); 28,080 bf16 rows with a scale and shift 110 and 184; 9,373 of 1,536 15.5 and 20.5.  6 rows: 5.3 and
// 9.7, launch and two trips to memory; the call is the host's.  Rows that are not whole 16-byte chunks are read and written by elements: 28,080 bf16 rows of 5,119
// take 333 and 486 us (of 5,120 118 and 186), 65,520 of 1,001 123 and 218 (of 1,000 43 and 98).
#include "icsa_kernels.h"

#define NM_THREADS 256
#define NM_MAX_THREADS 512                            // 8,192 elements, two chunks of 8 a thread
#define NM_WAVES 1024                                 // one a SIMD
#define NM_FEW_ROWS 2                                 // of a group: one workgroup, which needs no second kernel
#define NM_FEW_TOTAL 8                                // rows of all groups, back: columns instead of rows to workgroups, in one launch
#define NM_FEW_COLS 512

namespace {

template <typename T> struct Raw8;
template <> struct Raw8<bf16> {
  bf16x8 v;
  __device__ __forceinline__ float at(int e) const { return (float)v[e]; }
  __device__ __forceinline__ void load(const bf16* p, int n, bool vec) {
    if (vec) { v = n > 0 ? *reinterpret_cast<const bf16x8*>(p) : bf16x8{}; return; }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : (bf16)0.f;
  }
};
template <> struct Raw8<float> {
  floatx4 v[2];
  __device__ __forceinline__ float at(int e) const { return v[e >> 2][e & 3]; }
  __device__ __forceinline__ void load(const float* p, int n, bool vec) {
    if (vec) {
      v[0] = n > 0 ? *reinterpret_cast<const floatx4*>(p) : floatx4{};
      v[1] = n > 0 ? *reinterpret_cast<const floatx4*>(p + 4) : floatx4{};
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e >> 2][e & 3] = e < n ? p[e] : 0.f;
  }
};

__device__ __forceinline__ void store8(bf16* p, const float v[8], int n, bool vec) {
  if (vec) {
    if (n > 0) *reinterpret_cast<bf16x8*>(p) = pack8_bf16(v);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) p[e] = (bf16)v[e];
}
__device__ __forceinline__ void store8(float* p, const float v[8], int n, bool vec) {
  if (vec) {
    if (n > 0) {
      *reinterpret_cast<floatx4*>(p) = floatx4{v[0], v[1], v[2], v[3]};
      *reinterpret_cast<floatx4*>(p + 4) = floatx4{v[4], v[5], v[6], v[7]};
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) p[e] = v[e];
}

// Sum over LPR = 16 or 64 neighbouring lanes, in all of them
template <int kCtrl> __device__ __forceinline__ float dpp_add(float x) {
  return x + __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), kCtrl, 0xf, 0xf, false));
}
template <int LPR> __device__ __forceinline__ float lanes_sum(float x) {
  x = dpp_add<0x128>(x);                              // rotations by 8, 4, 2, 1 within 16 lanes
  x = dpp_add<0x124>(x);
  x = dpp_add<0x122>(x);
  x = dpp_add<0x121>(x);
  if constexpr (LPR > 16) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    x = xhalf_sum(x);
  }
  return x;
}

// Sums of N values over a row's lanes (LPR 0: the workgroup's).  red: buffers used in turn, so that one barrier is enough.
template <int LPR, int N> __device__ __forceinline__ void row_sums(float (&x)[N], float (*red)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = lanes_sum<LPR == 16 ? 16 : 64>(x[i]);
  if constexpr (LPR == 0) {
    const int waves = blockDim.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) red[threadIdx.x >> 6][i] = x[i];
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");    // the next row's loads stay in flight
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = red[0][i];
    for (int w = 1; w < waves; ++w) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] += red[w][i];
    }
  }
}

// a or b of the lane's elements, f32: `none` where there is none, or plus + the parameter
template <int NCH>
__device__ __forceinline__ void load_params(const NormParams& p, const void* src, int64_t at, int t, int lanes, float v[NCH][8],
                                            const int n[NCH], float none, float plus) {
#pragma unroll
  for (int u = 0; u < NCH; ++u) {
    const int64_t i = at + 8 * (t + u * lanes);
    if (src == nullptr) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[u][e] = none;
    } else if (p.p_dtype == ICSA_DT_F32) {
      Raw8<float> x;
      x.load(reinterpret_cast<const float*>(src) + i, n[u], p.vec_p);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[u][e] = plus + x.at(e);
    } else {
      Raw8<bf16> x;
      x.load(reinterpret_cast<const bf16*>(src) + i, n[u], p.vec_p);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[u][e] = plus + x.at(e);
    }
  }
}

}  // namespace

template <typename TX, typename TY, bool RMS, int LPR, int NCH>
__global__ void __launch_bounds__(LPR == 0 ? NM_MAX_THREADS : NM_THREADS) icsa_norm_fwd_kernel(NormParams p) {
  constexpr int kRows = LPR == 0 ? 1 : NM_THREADS / (LPR == 0 ? 1 : LPR);
  __shared__ float red[4][NM_MAX_THREADS / 64][1];
  const int lanes = LPR == 0 ? blockDim.x : LPR, t = LPR == 0 ? threadIdx.x : threadIdx.x % (LPR == 0 ? 1 : LPR),
            sub = LPR == 0 ? 0 : threadIdx.x / (LPR == 0 ? 1 : LPR), g = blockIdx.y;
  int n[NCH];
#pragma unroll
  for (int u = 0; u < NCH; ++u) n[u] = p.dim - 8 * (t + u * lanes);
  float a[NCH][8], b[NCH][8];
  load_params<NCH>(p, p.gain, g * p.p_sg, t, lanes, a, n, 1.f, p.plus_one ? 1.f : 0.f);
  load_params<NCH>(p, p.shift, g * p.p_sg, t, lanes, b, n, 0.f, 0.f);
  const float inv_n = 1.f / (float)p.dim;
  const TX* x = reinterpret_cast<const TX*>(p.x) + 8 * t;
  TY* y = reinterpret_cast<TY*>(p.y) + 8 * t;
  const bool vx = p.vec_x, vy = p.vec_y;
  const int64_t row0 = (int64_t)g * p.rows, step = (int64_t)gridDim.x * kRows;
  Raw8<TX> next[NCH];
  auto fetch = [&](int64_t r) {
    const TX* src = x + (row0 + min(r, p.rows - 1)) * p.x_ss;
#pragma unroll
    for (int u = 0; u < NCH; ++u) next[u].load(src + 8 * u * lanes, n[u], vx);
  };
  int turn = 0;
  int64_t r = (int64_t)blockIdx.x * kRows + sub;
  fetch(r);
  for (int64_t r_wg = (int64_t)blockIdx.x * kRows; r_wg < p.rows; r_wg += step, r += step) {
    float v[NCH][8], s[1] = {0.f};
#pragma unroll
    for (int u = 0; u < NCH; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[u][e] = next[u].at(e);
        s[0] += v[u][e];
      }
    fetch(r + step);
    float mean = 0.f;
    if constexpr (!RMS) {
      row_sums<LPR>(s, red[turn]);
      turn = (turn + 1) & 3;
      mean = s[0] * inv_n;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int u = 0; u < NCH; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[u][e] = e < n[u] ? v[u][e] - mean : 0.f;
        q[0] = fmaf(v[u][e], v[u][e], q[0]);
      }
    row_sums<LPR>(q, red[turn]);
    turn = (turn + 1) & 3;
    const float rstd = 1.f / sqrtf(q[0] * inv_n + p.eps);
    if (r >= p.rows) continue;
    TY* dst = y + (row0 + r) * p.y_ss;
#pragma unroll
    for (int u = 0; u < NCH; ++u) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = fmaf(v[u][e] * rstd, a[u][e], b[u][e]);
      store8(dst + 8 * u * lanes, o, n[u], vy);
    }
    if (t == 0) {
      if (p.rstd != nullptr) p.rstd[row0 + r] = rstd;
      if (!RMS && p.mean != nullptr) p.mean[row0 + r] = mean;
    }
  }
}

template <typename TX, typename TY, bool RMS, int LPR, int NCH>
__global__ void __launch_bounds__(LPR == 0 ? NM_MAX_THREADS : NM_THREADS) icsa_norm_bwd_kernel(NormParams p) {
  constexpr int kRows = LPR == 0 ? 1 : NM_THREADS / (LPR == 0 ? 1 : LPR);
  __shared__ float red[2][NM_MAX_THREADS / 64][2];
  const int lanes = LPR == 0 ? blockDim.x : LPR, t = LPR == 0 ? threadIdx.x : threadIdx.x % (LPR == 0 ? 1 : LPR),
            sub = LPR == 0 ? 0 : threadIdx.x / (LPR == 0 ? 1 : LPR), g = blockIdx.y;
  int n[NCH];
#pragma unroll
  for (int u = 0; u < NCH; ++u) n[u] = p.dim - 8 * (t + u * lanes);
  float a[NCH][8], da[NCH][8], db[NCH][8];
  load_params<NCH>(p, p.gain, g * p.p_sg, t, lanes, a, n, 1.f, p.plus_one ? 1.f : 0.f);
#pragma unroll
  for (int u = 0; u < NCH; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e) da[u][e] = db[u][e] = 0.f;
  const float inv_n = 1.f / (float)p.dim;
  const TX* x = reinterpret_cast<const TX*>(p.x) + 8 * t;
  const TY* y = reinterpret_cast<const TY*>(p.dy) + 8 * t;
  TX* dx = reinterpret_cast<TX*>(p.dx) + 8 * t;
  const bool vx = p.vec_x, vy = p.vec_y, vd = p.vec_dx;
  const int64_t row0 = (int64_t)g * p.rows, step = (int64_t)gridDim.x * kRows;
  Raw8<TX> nx[NCH];
  Raw8<TY> ny[NCH];
  float n_mean = 0.f, n_rstd = 0.f;
  auto fetch = [&](int64_t r) {
    const int64_t at = row0 + min(r, p.rows - 1);
#pragma unroll
    for (int u = 0; u < NCH; ++u) {
      nx[u].load(x + at * p.x_ss + 8 * u * lanes, n[u], vx);
      ny[u].load(y + at * p.dy_ss + 8 * u * lanes, n[u], vy);
    }
    if (!RMS) n_mean = p.mean[at];
    n_rstd = p.rstd[at];
  };
  int turn = 0;
  int64_t r = (int64_t)blockIdx.x * kRows + sub;
  fetch(r);
  for (int64_t r_wg = (int64_t)blockIdx.x * kRows; r_wg < p.rows; r_wg += step, r += step) {
    const float mean = n_mean, rstd = n_rstd, on = r < p.rows ? 1.f : 0.f;
    float xh[NCH][8], u8[NCH][8], s[2] = {0.f, 0.f};
#pragma unroll
    for (int u = 0; u < NCH; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = ny[u].at(e);
        xh[u][e] = e < n[u] ? (nx[u].at(e) - mean) * rstd : 0.f;
        u8[u][e] = d * a[u][e];
        s[0] = fmaf(u8[u][e], xh[u][e], s[0]);
        s[1] += u8[u][e];
        if (kRows == 1 || on != 0.f) {                // rows past the last: nothing to the sums
          da[u][e] = fmaf(d, xh[u][e], da[u][e]);
          db[u][e] += d;
        }
      }
    fetch(r + step);
    row_sums<LPR>(s, red[turn]);
    turn ^= 1;
    if (r >= p.rows || p.dx == nullptr) continue;
    const float m1 = s[0] * inv_n, m0 = RMS ? 0.f : s[1] * inv_n;
    TX* dst = dx + (row0 + r) * p.dx_ss;
#pragma unroll
    for (int u = 0; u < NCH; ++u) {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = rstd * (u8[u][e] - m0 - xh[u][e] * m1);
      store8(dst + 8 * u * lanes, o, n[u], vd);
    }
  }
  if (p.part == nullptr) {
    if (kRows > 1 || (p.dgain == nullptr && p.dshift == nullptr)) return;
    // the group's only workgroup: its sums are the result
#pragma unroll
    for (int u = 0; u < NCH; ++u) {
      const int64_t at = (int64_t)g * p.dim + 8 * (t + u * lanes);
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        void* const out = which ? p.dshift : p.dgain;
        if (out == nullptr) continue;
        if (p.p_dtype == ICSA_DT_F32) store8(reinterpret_cast<float*>(out) + at, which ? db[u] : da[u], n[u], false);
        else store8(reinterpret_cast<bf16*>(out) + at, which ? db[u] : da[u], n[u], false);
      }
    }
    return;
  }
  // this workgroup's sums: [group][workgroup][da, db][dim padded to 4]
  float* part = p.part + ((int64_t)g * gridDim.x + blockIdx.x) * 2 * p.dim4;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int u = 0; u < NCH; ++u)
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        if (e < n[u]) {                               // whole fours: dim4 is padded
          const int at = 8 * (t + u * lanes) + e;
          *reinterpret_cast<floatx4*>(part + at) = floatx4{da[u][e], da[u][e + 1], da[u][e + 2], da[u][e + 3]};
          *reinterpret_cast<floatx4*>(part + p.dim4 + at) = floatx4{db[u][e], db[u][e + 1], db[u][e + 2], db[u][e + 3]};
        }
  } else {                                            // the workgroup's rows side by side, added in their order
    __shared__ float all[kRows][8 * NCH * (LPR == 0 ? 1 : LPR)];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < NCH; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) all[sub][8 * (t + u * lanes) + e] = which ? db[u][e] : da[u][e];
      __syncthreads();
      for (int d = threadIdx.x; d < p.dim; d += NM_THREADS) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < kRows; ++i) s += all[i][d];
        part[which * p.dim4 + d] = s;
      }
    }
  }
}

// Backward of few rows in one launch: a workgroup takes NM_FEW_COLS columns of a group's rows, the sums over whole rows for itself, a
// row a wave, and adds its columns' da and db over the rows in their order.  One launch and no workspace, 4 us of the host's time, against the two
// kernels' time: 8 rows of 5,120 f32 elements 10.4 us and 8.4 with a launch between them, of 1,536 6.4 and 6.6, of 128 4.9 and 5.0; 16 rows
// of 5,120 16.3 and 8.6.
template <typename TX, typename TY, bool RMS>
__global__ void __launch_bounds__(NM_FEW_COLS) icsa_norm_bwd_few_kernel(NormParams p) {
  __shared__ float sums[NM_FEW_TOTAL][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = blockIdx.y, rows = (int)p.rows;
  const int64_t row0 = (int64_t)g * p.rows;
  const TX* x = reinterpret_cast<const TX*>(p.x) + row0 * p.x_ss;
  const TY* dy = reinterpret_cast<const TY*>(p.dy) + row0 * p.dy_ss;
  if (p.dx != nullptr) {
    for (int r = wave; r < rows; r += NM_FEW_COLS / 64) {
      const float mean = RMS ? 0.f : p.mean[row0 + r], rstd = p.rstd[row0 + r];
      float s0 = 0.f, s1 = 0.f;
#pragma unroll 4
      for (int d = 8 * lane; d < p.dim; d += 512) {
        const int n[1] = {p.dim - d};
        Raw8<TX> vx;
        Raw8<TY> vy;
        float a[1][8];
        vx.load(x + r * p.x_ss + d, n[0], p.vec_x);
        vy.load(dy + r * p.dy_ss + d, n[0], p.vec_y);
        load_params<1>(p, p.gain, g * p.p_sg + d, 0, 0, a, n, 1.f, p.plus_one ? 1.f : 0.f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float u = vy.at(e) * a[0][e];         // 0 past the row's end
          s0 = fmaf(u, e < n[0] ? (vx.at(e) - mean) * rstd : 0.f, s0);
          s1 += u;
        }
      }
      s0 = lanes_sum<64>(s0);
      s1 = lanes_sum<64>(s1);
      if (lane == 0) { sums[r][0] = s0; sums[r][1] = s1; }
    }
    __syncthreads();
  }
  const int d = blockIdx.x * NM_FEW_COLS + threadIdx.x;
  if (d >= p.dim) return;
  const float inv_n = 1.f / (float)p.dim;
  const int64_t at = g * p.p_sg + d;
  const float a = p.gain == nullptr ? 1.f : (p.plus_one ? 1.f : 0.f) + (p.p_dtype == ICSA_DT_F32 ? reinterpret_cast<const float*>(p.gain)[at] :
                                                                        (float)reinterpret_cast<const bf16*>(p.gain)[at]);
  float da = 0.f, db = 0.f;
#pragma unroll 4
  for (int r = 0; r < rows; ++r) {
    const float mean = RMS ? 0.f : p.mean[row0 + r], rstd = p.rstd[row0 + r];
    const float v = (float)dy[r * p.dy_ss + d], xh = ((float)x[r * p.x_ss + d] - mean) * rstd;
    da = fmaf(v, xh, da);
    db += v;
    if (p.dx != nullptr) {
      const float m1 = sums[r][0] * inv_n, m0 = RMS ? 0.f : sums[r][1] * inv_n;
      reinterpret_cast<TX*>(p.dx)[(row0 + r) * p.dx_ss + d] = (TX)(rstd * (v * a - m0 - xh * m1));
    }
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    void* const out = which ? p.dshift : p.dgain;
    if (out == nullptr) continue;
    if (p.p_dtype == ICSA_DT_F32) reinterpret_cast<float*>(out)[(int64_t)g * p.dim + d] = which ? db : da;
    else reinterpret_cast<bf16*>(out)[(int64_t)g * p.dim + d] = (bf16)(which ? db : da);
  }
}

// da and db of a group from its workgroups' sums: 64 columns a workgroup, 16 threads of 4 columns by 16 shares of the parts
__global__ void __launch_bounds__(256) icsa_norm_join_kernel(NormParams p) {
  __shared__ __attribute__((aligned(16))) float all[16][64];
  const int c = threadIdx.x & 15, share = threadIdx.x >> 4, which = blockIdx.y, g = blockIdx.z;
  void* const out = which ? p.dshift : p.dgain;
  if (out == nullptr) return;
  const int at = blockIdx.x * 64 + 4 * c;
  floatx4 s = {};
  if (at < p.dim4) {
    const float* src = p.part + ((int64_t)g * p.n_wg * 2 + which) * p.dim4 + at;
#pragma unroll 8
    for (int i = share; i < p.n_wg; i += 16) {
      const floatx4 v = *reinterpret_cast<const floatx4*>(src + (int64_t)i * 2 * p.dim4);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += v[e];
    }
  }
  *reinterpret_cast<floatx4*>(&all[share][4 * c]) = s;
  __syncthreads();
  const int d = blockIdx.x * 64 + threadIdx.x;
  if (threadIdx.x >= 64 || d >= p.dim) return;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += all[i][threadIdx.x];
  if (p.p_dtype == ICSA_DT_F32) reinterpret_cast<float*>(out)[(int64_t)g * p.dim + d] = sum;
  else reinterpret_cast<bf16*>(out)[(int64_t)g * p.dim + d] = (bf16)sum;
}

namespace {

// Threads of a row: a quarter wave, a wave, four waves with one to three chunks a thread, or eight with two.  Other counts of waves
// leave the SIMDs unequal work: 5,120 elements (28,080 bf16 rows) by 320 threads of two whole chunks 134 us forward and 287 back, by
// 256 of three, the last half empty, 122 and 185; 8,192 elements (20,000 rows) by 256 of four 180 and 270, by 512 of two 134 and 231.
int threads_of(int dim) { return dim <= 256 ? 16 : dim <= 1024 ? 64 : dim <= 6144 ? 256 : 512; }

// Workgroups that a group of rows is dealt to, over all groups, as few as leave no round incomplete by much: three waves a SIMD
// forward (5,120 f32 elements, 65,520 rows: 394 us, with four 414; 1,000 bf16 elements, 40,000 rows: 40 and 44), four where a row
// takes eight waves (8,192 elements: 134 us, with three 155); four back, two where their registers leave no more (28,080
// rows of 5,120: 185, with one and a half 214).  Few rows of a group back: one workgroup, which needs no second kernel for the parameters' gradients (2 rows of 1,536: 4.9 us).
int workgroups(int64_t rows, int dim, int groups, bool back) {
  const int t = threads_of(dim), waves = t <= 64 ? 4 : t / 64;
  const int64_t per = t <= 64 ? NM_THREADS / t : 1, n = (rows + per - 1) / per;
  if (back && per == 1 && n <= NM_FEW_ROWS) return 1;
  const int a_simd = back ? (dim > 4096 ? 2 : 4) : dim > 6144 ? 4 : 3, most = NM_WAVES * a_simd / waves;
  const int64_t cap = most / groups > 0 ? most / groups : 1, rounds = (n + cap - 1) / cap;
  return (int)((n + rounds - 1) / (rounds > 0 ? rounds : 1));
}

template <typename TX, typename TY, bool RMS, int LPR, int NCH>
void go(const NormParams& p, bool back, hipStream_t stream) {
  const dim3 grid(p.n_wg, p.groups), threads(LPR == 0 ? threads_of(p.dim) : NM_THREADS);
  if (back) hipLaunchKernelGGL((icsa_norm_bwd_kernel<TX, TY, RMS, LPR, NCH>), grid, threads, 0, stream, p);
  else hipLaunchKernelGGL((icsa_norm_fwd_kernel<TX, TY, RMS, LPR, NCH>), grid, threads, 0, stream, p);
}

template <typename TX, typename TY, bool RMS>
void by_size(const NormParams& p, bool back, hipStream_t stream) {
  const int n = p.dim;
  if (back && norm_bwd_few(p.rows, p.groups))
    hipLaunchKernelGGL((icsa_norm_bwd_few_kernel<TX, TY, RMS>), dim3((n + NM_FEW_COLS - 1) / NM_FEW_COLS, p.groups), dim3(NM_FEW_COLS), 0, stream, p);
  else if (n <= 128) go<TX, TY, RMS, 16, 1>(p, back, stream);
  else if (n <= 256) go<TX, TY, RMS, 16, 2>(p, back, stream);
  else if (n <= 512) go<TX, TY, RMS, 64, 1>(p, back, stream);
  else if (n <= 1024) go<TX, TY, RMS, 64, 2>(p, back, stream);
  else if (n <= 2048) go<TX, TY, RMS, 0, 1>(p, back, stream);
  else if (n <= 4096 || n > 6144) go<TX, TY, RMS, 0, 2>(p, back, stream);
  else go<TX, TY, RMS, 0, 3>(p, back, stream);
}

template <bool RMS>
void by_type(const NormParams& p, bool back, hipStream_t stream) {
  const bool x32 = p.x_dtype == ICSA_DT_F32, y32 = p.y_dtype == ICSA_DT_F32;
  if (x32) return y32 ? by_size<float, float, RMS>(p, back, stream) : by_size<float, bf16, RMS>(p, back, stream);
  return y32 ? by_size<bf16, float, RMS>(p, back, stream) : by_size<bf16, bf16, RMS>(p, back, stream);
}

hipError_t run_norm(const NormParams& p, bool back, hipStream_t stream) {
  if (p.rms) by_type<true>(p, back, stream);
  else by_type<false>(p, back, stream);
  return hipGetLastError();
}

}  // namespace

bool norm_bwd_few(int64_t rows, int groups) { return rows * groups <= NM_FEW_TOTAL; }

int norm_bwd_workgroups(int64_t rows, int dim, int groups) { return workgroups(rows, dim, groups, true); }

hipError_t launch_norm_fwd(NormParams p, hipStream_t stream) {
  p.n_wg = workgroups(p.rows, p.dim, p.groups, false);
  return run_norm(p, false, stream);
}

hipError_t launch_norm_bwd(NormParams p, hipStream_t stream) {
  p.n_wg = norm_bwd_workgroups(p.rows, p.dim, p.groups);
  if (norm_bwd_few(p.rows, p.groups)) p.part = nullptr;
  if (p.n_wg == 1 && threads_of(p.dim) > 64) p.part = nullptr;      // written by the workgroup itself
  const hipError_t e = run_norm(p, true, stream);
  if (e != hipSuccess || p.part == nullptr) return e;
  hipLaunchKernelGGL(icsa_norm_join_kernel, dim3((p.dim + 63) / 64, 2, p.groups), dim3(256), 0, stream, p);
  return hipGetLastError();
}
