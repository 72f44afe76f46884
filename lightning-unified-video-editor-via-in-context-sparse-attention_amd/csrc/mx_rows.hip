// The 4-bit product for few token rows: bound by the weights' bytes, so every weight is read once, straight into the
// matrix instruction's registers.
//
// A workgroup has 32 outputs and up to 32 MT tokens; its waves share the groups of k between them and add their
// sums through LDS in wave order (bitwise reproducible).  A lane reads 64 contiguous bytes of its weight row and of its token rows a
// group, the next group's while it multiplies (the token rows' without that: 1 x 30,720 x 5,120 21.6 us against 19.6, 64 x 5,120 x
// 13,824 24.2 against 22.8).  For up to MXR_RAW_ROWS rows of bf16 or f32 the workgroup quantises x itself into LDS:
// one launch instead of two.
#include "mx_tile.h"

#define MXR_RAW_ROWS 2
#define MXR_PAD 16                                     // bytes between rows of codes in LDS: other banks

namespace {

struct MxFrag {
  i32x4 c[4];                                          // codes of the four steps
  int s;                                               // their scale bytes
};

__device__ __forceinline__ MxFrag load_frag(const unsigned char* codes, const unsigned char* scales, int64_t line, int R, int r, int g, int hl) {
  MxFrag f;
  const i32x4* src = reinterpret_cast<const i32x4*>(codes + r * line + g * MXG_LINE + 64 * hl);
#pragma unroll
  for (int s = 0; s < 4; ++s) f.c[s] = src[s];
  f.s = *reinterpret_cast<const int*>(scales + ((int64_t)g * R + r) * MX_GROUP_BLOCKS + 4 * hl);
  return f;
}

}  // namespace

// most waves of a workgroup: two token tiles' operands, read a group ahead, need 154 registers
constexpr int mx_rows_waves(int mt) { return mt == 1 ? 16 : 8; }

// kSrc: x in 4 bits (0), bf16 (1) or f32 (2)
template <int MT, int kSrc, int kOut>
__global__ void __launch_bounds__(64 * mx_rows_waves(MT)) icsa_mx_rows_kernel(MxGemmParams p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, li = lane & 31, hl = lane >> 5, nw = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = blockIdx.x * 32, Kp = p.groups * MX_GROUP;
  const int64_t line = (int64_t)p.groups * MXG_LINE;
  const int wr = min(n0 + li, p.N - 1);                // rows past the last repeat it: their sums are not stored
  const int lds_line = (int)line + MXR_PAD;
  unsigned char* const xs = smem + p.M * lds_line;     // scales [group][row][8]
  float* const red = reinterpret_cast<float*>(smem + (kSrc != 0 ? (p.M * (lds_line + Kp / MX_BLOCK) + 15) / 16 * 16 : 0));

  auto weight_frag = [&](int g) { return load_frag(p.w, p.w_scales, line, p.N, wr, g, hl); };
  MxFrag wnext;
  if (wave < p.groups) wnext = weight_frag(wave);      // requested before x is quantised
  if constexpr (kSrc != 0) {
    const int per_row = Kp / 8;
    for (int u = threadIdx.x; u < p.M * per_row; u += blockDim.x) {      // 8 values; 4 lanes share a block
      const int m = u / per_row, k = u % per_row * 8;
      float v[8];
      if constexpr (kSrc == 1) load8_row<bf16>(reinterpret_cast<const bf16*>(p.x_raw) + m * p.x_ss, k, p.K, v);
      else load8_row<float>(reinterpret_cast<const float*>(p.x_raw) + m * p.x_ss, k, p.K, v);
      const unsigned s = mx_quantize8(v);
      *reinterpret_cast<unsigned*>(smem + m * lds_line + k / 2) = mx_codes8(v, s);
      if ((lane & 3) == 0) xs[(k / MX_GROUP * p.M + m) * MX_GROUP_BLOCKS + k / MX_BLOCK % MX_GROUP_BLOCKS] = (unsigned char)s;
    }
    __syncthreads();
  }
  auto token_frag = [&](int t, int gg) -> MxFrag {
    const int m = min(p.m_first + 32 * t + li, p.m_last - 1);
    if constexpr (kSrc == 0) return load_frag(p.x, p.x_scales, line, p.M, m, gg, hl);
    else return load_frag(smem, xs, lds_line, p.M, m, gg, hl);
  };
  floatx16 acc[MT] = {};
  MxFrag xnext[MT];
  if (wave < p.groups) {
#pragma unroll
    for (int t = 0; t < MT; ++t) xnext[t] = token_frag(t, wave);
  }
  for (int g = wave; g < p.groups; g += nw) {
    const MxFrag wf = wnext;
    MxFrag xf[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xf[t] = xnext[t];
    if (g + nw < p.groups) {
      wnext = weight_frag(g + nw);
#pragma unroll
      for (int t = 0; t < MT; ++t) xnext[t] = token_frag(t, g + nw);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      acc[t] = mx_mfma<0>(wf.c[0], xf[t].c[0], acc[t], wf.s, xf[t].s);
      acc[t] = mx_mfma<1>(wf.c[1], xf[t].c[1], acc[t], wf.s, xf[t].s);
      acc[t] = mx_mfma<2>(wf.c[2], xf[t].c[2], acc[t], wf.s, xf[t].s);
      acc[t] = mx_mfma<3>(wf.c[3], xf[t].c[3], acc[t], wf.s, xf[t].s);
    }
  }
  // ---- the waves' sums: [wave][token tile][quarter][lane][4] ----  a wave adds up one quarter of one tile
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<floatx4*>(red + (((wave * MT + t) * 4 + q) * 64 + lane) * 4) =
          floatx4{acc[t][4 * q], acc[t][4 * q + 1], acc[t][4 * q + 2], acc[t][4 * q + 3]};
  __syncthreads();
  auto total = [&](int t, int q) -> floatx4 {
    const float* src = red + ((t * 4 + q) * 64 + lane) * 4;
    floatx4 s = *reinterpret_cast<const floatx4*>(src);
    for (int v = 1; v < nw; ++v) {
      const floatx4 x = *reinterpret_cast<const floatx4*>(src + v * MT * 1024);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += x[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[e] += bias_at(p, n0 + 8 * q + 4 * hl + e);
      if (p.gelu) s[e] = gelu_tanh(s[e]);
    }
    return s;
  };
  if constexpr (kOut == MX_OUT_MXFP4) {
    if (wave >= MT) return;                            // a block's scale takes all of its 32 outputs
    float v[16];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const floatx4 s = total(wave, q);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * q + e] = s[e];
    }
    store_mx(p, v, n0, p.m_first + 32 * wave + li);
  } else {
    for (int u = wave; u < 4 * MT; u += nw) {
      const floatx4 s = total(u >> 2, u & 3);
      const int n = n0 + 8 * (u & 3) + 4 * hl, m = p.m_first + 32 * (u >> 2) + li;
      if (m >= p.m_last) continue;
      if constexpr (kOut == MX_OUT_F32) {
        float* dst = reinterpret_cast<float*>(p.out) + (int64_t)m * p.o_ss + n;
        if (n + 4 <= p.N) *reinterpret_cast<floatx4_a4*>(dst) = s;
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) if (n + e < p.N) dst[e] = s[e];
      } else {
        bf16* dst = reinterpret_cast<bf16*>(p.out) + (int64_t)m * p.o_ss + n;
        bf16x4 b;
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = (bf16)s[e];
        if (n + 4 <= p.N) *reinterpret_cast<bf16x4_a2*>(dst) = b;
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) if (n + e < p.N) dst[e] = b[e];
      }
    }
  }
}

// 30,720 x 5,120 with the quantisation in the call: 18.3 us at one row, 21.5 in two launches; 25.1 at four rows, 21.5 in two
bool mx_rows_takes_raw(int64_t M, int K) {
  return M <= MXR_RAW_ROWS && M * (mx_padded(K) / 2 + MXR_PAD + mx_padded(K) / MX_BLOCK) <= 64 * 1024;
}

namespace {

template <int MT, int kSrc, int kOut>
hipError_t run_mx_rows(const MxGemmParams& p, hipStream_t stream) {
  const int blocks = (out_columns(p) + 31) / 32;
  // waves: 16 a CU and more, not more than groups; 16 in a workgroup where each CU has one at most.  8 against 16 (us, codes in, 1 /
  // 16 / 32 rows): 13,824 x 5,120 10.7 / 13.2 / 16.2 to 12.0 / 13.7 / 16.1; 16,384 x 2,048 5.7 / 6.4 / 7.1 to 5.8 / 6.5 / 7.1.  Where
  // 16 are taken: 5,120 x 5,120 6.0 / 7.0 / 7.9 to 6.2 / 7.1 / 8.0 and 5,120 x 13,824 11.8 / 15.1 / 18.8 to 13.1 / 15.3 / 18.8 with
  // codes, two rows quantised in the call 7.2 to 6.8 and 15.1 to 15.4; 2,000 x 5,120 so 7.0 to 6.5.
  int nw = 4;
  while (nw < mx_rows_waves(MT) && blocks * nw < (nw < 8 ? 4096 : 2048) && nw < p.groups) nw *= 2;
  const int lds = nw * MT * 4096 + (kSrc != 0 ? p.M * (p.groups * (MXG_LINE + MX_GROUP_BLOCKS) + MXR_PAD) + 16 : 0);
  static std::atomic<unsigned> lds_set{0u};
  const hipError_t e = ensure_lds_limit(reinterpret_cast<const void*>(icsa_mx_rows_kernel<MT, kSrc, kOut>), 160 * 1024, &lds_set);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((icsa_mx_rows_kernel<MT, kSrc, kOut>), dim3(blocks), dim3(64 * nw), lds, stream, p);
  return hipGetLastError();
}

template <int kOut>
hipError_t pick_mx_rows(const MxGemmParams& p, hipStream_t stream) {
  if (p.x_raw != nullptr) {
    return p.x_dtype == ICSA_DT_F32 ? run_mx_rows<1, 2, kOut>(p, stream) : run_mx_rows<1, 1, kOut>(p, stream);
  }
  if (p.m_last - p.m_first <= 32) return run_mx_rows<1, 0, kOut>(p, stream);
  return run_mx_rows<2, 0, kOut>(p, stream);
}

}  // namespace

hipError_t launch_mx_rows(const MxGemmParams& p, hipStream_t stream) {
  switch (p.out_kind) {
    case MX_OUT_BF16: return pick_mx_rows<MX_OUT_BF16>(p, stream);
    case MX_OUT_F32: return pick_mx_rows<MX_OUT_F32>(p, stream);
    default: return pick_mx_rows<MX_OUT_MXFP4>(p, stream);
  }
}
