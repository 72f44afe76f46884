// Product of microscaled 4-bit operands: y[m][n] = act(sum_k x[m][k] w[n][k] + bias[n]).
//
// v_mfma_scale_f32_32x32x64_f8f6f4 takes one block of 32 codes (16 bytes) and its scale byte from
// each lane: lane l holds row l % 32, and k block l / 32 of the two that a step covers.  Which two blocks
// of a row's group of eight go together is free as long as both operands agree: step s takes
// blocks s (lanes 0-31) and 4 + s (lanes 32-63), so that a lane's four scale bytes of a group are
// one aligned dword of the scale layout, picked by the instruction's own byte select.
//
// The weights are the A operand: a lane then holds one token (accumulator column) and, of every 32
// outputs, 4 groups of 4 consecutive ones.
//
// A workgroup of 4 waves computes TN x TM outputs (n x m); tiles of one group (256 k, a full
// 128-byte line of every row) arrive by direct global->LDS loads, two buffers.  16-byte chunk c of tile row r
// sits at chunk c ^ (r / 2 % 8): 16 consecutive rows' reads of one chunk touch every bank once.
// A group is 4 steps.  The operands of step s + 1 are read while step s multiplies; the wait for the
// next group and the barrier come before the last step's products, whose operands are in registers by then, so
// the matrix pipe runs through them, and the tile after next can overwrite the buffer at once.
#include "attn_tile.h"
#include "icsa_kernels.h"
#include "mx_common.h"

#define MXG_THREADS 256
#define MXG_LINE 128                                   // bytes of codes of one row and group

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// byte `kSel` of each scale register, both operands e2m1 (format 4)
template <int kSel>
__device__ __forceinline__ floatx16 mx_mfma(i32x4 a, i32x4 b, floatx16 c, int sa, int sb) {
  const i32x8 a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, kSel, sa, kSel, sb);
}

__device__ __forceinline__ int mxg_off(int row, int chunk) {           // bytes in a code tile
  return row * MXG_LINE + ((chunk ^ ((row >> 1) & 7)) << 4);
}

// gelu(t) = t / (1 + exp(-2 sqrt(2 / pi) (t + 0.044715 t^3))): no difference of near values on
// either side of zero.  exp2 of a large argument is infinity and the quotient 0.
__device__ __forceinline__ float gelu_tanh(float t) {
  const float u = t * fmaf(0.044715f * t, t, 1.f);
  return t / (1.f + __builtin_amdgcn_exp2f(u * (-2.f * 0.7978845608028654f * 1.4426950408889634f)));
}

// LDS DMA with a uniform byte offset
__device__ __forceinline__ void lds_dma16s(unsigned lds_addr, int voff, u32x4 rs, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :: "s"(lds_addr), "v"(voff), "s"(rs), "s"(soff) : "memory", "m0");
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

// One 32 (n) x 32 (m) accumulator tile: bias, activation, and the row's outputs in the asked type.
// n0: its first output; m: this lane's token.
template <int kOut>
__device__ __forceinline__ void store_tile(const MxGemmParams& p, const floatx16& acc, int n0, int m, const float* bias) {
  const int hl = (threadIdx.x & 63) >> 5;
  float v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    v[i] = acc[i] + bias[i];
    if (p.gelu) v[i] = gelu_tanh(v[i]);
  }
  if constexpr (kOut == MX_OUT_MXFP4) {
    const int Np = mx_padded(p.N);
    unsigned amax = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (n0 + 8 * (i >> 2) + 4 * hl + (i & 3) >= p.N) v[i] = 0.f;       // the padding: zeros
      amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    const auto w = __builtin_amdgcn_permlane32_swap(amax, amax, false, false);
    const unsigned s = mx_scale_byte(max(w[0], w[1]));
    const float f = mx_inv_scale(s);
    unsigned q[2];                                     // 4 groups of 4 codes: 16 bits each
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
    const unsigned lo = x[0], hi = x[1];               // this half's codes of groups 2 hl, 2 hl + 1: from hl = 0, 1
    const u32x2 c = {(lo & 0xffffu) | hi << 16, lo >> 16 | (hi & 0xffff0000u)};
    if (m < p.M && n0 < Np) {
      unsigned char* row = reinterpret_cast<unsigned char*>(p.out) + (int64_t)m * p.o_ss;
      *reinterpret_cast<u32x2*>(row + n0 / 2 + 8 * hl) = c;
      if (hl == 0)
        p.out_scales[((int64_t)(n0 / MX_GROUP) * p.M + m) * MX_GROUP_BLOCKS + n0 / MX_BLOCK % MX_GROUP_BLOCKS] = (unsigned char)s;
    }
  } else {
    if (m >= p.M) return;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int n = n0 + 8 * g + 4 * hl;
      if constexpr (kOut == MX_OUT_F32) {
        float* dst = reinterpret_cast<float*>(p.out) + (int64_t)m * p.o_ss + n;
        if (n + 4 <= p.N && (p.o_ss & 3) == 0) *reinterpret_cast<floatx4*>(dst) = floatx4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) if (n + e < p.N) dst[e] = v[4 * g + e];
      } else {
        bf16* dst = reinterpret_cast<bf16*>(p.out) + (int64_t)m * p.o_ss + n;
        bf16x4 b;
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = (bf16)v[4 * g + e];
        if (n + 4 <= p.N && (p.o_ss & 3) == 0) *reinterpret_cast<bf16x4*>(dst) = b;
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) if (n + e < p.N) dst[e] = b[e];
      }
    }
  }
}

}  // namespace

// WN x WM accumulator tiles of 32 x 32 a wave, waves 2 x 2: TN = 64 WN outputs, TM = 64 WM tokens
template <int WN, int WM, int kOut>
__global__ void __launch_bounds__(MXG_THREADS) icsa_mx_gemm_kernel(MxGemmParams p) {
  constexpr int TN = 64 * WN, TM = 64 * WM;
  constexpr int kCodes = (TN + TM) * MXG_LINE, kBuf = kCodes + (TN + TM) * MX_GROUP_BLOCKS;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, li = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave >> 1, wm = wave & 1;

  // tile order: 8 token tiles at a time, output tiles outermost among them: the 32 workgroups that an
  // XCD runs together read 8 token tiles and 4 weight tiles
  const int tiles_n = (out_columns(p) + TN - 1) / TN, tiles_m = (p.M + TM - 1) / TM;
  const int w = xcd_remap(blockIdx.x, tiles_n * tiles_m);
  if (w < 0) return;
  const int band = w / (8 * tiles_n), in_band = w - band * 8 * tiles_n;
  const int rows = min(8, tiles_m - band * 8);
  const int m0 = (band * 8 + in_band % rows) * TM, n0 = in_band / rows * TN;

  // ---- loads: 8 rows of codes an instruction, 128 rows of scales an instruction ----
  const int64_t line = (int64_t)p.groups * MXG_LINE;                   // bytes of a row of codes
  const u32x4 rs_w = dma_rsrc(p.w + n0 * line, min(TN, p.N - n0) * line);
  const u32x4 rs_x = dma_rsrc(p.x + m0 * line, min(TM, p.M - m0) * line);
  const unsigned lds0 = lds_u32(smem);
  constexpr int kRowsW = TN / 4, kRowsX = TM / 4;                      // rows of each tile that a wave loads
  auto code_off = [&](int row) { return (int)(row * line) + (((lane & 7) ^ ((row >> 1) & 7)) << 4); };
  auto load_group = [&](int g, int buf) __attribute__((always_inline)) {
    const unsigned base = lds0 + buf * kBuf;
#pragma unroll
    for (int i = 0; i < kRowsW / 8; ++i) {
      const int r = wave * kRowsW + 8 * i;
      lds_dma16s(base + r * MXG_LINE, code_off(r + (lane >> 3)), rs_w, g * MXG_LINE);
    }
#pragma unroll
    for (int i = 0; i < kRowsX / 8; ++i) {
      const int r = wave * kRowsX + 8 * i;
      lds_dma16s(base + (TN + r) * MXG_LINE, code_off(r + (lane >> 3)), rs_x, g * MXG_LINE);
    }
    // scales: waves 0, 1 the weights', waves 2, 3 the tokens', half a tile each, 4 bytes a lane and load
    const bool tok = wave >= 2;
    const int R = tok ? p.M : p.N, r0 = tok ? m0 : n0, T = tok ? TM : TN;
    const u32x4 rs = dma_rsrc((tok ? p.x_scales : p.w_scales) + ((int64_t)g * R + r0) * MX_GROUP_BLOCKS,
                              (int64_t)min(T, R - r0) * MX_GROUP_BLOCKS);
    const int at = (wave & 1) * (T / 2) * MX_GROUP_BLOCKS;
#pragma unroll
    for (int i = 0; i < (TN > TM ? TN : TM) / 2 * MX_GROUP_BLOCKS / 256; ++i)
      if (i < T / 2 * MX_GROUP_BLOCKS / 256)
        lds_dma4(base + kCodes + (tok ? TN * MX_GROUP_BLOCKS : 0) + at + 256 * i, at + 256 * i + 4 * lane, rs);
  };

  floatx16 acc[WN][WM] = {};
  i32x4 a[2][WN], b[2][WM];
  int sa[2][WN], sb[2][WM];
  auto read_step = [&](int buf, int s, int to) __attribute__((always_inline)) {
    const unsigned char* t = smem + buf * kBuf;
#pragma unroll
    for (int i = 0; i < WN; ++i) a[to][i] = *reinterpret_cast<const i32x4*>(t + mxg_off((wn * WN + i) * 32 + li, 4 * hl + s));
#pragma unroll
    for (int j = 0; j < WM; ++j) b[to][j] = *reinterpret_cast<const i32x4*>(t + mxg_off(TN + (wm * WM + j) * 32 + li, 4 * hl + s));
  };
  auto read_scales = [&](int buf, int to) __attribute__((always_inline)) {
    const unsigned char* t = smem + buf * kBuf + kCodes + 4 * hl;
#pragma unroll
    for (int i = 0; i < WN; ++i) sa[to][i] = *reinterpret_cast<const int*>(t + ((wn * WN + i) * 32 + li) * MX_GROUP_BLOCKS);
#pragma unroll
    for (int j = 0; j < WM; ++j) sb[to][j] = *reinterpret_cast<const int*>(t + (TN + (wm * WM + j) * 32 + li) * MX_GROUP_BLOCKS);
  };
#define MXG_STEP(from, sel, ss)                                                              \
  _Pragma("unroll") for (int i = 0; i < WN; ++i) _Pragma("unroll") for (int j = 0; j < WM; ++j) \
      acc[i][j] = mx_mfma<sel>(a[from][i], b[from][j], acc[i][j], sa[ss][i], sb[ss][j]);

  load_group(0, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  ATT_BARRIER();
  if (p.groups > 1) load_group(1, 1);
  read_scales(0, 0);
  read_step(0, 0, 0);
  for (int g = 0; g < p.groups; ++g) {
    const int buf = g & 1;
    read_step(buf, 1, 1);
    MXG_STEP(0, 0, 0)
    read_step(buf, 2, 0);
    MXG_STEP(1, 1, 0)
    read_step(buf, 3, 1);
    MXG_STEP(0, 2, 0)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                   // group g + 1
    ATT_BARRIER();                                                     // everybody has read group g
    if (g + 2 < p.groups) load_group(g + 2, buf);
    if (g + 1 < p.groups) { read_step(buf ^ 1, 0, 0); read_scales(buf ^ 1, 1); }
    MXG_STEP(1, 3, 0)
#pragma unroll
    for (int i = 0; i < WN; ++i) sa[0][i] = sa[1][i];
#pragma unroll
    for (int j = 0; j < WM; ++j) sb[0][j] = sb[1][j];
  }
#pragma unroll
  for (int i = 0; i < WN; ++i) {
    const int n = n0 + (wn * WN + i) * 32;
    float bias[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) bias[e] = bias_at(p, n + 8 * (e >> 2) + 4 * hl + (e & 3));
#pragma unroll
    for (int j = 0; j < WM; ++j) store_tile<kOut>(p, acc[i][j], n, m0 + (wm * WM + j) * 32 + li, bias);
  }
#undef MXG_STEP
}

namespace {

template <int WN, int WM, int kOut>
hipError_t run_mx_gemm(const MxGemmParams& p, hipStream_t stream) {
  constexpr int TN = 64 * WN, TM = 64 * WM, kLds = 2 * (TN + TM) * (MXG_LINE + MX_GROUP_BLOCKS);
  static std::atomic<unsigned> lds_set{0u};
  const hipError_t e = ensure_lds_limit(reinterpret_cast<const void*>(icsa_mx_gemm_kernel<WN, WM, kOut>), kLds, &lds_set);
  if (e != hipSuccess) return e;
  const int64_t tiles = (int64_t)((out_columns(p) + TN - 1) / TN) * ((p.M + TM - 1) / TM);
  if (tiles > 0x7ffffff0LL) return hipErrorInvalidValue;
  hipLaunchKernelGGL((icsa_mx_gemm_kernel<WN, WM, kOut>), dim3(xcd_grid((int)tiles)), dim3(MXG_THREADS), kLds, stream, p);
  return hipGetLastError();
}

template <int kOut>
hipError_t pick_mx_gemm(const MxGemmParams& p, hipStream_t stream) {
  const int64_t big = (int64_t)((p.N + 255) / 256) * ((p.M + 255) / 256);
  if (big >= 256) return run_mx_gemm<4, 4, kOut>(p, stream);
  return run_mx_gemm<2, 2, kOut>(p, stream);
}

}  // namespace

hipError_t launch_mx_gemm(const MxGemmParams& p, hipStream_t stream) {
  // a tile's rows must be addressable with 32-bit offsets
  if ((int64_t)p.groups * MXG_LINE * 256 > 0x7fffffffLL) return hipErrorInvalidValue;
  switch (p.out_kind) {
    case MX_OUT_BF16: return pick_mx_gemm<MX_OUT_BF16>(p, stream);
    case MX_OUT_F32: return pick_mx_gemm<MX_OUT_F32>(p, stream);
    default: return pick_mx_gemm<MX_OUT_MXFP4>(p, stream);
  }
}
