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
// A workgroup of 4 waves computes TN x TM outputs (n x m) over tiles of 128 k (64 bytes of every row), which arrive by
// direct global->LDS loads, three buffers.  16-byte chunk c of tile row r sits at chunk c ^ (r / 4 % 4): 16
// consecutive rows' reads of one chunk touch every bank once.  A tile is 2 steps.  The operands of a step are read
// while the one before multiplies; the wait for the next tile and the barrier come before the
// second step's products, whose operands are in registers by then, so the matrix pipe runs through them, and the
// freed buffer takes the tile three further on.  Two workgroups share a CU: one's waits, barriers and
// epilogue run beside the other's products.
#include <type_traits>

#include "attn_tile.h"
#include "icsa_kernels.h"
#include "mx_common.h"

#define MXG_THREADS 256
#define MXG_ROW 64                                     // bytes of codes of a tile row (128 k)
#define MXG_BUFS 3

namespace {

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

// Rows may start at any element: vectors of the element's alignment (global memory takes them)
typedef u32x4 u32x4_a2 __attribute__((aligned(2)));
typedef floatx4 floatx4_a4 __attribute__((aligned(4)));

// bias and activation of one 32 (n) x 32 (m) accumulator tile
__device__ __forceinline__ void tile_values(const MxGemmParams& p, const floatx16& acc, const float* bias, float v[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = acc[i] + bias[i];
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
  if (m < p.M && n0 < Np) {
    *reinterpret_cast<u32x2*>(reinterpret_cast<unsigned char*>(p.out) + (int64_t)m * p.o_ss + n0 / 2 + 8 * hl) = c;
    if (hl == 0)
      p.out_scales[((int64_t)(n0 / MX_GROUP) * p.M + m) * MX_GROUP_BLOCKS + n0 / MX_BLOCK % MX_GROUP_BLOCKS] = (unsigned char)s;
  }
}

__device__ __forceinline__ void store_f32(const MxGemmParams& p, const float v[16], int n0, int m) {
  const int hl = (threadIdx.x & 63) >> 5;
  if (m >= p.M) return;
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

// bf16 rows pass through 4 KB of the wave's LDS, 64 outputs of 32 tokens at a time, so that a store
// instruction writes 8 full lines of 128 bytes.  16-byte chunk c of row r at c ^ (r / 2 % 8).
__device__ __forceinline__ void stage_bf16(unsigned char* stage, const float v[16], int i) {
  const int lane = threadIdx.x & 63, li = lane & 31, hl = lane >> 5;
#pragma unroll
  for (int pr = 0; pr < 2; ++pr) {                     // lane halves swap: outputs 8 (2 pr + hl) .. + 7
    bf16x4 lo, hi;
#pragma unroll
    for (int e = 0; e < 4; ++e) { lo[e] = (bf16)v[8 * pr + e]; hi[e] = (bf16)v[8 * pr + 4 + e]; }
    const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
    const auto w0 = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false);
    const auto w1 = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
    *reinterpret_cast<u32x4*>(stage + li * 128 + (((4 * i + 2 * pr + hl) ^ ((li >> 1) & 7)) << 4)) = u32x4{w0[0], w1[0], w0[1], w1[1]};
  }
}
__device__ __forceinline__ void store_staged(const MxGemmParams& p, const unsigned char* stage, int n0, int m0) {
  const int lane = threadIdx.x & 63, n = n0 + 8 * (lane & 7);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const int r = 8 * x + (lane >> 3), m = m0 + r;
    const u32x4 c = *reinterpret_cast<const u32x4*>(stage + r * 128 + (((lane & 7) ^ ((r >> 1) & 7)) << 4));
    bf16* dst = reinterpret_cast<bf16*>(p.out) + (int64_t)m * p.o_ss + n;
    if (m < p.M && n + 8 <= p.N) *reinterpret_cast<u32x4_a2*>(dst) = c;
    else if (m < p.M) {
      const bf16x8 b = __builtin_bit_cast(bf16x8, c);
#pragma unroll
      for (int e = 0; e < 8; ++e) if (n + e < p.N) dst[e] = b[e];
    }
  }
}

}  // namespace

// WN x WM accumulator tiles of 32 x 32 a wave, waves 2 x 2: TN = 64 WN outputs, TM = 64 WM tokens
template <int WN, int WM, int kOut>
__global__ void __launch_bounds__(MXG_THREADS, 2) icsa_mx_gemm_kernel(MxGemmParams p) {
  constexpr int TN = 64 * WN, TM = 64 * WM, kBuf = (TN + TM) * MXG_ROW, kScales = (TN + TM) * MX_GROUP_BLOCKS;
  constexpr int kLoads = (TN + TM) / 64;                               // code loads of a wave and tile: 16 rows each
  constexpr int kScaleLoads = (TN + TM) / 128;                         // scale loads of a wave and group: 32 rows each
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, li = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave >> 1, wm = wave & 1;

  // tile order: 8 token tiles at a time, output tiles outermost among them: the workgroups that an
  // XCD runs together share few token and weight tiles
  const int tiles_n = (out_columns(p) + TN - 1) / TN, tiles_m = (p.M + TM - 1) / TM;
  const int w = xcd_remap(blockIdx.x, tiles_n * tiles_m);
  if (w < 0) return;
  const int band = w / (8 * tiles_n), in_band = w - band * 8 * tiles_n;
  const int rows = min(8, tiles_m - band * 8);
  const int m0 = (band * 8 + in_band % rows) * TM, n0 = in_band / rows * TN;

  // ---- loads ----  rows are checked by the resources' ranges (in the lane's offset alone: k, which is
  // always inside a row, is the scalar offset)
  const int64_t line = (int64_t)p.groups * (MX_GROUP / 2);             // bytes of a row of codes
  const u32x4 rs_w = dma_rsrc(p.w + n0 * line, min(TN, p.N - n0) * line);
  const u32x4 rs_x = dma_rsrc(p.x + m0 * line, min(TM, p.M - m0) * line);
  const unsigned lds0 = lds_u32(smem), lds_scales = lds0 + MXG_BUFS * kBuf;
  const int lr = lane >> 2, lchunk = ((lane & 3) ^ ((lr >> 2) & 3)) << 4;
  int ofs[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i)
    ofs[i] = (int)(((i < WN ? wave * 16 * WN + 16 * i : wave * 16 * WM + 16 * (i - WN)) + lr) * line) + lchunk;
  const int n_tiles = 2 * p.groups;
  // past the last tile: an empty range, into a buffer that nobody reads any more
  auto load_codes = [&](int t, unsigned buf, int i) __attribute__((always_inline)) {
    const bool is_w = i < WN;
    u32x4 rs = is_w ? rs_w : rs_x;
    rs[2] = t < n_tiles ? rs[2] : 0;
    const int row = is_w ? wave * 16 * WN + 16 * i : TN + wave * 16 * WM + 16 * (i - WN);
    lds_dma16s(buf + row * MXG_ROW, ofs[i], rs, t * MXG_ROW);
  };
  // a group's scales, with its first tile: 32 rows a load (4 bytes a lane: the range ends at a row, 8 bytes)
  unsigned long long s_ptr[kScaleLoads];
  unsigned s_len[kScaleLoads], s_step[kScaleLoads];
#pragma unroll
  for (int i = 0; i < kScaleLoads; ++i) {
    const int at = 32 * (wave * kScaleLoads + i);
    const bool tok = at >= TN;
    const int R = tok ? p.M : p.N, r0 = tok ? m0 + at - TN : n0 + at;
    const u32x4 rs = dma_rsrc((tok ? p.x_scales : p.w_scales) + (int64_t)r0 * MX_GROUP_BLOCKS, (int64_t)min(32, R - r0) * MX_GROUP_BLOCKS);
    s_ptr[i] = (unsigned long long)rs[1] << 32 | rs[0];
    s_len[i] = rs[2];
    s_step[i] = (unsigned)R * MX_GROUP_BLOCKS;
  }
  auto load_scales = [&](int g, int i) __attribute__((always_inline)) {      // called for g = 0, 1, 2, ...
    const u32x4 rs = {(unsigned)s_ptr[i], (unsigned)(s_ptr[i] >> 32), g < p.groups ? s_len[i] : 0, 0x00020000u};
    lds_dma4(lds_scales + (g & 1) * kScales + 256 * (wave * kScaleLoads + i), 4 * lane, rs);
    s_ptr[i] += s_step[i];
  };

  floatx16 acc[WN][WM] = {};
  i32x4 a[2][WN], b[2][WM];
  u32x2 ga[WN], gb[WM];                                                // a group's scales
  int sa[WN], sb[WM];                                                  // a tile's: bytes 0, 1 for steps 0, 1
  int rd[2];                                                           // operand read offsets of steps 0, 1; + 32 rows a sub-tile
#pragma unroll
  for (int s = 0; s < 2; ++s) rd[s] = li * MXG_ROW + (((2 * hl + s) ^ ((li >> 2) & 3)) << 4);
  const unsigned char* base = smem;                                    // of the tile that is read
  auto read_a = [&](int s, int i) { a[s][i] = *reinterpret_cast<const i32x4*>(base + rd[s] + (wn * WN + i) * 32 * MXG_ROW); };
  auto read_b = [&](int s, int j) { b[s][j] = *reinterpret_cast<const i32x4*>(base + rd[s] + (TN + (wm * WM + j) * 32) * MXG_ROW); };
  auto read_scales = [&](int g) __attribute__((always_inline)) {
    const unsigned char* t = smem + MXG_BUFS * kBuf + (g & 1) * kScales + li * MX_GROUP_BLOCKS;
#pragma unroll
    for (int i = 0; i < WN; ++i) ga[i] = *reinterpret_cast<const u32x2*>(t + (wn * WN + i) * 32 * MX_GROUP_BLOCKS);
#pragma unroll
    for (int j = 0; j < WM; ++j) gb[j] = *reinterpret_cast<const u32x2*>(t + (TN + (wm * WM + j) * 32) * MX_GROUP_BLOCKS);
  };
  auto tile_scales = [&](int half) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < WN; ++i) sa[i] = (int)(ga[i][half] >> (16 * hl));
#pragma unroll
    for (int j = 0; j < WM; ++j) sb[j] = (int)(gb[j][half] >> (16 * hl));
  };

  unsigned cur = 0, nxt = kBuf, nn = 2 * kBuf;                         // buffers of tiles t, t + 1, t + 2
#pragma unroll
  for (int t = 0; t < 3; ++t) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_codes(t, lds0 + t * kBuf, i);
    if ((t & 1) == 0)
#pragma unroll
      for (int i = 0; i < kScaleLoads; ++i) load_scales(t >> 1, i);
  }
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"(2 * kLoads + kScaleLoads) : "memory");   // tile 0
  ATT_BARRIER();
  read_scales(0);
#pragma unroll
  for (int i = 0; i < WN; ++i) read_a(0, i);
#pragma unroll
  for (int j = 0; j < WM; ++j) read_b(0, j);
  // one tile: kHalf 0 or 1 of its group
  auto tile_pass = [&](auto half_c, int t) __attribute__((always_inline)) {
    constexpr int kHalf = decltype(half_c)::value;
    tile_scales(kHalf);
    // step 0; the operands of step 1 are read meanwhile
#pragma unroll
    for (int x = 0; x < WN * WM; ++x) {
      if (x < WN) read_a(1, x);
      else if (x < WN + WM) read_b(1, x - WN);
      if (WN * WM < WN + WM && x == WN * WM - 1) {                     // fewer products than operands
#pragma unroll
        for (int y = WN * WM; y < WN + WM; ++y) read_b(1, y - WN);
      }
      __builtin_amdgcn_sched_barrier(0);
      acc[x / WM][x % WM] = mx_mfma<0>(a[0][x / WM], b[0][x % WM], acc[x / WM][x % WM], sa[x / WM], sb[x % WM]);
      __builtin_amdgcn_sched_barrier(0);
    }
    // tile t + 1 is there when the loads of t + 2 alone are left (with its group's scales if t is even)
    if (kHalf == 0) asm volatile("s_waitcnt vmcnt(%0)" :: "n"(kLoads + kScaleLoads) : "memory");
    else asm volatile("s_waitcnt vmcnt(%0)" :: "n"(kLoads) : "memory");
    ATT_BARRIER();                                                     // everybody's; and everybody has read tile t
    base = smem + nxt;
    if (kHalf == 1) read_scales((t + 1) >> 1);
    // step 1; the operands of the next tile's step 0 are read and tile t + 3 is requested meanwhile
#pragma unroll
    for (int x = 0; x < WN * WM; ++x) {
      if (x < WN) read_a(0, x);
      else if (x < WN + WM) read_b(0, x - WN);
      if (WN * WM < WN + WM && x == WN * WM - 1) {
#pragma unroll
        for (int y = WN * WM; y < WN + WM; ++y) read_b(0, y - WN);
      }
      if (kHalf == 1 && x < kScaleLoads) load_scales((t + 3) >> 1, x);
      if (x < kLoads) load_codes(t + 3, lds0 + cur, x);
      if (x == WN * WM - 1) {
#pragma unroll
        for (int y = WN * WM; y < kLoads; ++y) load_codes(t + 3, lds0 + cur, y);
      }
      __builtin_amdgcn_sched_barrier(0);
      acc[x / WM][x % WM] = mx_mfma<1>(a[1][x / WM], b[1][x % WM], acc[x / WM][x % WM], sa[x / WM], sb[x % WM]);
      __builtin_amdgcn_sched_barrier(0);
    }
    const unsigned done = cur;
    cur = nxt; nxt = nn; nn = done;
  };
  for (int t = 0; t < n_tiles; t += 2) {
    tile_pass(std::integral_constant<int, 0>{}, t);
    tile_pass(std::integral_constant<int, 1>{}, t + 1);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                     // the empty loads
  ATT_BARRIER();                                                       // everybody's: the buffers are free
  float bias[WN][16];
#pragma unroll
  for (int i = 0; i < WN; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) bias[i][e] = bias_at(p, n0 + (wn * WN + i) * 32 + 8 * (e >> 2) + 4 * hl + (e & 3));
  unsigned char* const stage = smem + wave * 4096;
  static_assert(WN == 2, "64 outputs of a token are staged together");
#pragma unroll
  for (int j = 0; j < WM; ++j) {
    const int mt = m0 + (wm * WM + j) * 32;
#pragma unroll
    for (int i = 0; i < WN; ++i) {
      const int n = n0 + (wn * WN + i) * 32;
      float v[16];
      tile_values(p, acc[i][j], bias[i], v);
      if constexpr (kOut == MX_OUT_MXFP4) store_mx(p, v, n, mt + li);
      else if constexpr (kOut == MX_OUT_F32) store_f32(p, v, n, mt + li);
      else stage_bf16(stage, v, i);
    }
    if constexpr (kOut == MX_OUT_BF16) store_staged(p, stage, n0 + wn * 64, mt);
  }
}

namespace {

template <int WN, int WM, int kOut>
hipError_t run_mx_gemm(const MxGemmParams& p, hipStream_t stream) {
  constexpr int TN = 64 * WN, TM = 64 * WM, kLds = (TN + TM) * (MXG_BUFS * MXG_ROW + 2 * MX_GROUP_BLOCKS);
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
  const int64_t big = (int64_t)((p.N + 127) / 128) * ((p.M + 255) / 256);
  if (big >= 512) return run_mx_gemm<2, 4, kOut>(p, stream);
  return run_mx_gemm<2, 2, kOut>(p, stream);
}

}  // namespace

hipError_t launch_mx_gemm(const MxGemmParams& p, hipStream_t stream) {
  // a tile's rows must be addressable with 32-bit offsets
  if ((int64_t)p.groups * (MX_GROUP / 2) * 256 > 0x7fffffffLL) return hipErrorInvalidValue;
  switch (p.out_kind) {
    case MX_OUT_BF16: return pick_mx_gemm<MX_OUT_BF16>(p, stream);
    case MX_OUT_F32: return pick_mx_gemm<MX_OUT_F32>(p, stream);
    default: return pick_mx_gemm<MX_OUT_MXFP4>(p, stream);
  }
}
