// Product of microscaled 4-bit operands: y[m][n] = act(sum_k x[m][k] w[n][k] + bias[n]).
//
// A workgroup computes tiles of TN x TM outputs (n x m) over groups of 256 k, a full 128-byte line of every row, which arrive by
// direct global->LDS loads.  16-byte chunk c of tile row r sits at chunk c ^ (r / 2 % 8): 16 consecutive rows' reads of one chunk
// touch every bank once.  A group is 4 steps of 64 k.  The operands of a step are read from LDS while the one before
// multiplies; the wait for the next group and the barrier come before the last step's products, whose operands are in
// registers by then, so the matrix pipe runs through them, and the freed buffer takes the group kBufs further on, its loads spread
// over that step and the next.  The stream of groups runs across a workgroup's tiles: the next tile's first groups arrive
// while this one's outputs are written.
//
// What bounds it: the loads into LDS.  Timing copies of an earlier form (128 x 256 tiles of 128 k, two workgroups a CU, 14,040 x 5,120
// x 13,824): 553 us; without loads in the loop 379; with half of them 438; the same bytes in full 128-byte lines instead of
// halves 460.  So: full lines, and the largest tile (256 x 256, 8 waves of 64 x 128, two a SIMD): a third fewer bytes an
// operation, 478 us, 4.2 PFLOP/s; loads spread over two steps instead of one 454.  65,520 x 13,824 x 5,120 with GELU: 2.37 ms,
// 3.92 PFLOP/s, 2.7 times the bf16 library product's rate at this size (6.46 ms); 1.6 of a tile's 43 us are the GELU (two
// transcendentals an output, nothing to overlap them with); an earlier form without loads in the loop 2.16 ms.  4 waves of 128 x 128,
// a third fewer bytes out of LDS but one wave a SIMD, were slower: 14,040 x 5,120 x 13,824 538 us against 462.  (Times of pairs are of
// the form at hand when it was measured.)  Long k does better, 13,056 x 5,120 x 13,824 4.75 PFLOP/s: of a tile's 43 us with 20
// groups some 5 are the accumulators' start and the stores, when all waves are out of the loop at once.
#include <type_traits>

#include "mx_plan.h"
#include "mx_tile.h"

#define MXG_STAGE 2048                                 // bytes of output staging of a wave
#define MXG_BAND 4                                     // token tiles that go together in the order; 8: 5 % more time at 65,520 x 13,824 x 5,120

namespace {

// LDS DMA with a uniform byte offset
__device__ __forceinline__ void lds_dma16s(unsigned lds_addr, int voff, u32x4 rs, int soff) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :: "s"(lds_addr), "v"(voff), "s"(rs), "s"(soff) : "memory", "m0");
}

}  // namespace

// WN x WM accumulator tiles of 32 x 32 a wave, NN x NM waves: TN = 32 WN NN outputs, TM = 32 WM NM tokens
template <int WN, int WM, int NN, int NM, int kBufs, int kOut>
__global__ void __launch_bounds__(64 * NN * NM, 2) icsa_mx_gemm_kernel(MxGemmParams p) {
  constexpr int TN = 32 * WN * NN, TM = 32 * WM * NM, kWaves = NN * NM, kRows = TN + TM;
  constexpr int kCodes = kRows * MXG_LINE, kBuf = kCodes + kRows * MX_GROUP_BLOCKS;
  constexpr int kCodeLoads = kRows / 8 / kWaves;                       // of a wave and group: 8 rows each
  constexpr int kScaleLoads = kRows / 32 / kWaves;                     // 32 rows each
  constexpr int kLoads = kCodeLoads + kScaleLoads, kLoadsW = TN / 8 / kWaves;
  constexpr int kProd = WN * WM, kOps = WN + WM;
  constexpr int kFirst = (kLoads + 2) / 4;                             // loads issued in the step behind the barrier
  static_assert(kCodeLoads * 8 * kWaves == kRows && kScaleLoads * 32 * kWaves == kRows && kLoadsW * 8 * kWaves == TN, "whole loads");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, li = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave / NM, wm = wave % NM;

  // ---- this workgroup's tiles ----  each XCD has one run of the tile order, its workgroups take turns.  In the order,
  // MXG_BAND token tiles go together, output tiles outermost among them: what an XCD runs at a time
  // shares few token and weight tiles
  const int tiles_n = (out_columns(p) + TN - 1) / TN, tiles_m = (p.m_last - p.m_first + TM - 1) / TM, n_work = tiles_n * tiles_m;
  const int per_xcd = (n_work + 7) / 8, slots = gridDim.x / 8;
  const int w_end = min(n_work, ((int)blockIdx.x % 8 + 1) * per_xcd);
  int w = (int)blockIdx.x % 8 * per_xcd + (int)blockIdx.x / 8;
  if (w >= w_end) return;

  // ---- loads ----  rows are checked by the resources' ranges (in the lane's offset alone: k, which is
  // always inside a row, is the scalar offset)
  const int64_t line = (int64_t)p.groups * MXG_LINE;                   // bytes of a row of codes
  int ofs[kCodeLoads];
#pragma unroll
  for (int i = 0; i < kCodeLoads; ++i) {
    const int r = (i < kLoadsW ? wave * kLoadsW + i : wave * (kCodeLoads - kLoadsW) + i - kLoadsW) * 8 + (lane >> 3);
    ofs[i] = (int)(r * line) + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
  }
  // what a tile is loaded from: [0] weights' codes, [1] tokens' codes, [2 ..] this wave's scale loads (32 rows; 4 bytes a
  // lane, as a range ends at a row's 8 bytes)
  struct Source {
    unsigned long long ptr[2 + kScaleLoads];
    unsigned len[2 + kScaleLoads];
    int m0, n0;
  };
  auto source = [&](int t) __attribute__((always_inline)) {            // of tile t (behind the last: empty ranges)
    const int band = t / (MXG_BAND * tiles_n), in_band = t - band * MXG_BAND * tiles_n;
    const int rows = max(1, min(MXG_BAND, tiles_m - band * MXG_BAND));
    Source s;
    s.m0 = __builtin_amdgcn_readfirstlane(p.m_first + (band * MXG_BAND + in_band % rows) * TM);      // (quotients and clamps are vector instructions)
    s.n0 = __builtin_amdgcn_readfirstlane(in_band / rows * TN);
    auto range = [&](int x, const unsigned char* base, int64_t row_bytes, int r0, int n) {
      s.ptr[x] = (unsigned long long)base + (t < w_end ? r0 * row_bytes : 0);
      s.len[x] = (unsigned)__builtin_amdgcn_readfirstlane(t < w_end ? max(n, 0) * (int)row_bytes : 0);
    };
    range(0, p.w, line, s.n0, min(TN, p.N - s.n0));
    range(1, p.x, line, s.m0, min(TM, p.m_last - s.m0));
#pragma unroll
    for (int i = 0; i < kScaleLoads; ++i) {
      const int at = 32 * (wave * kScaleLoads + i);
      const bool tok = at >= TN;
      const int r0 = tok ? s.m0 + at - TN : s.n0 + at;
      range(2 + i, tok ? p.x_scales : p.w_scales, MX_GROUP_BLOCKS, r0, min(32, (tok ? p.m_last : p.N) - r0));
    }
    return s;
  };
  const unsigned lds0 = lds_u32(smem);
  Source src = source(w), nsrc = source(w + slots);                    // of the load cursor's tile, and of the one after it
  int lg = 0;                                                          // its group
  auto load = [&](unsigned buf, int i) __attribute__((always_inline)) {
    const int x = i < kLoadsW ? 0 : i < kCodeLoads ? 1 : 2 + i - kCodeLoads;
    const u32x4 rs = {(unsigned)src.ptr[x], (unsigned)(src.ptr[x] >> 32) & 0xffffu, src.len[x], 0x00020000u};
    if (i < kCodeLoads) {
      const int row = i < kLoadsW ? (wave * kLoadsW + i) * 8 : TN + (wave * (kCodeLoads - kLoadsW) + i - kLoadsW) * 8;
      lds_dma16s(buf + row * MXG_LINE, ofs[i], rs, lg * MXG_LINE);
    } else {
      lds_dma4(buf + kCodes + 256 * (wave * kScaleLoads + i - kCodeLoads), 4 * lane, rs);
    }
  };
  auto advance = [&]() __attribute__((always_inline)) {                // by selects: the loop's body stays one block
    ++lg;
    const bool wrap = lg == p.groups;
    lg = wrap ? 0 : lg;
#pragma unroll
    for (int x = 0; x < 2 + kScaleLoads; ++x) {
      if (x >= 2) {
        const int at = 32 * (wave * kScaleLoads + x - 2);
        src.ptr[x] += (unsigned)(at >= TN ? p.M : p.N) * (unsigned long long)MX_GROUP_BLOCKS;
      }
      src.ptr[x] = wrap ? nsrc.ptr[x] : src.ptr[x];
      src.len[x] = wrap ? nsrc.len[x] : src.len[x];
    }
  };

  floatx16 acc[WN][WM];
  i32x4 a[2][WN], b[2][WM];
  int sa[WN], sb[WM], na[WN], nb[WM];                                  // scales: byte s for step s; of this group, the next
  int rd[4];                                                           // operand read offsets of the steps; + 32 rows a sub-tile
#pragma unroll
  for (int s = 0; s < 4; ++s) rd[s] = li * MXG_LINE + (((4 * hl + s) ^ ((li >> 1) & 7)) << 4);
  auto read_op = [&](unsigned buf, int s, int to, int x) __attribute__((always_inline)) {
    const unsigned char* t = smem + buf + rd[s];
    if (x < WN) a[to][x] = *reinterpret_cast<const i32x4*>(t + (wn * WN + x) * 32 * MXG_LINE);
    else if (x < kOps) b[to][x - WN] = *reinterpret_cast<const i32x4*>(t + (TN + (wm * WM + x - WN) * 32) * MXG_LINE);
  };
  auto read_scales = [&](unsigned buf) __attribute__((always_inline)) {
    const unsigned char* t = smem + buf + kCodes + li * MX_GROUP_BLOCKS + 4 * hl;
#pragma unroll
    for (int i = 0; i < WN; ++i) na[i] = *reinterpret_cast<const int*>(t + (wn * WN + i) * 32 * MX_GROUP_BLOCKS);
#pragma unroll
    for (int j = 0; j < WM; ++j) nb[j] = *reinterpret_cast<const int*>(t + (TN + (wm * WM + j) * 32) * MX_GROUP_BLOCKS);
  };
  // the products of step kS; the operands of the step after it (of buffer `buf`) are read between them, and loads
  // l0 .. l1 - 1 of the cursor's group go out to buffer `to`
  auto step = [&](auto s_c, unsigned buf, int l0, int l1, unsigned to) __attribute__((always_inline)) {
    constexpr int kS = decltype(s_c)::value, kFrom = kS & 1, kNext = (kS + 1) & 3;
#pragma unroll
    for (int x = 0; x < kProd; ++x) {
      read_op(buf, kNext, kFrom ^ 1, x);
      if (x == kProd - 1) {                                            // fewer products than operands
#pragma unroll
        for (int y = kProd; y < kOps; ++y) read_op(buf, kNext, kFrom ^ 1, y);
      }
#pragma unroll
      for (int y = l0; y < l1; ++y)
        if ((y - l0) * kProd / (l1 - l0) == x) load(lds0 + to, y);
      __builtin_amdgcn_sched_barrier(0);
      acc[x / WM][x % WM] = mx_mfma<kS>(a[kFrom][x / WM], b[kFrom][x % WM], acc[x / WM][x % WM], sa[x / WM], sb[x % WM]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  unsigned char* const stage = smem + kBufs * kBuf + wave * MXG_STAGE;

  // The accumulators start with the bias: lane l holds the wave's output l's.  The next tile's is loaded before the products and
  // taken where the wait for a group's loads stands: at the tile's end that wait would include the outputs' stores (2 % more
  // time at 65,520 x 13,824 x 5,120, 9 % at 512 x 5,120 x 4,096)
  static_assert(WN == 2, "a bias value a lane");
  const bool bias32 = p.bias_dtype == ICSA_DT_F32;
  auto wave_bias = [&](int n) {                                        // its bits as they are: a conversion would wait for them
    const int at = n + wn * 64 + lane;
    if (p.bias == nullptr || (unsigned)at >= (unsigned)p.N) return 0;   // (past the last tile n may be anything)
    return bias32 ? reinterpret_cast<const int*>(p.bias)[at] : (int)reinterpret_cast<const unsigned short*>(p.bias)[at];
  };
  int bias = wave_bias(src.n0);

  unsigned cur = 0, last = (kBufs - 1) * kBuf;                         // buffer of group g; of the cursor's group (g + kBufs - 1)
#pragma unroll
  for (int g = 0; g < kBufs; ++g) {
    if (g > 0) advance();
#pragma unroll
    for (int i = 0; i < (g == kBufs - 1 ? kFirst : kLoads); ++i) load(lds0 + g * kBuf, i);
  }
  asm volatile("s_waitcnt vmcnt(%0)" :: "n"((kBufs - 2) * kLoads + kFirst) : "memory");    // group 0
  ATT_BARRIER();
  read_scales(0);
#pragma unroll
  for (int x = 0; x < kOps; ++x) read_op(0, 0, 0, x);

  int m0 = src.m0, n0 = src.n0;
  asm volatile("" : "+v"(bias));
  for (;;) {
    bias <<= bias32 ? 0 : 16;
#pragma unroll
    for (int i = 0; i < WN; ++i) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int at = 32 * i + 8 * (e >> 2) + (e & 3);
        const float x = __int_as_float(__builtin_amdgcn_ds_bpermute(4 * (at + 4 * hl), bias));
#pragma unroll
        for (int j = 0; j < WM; ++j) acc[i][j][e] = x;
      }
#pragma unroll
      for (int j = 0; j < WM; ++j) asm volatile("" : "+v"(acc[i][j]));   // registers of their own: one value for all is copied too late
      __builtin_amdgcn_sched_barrier(0);
    }
    bias = wave_bias(nsrc.n0);                         // (past the last tile: not used)
    int g = 0;
    do {
#pragma unroll
      for (int i = 0; i < WN; ++i) sa[i] = na[i];
#pragma unroll
      for (int j = 0; j < WM; ++j) sb[j] = nb[j];
      step(std::integral_constant<int, 0>{}, cur, kFirst, kLoads, last);
      step(std::integral_constant<int, 1>{}, cur, 0, 0, 0);
      step(std::integral_constant<int, 2>{}, cur, 0, 0, 0);
      asm volatile("s_waitcnt vmcnt(%0)" :: "n"((kBufs - 2) * kLoads) : "memory");         // group g + 1
      if constexpr (kBufs == 2) asm volatile("" : "+v"(bias));
      ATT_BARRIER();                                                   // everybody's; and everybody has read group g
      last = cur;
      cur = cur == (kBufs - 1) * kBuf ? 0 : cur + kBuf;
      read_scales(cur);
      advance();
      step(std::integral_constant<int, 3>{}, cur, 0, kFirst, last);
    } while (++g < p.groups);
    // ---- this tile's outputs, while the next one's first groups arrive ----
#pragma unroll
    for (int j = 0; j < WM; ++j)
#pragma unroll
      for (int i = 0; i < WN; ++i) {
        const int n = n0 + (wn * WN + i) * 32, mt = m0 + (wm * WM + j) * 32;
        float v[16];
        tile_values(p, acc[i][j], v);
        if constexpr (kOut == MX_OUT_MXFP4) store_mx(p, v, n, mt + li);
        else if constexpr (kOut == MX_OUT_F32) store_f32(p, v, n, mt + li);
        else store_bf16(p, stage, v, n, mt);
        __builtin_amdgcn_sched_barrier(0);                             // one sub-tile's temporaries at a time
      }
    w += slots;
    if (w >= w_end) break;
    m0 = nsrc.m0; n0 = nsrc.n0;
    nsrc = source(w + slots);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                     // the empty loads
}

namespace {

template <int WN, int WM, int NN, int NM, int kBufs, int kOut>
hipError_t run_mx_gemm(const MxGemmParams& p, hipStream_t stream) {
  constexpr int TN = 32 * WN * NN, TM = 32 * WM * NM;
  constexpr int kLds = kBufs * (TN + TM) * (MXG_LINE + MX_GROUP_BLOCKS) + NN * NM * MXG_STAGE;
  static_assert(kLds <= 160 * 1024, "LDS of a CU");
  static std::atomic<unsigned> lds_set{0u};
  const hipError_t e = ensure_lds_limit(reinterpret_cast<const void*>(icsa_mx_gemm_kernel<WN, WM, NN, NM, kBufs, kOut>), kLds, &lds_set);
  if (e != hipSuccess) return e;
  const int64_t tiles = (int64_t)((out_columns(p) + TN - 1) / TN) * ((p.m_last - p.m_first + TM - 1) / TM);
  if (tiles > 0x3ffffff0LL) return hipErrorInvalidValue;
  // several tiles a workgroup where its loads run at most one tile ahead, and where a CU holds one workgroup
  const int64_t most = p.groups >= kBufs && 2 * kLds > 160 * 1024 ? MXG_CUS : tiles;
  hipLaunchKernelGGL((icsa_mx_gemm_kernel<WN, WM, NN, NM, kBufs, kOut>), dim3(xcd_grid((int)(tiles < most ? tiles : most))),
                     dim3(64 * NN * NM), kLds, stream, p);
  return hipGetLastError();
}

template <int kOut>
hipError_t pick_mx_gemm(MxGemmParams p, hipStream_t stream) {
  const int large = (int)mx_large_rows(p.M, out_columns(p), p.groups, p.gelu != 0);
  if (large > 0) {
    p.m_last = large;
    const hipError_t e = run_mx_gemm<2, 4, 4, 2, 2, kOut>(p, stream);
    if (e != hipSuccess || large == p.M) return e;
    p.m_first = large;
    p.m_last = p.M;
    if (mx_rows_takes(p.M - large, p.N)) return launch_mx_rows(p, stream);
  }
  return run_mx_gemm<2, 2, 2, 2, 4, kOut>(p, stream);
}

}  // namespace

hipError_t launch_mx_gemm(MxGemmParams p, hipStream_t stream) {
  p.m_first = 0;
  p.m_last = p.M;
  if (mx_rows_takes(p.M, p.N)) return launch_mx_rows(p, stream);
  switch (p.out_kind) {
    case MX_OUT_BF16: return pick_mx_gemm<MX_OUT_BF16>(p, stream);
    case MX_OUT_F32: return pick_mx_gemm<MX_OUT_F32>(p, stream);
    default: return pick_mx_gemm<MX_OUT_MXFP4>(p, stream);
  }
}
