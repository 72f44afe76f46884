// Backward of attention over documents (the cross attention's): with P = exp2(c q.k - lse), c = scale log2 e, and
// D = rowsum(dO * O),
//   dS = P * (dO V^T - D);  dq = scale dS K;  dk = scale dS^T Q;  dv = P^T dO.
//
// Two kernels of one body, without atomics, so that the same inputs give the same bits: query-major (dq, and D on the way)
// and key-major (dk, dv), which compute S and dP each.  A workgroup of 4 waves holds 128 rows of one side in registers, 32 a
// wave (queries with dO, or keys with values), and walks the other side in tiles of 64 rows, whose two row-major arrays arrive by
// direct global->LDS loads, two buffers, one barrier a tile; two workgroups share a CU, three with heads of 64.  Products by v_mfma_f32_32x32x16_bf16: S
// and dP with the tile's rows as the first operand and the held rows as the second, so that a lane holds one of its wave's rows; P
// and dS go from there to the second products, whose first operand is read transposed from the same tile.  Where few blocks of a
// side exist, the walk is cut in parts, whose f32 sums a third kernel joins.
//
// A row of the query side is a (query, head) pair; the H / Hk heads of a key head's group are consecutive rows, and the
// key-major walk goes over all of them: dk and dv are summed over the group in the accumulators.
//
// What a row sees of the other side is one range in either direction, its document's.  Only tiles that some row sees in part are masked:
// P and dS of unseen pairs are cleared by bits.  There, rows of the tile that hold a NaN or an infinity are cleared too, as
// 0 times such a value would reach rows that do not see it; the rows that do get NaN at the end, as they would have:
// from a NaN of lse or a D that is not finite, which every such row has unless its weight there is 0.
//
// What bounds it: the matrix pipe, the elementwise work (an exponential, a multiplication or two and two conversions a pair), the
// operands' way from LDS and the clock, side by side: 8,192 x 8,192 rows of 8 heads of 128 take 372 us (dq, 1.11 PFLOP/s of its three
// products; 354 without the rows' totals) and 455 (dk and dv, 1.21 of four); the same without exponentials 342, without operand reads 299, with neither 274, without
// the tiles' loads 327 (dq).  Short walks add a workgroup's start and end: over 512 keys (eight tiles) dq of 65,520 queries of 40 heads
// takes 1.25 ms (0.82), 0.60 of it for the rows' bytes alone, which the other workgroup of the CU does not hide whole; dk and dv 1.24
// (1.10; the matrix pipe busy 64 % at 1.6 GHz, in dq 43 % at 1.9).  Heads of 64 halve the products of a pair and none of its elementwise work:
// 2 x 9,373 queries of 24 heads on 8, padded prompts, dq 155 us with vector instructions active 73 % of the time, at heads of 128 49 %.  Tried: 64 held rows a wave, whose operands serve two products (one
// wave a SIMD, accumulators moved between register files: dq 8,192 x 8,192 402, dk and dv spill); elementwise work between the
// products of key-major 128 dims (registers); the first tile
// requested before the held rows, starts staggered, the next workgroup's lines requested ahead: no change, or slower.
#include <algorithm>
#include <utility>

#include "attn_rows.h"

#define AB_THREADS 256
#define AB_WAVES 4
#define AB_ROWS (32 * AB_WAVES)                         // held by a workgroup
#define AB_SCRATCH_WAVE (3 * 1024)                    // staged output rows, at most 2 KB; in the loop: ranges, operands
#define AB_CTL_BYTES 256
#define AB_LOG2E 1.4426950408889634f

namespace {

// A tile: 64 rows.  A load instruction lands 1 KB, 16 bytes a lane in their order: four rows of 128 dims or eight of 64, in pieces
// of 64 bytes (32 dims) of each row in turn: chunk c (16 bytes) of the instruction's row x at kPiece (c / 4) + 64 x + 16 (c % 4), and
// of 64 dims with c's lowest bit flipped where x >= 4.  Instructions are set apart by a little more than 1 KB.  So 16 rows' reads of
// one chunk, and a half wave's transposing read, touch every bank once, and what a read's address depends on besides the
// lane is a constant in the instruction: with chunks exclusive-ored by the row's number, as in the framework's other
// kernels, the addresses took 16 registers, and these kernels have none to spare.
template <int D> struct BTile {
  static constexpr int kChunks = D / 8, kRowsPerLoad = 512 / D, kLoads = 16 / kRowsPerLoad;   // of a wave's 16 rows
  static constexpr int kLoad = D == 128 ? 1040 : 1056, kPiece = 64 * kRowsPerLoad;
  static constexpr int kBytes = 64 / kRowsPerLoad * kLoad, kRows16 = kLoads * kLoad;
  static __device__ __forceinline__ int flip(int r) { return D == 64 ? (r >> 2) & 1 : 0; }
  // chunk c of row r
  static __device__ __forceinline__ int at(int r, int c) {
    return r / kRowsPerLoad * kLoad + (c >> 2) * kPiece + r % kRowsPerLoad * 64 + (((c & 3) ^ flip(r)) << 4);
  }
};

// f(0), f(1) .. f(N - 1) with their numbers as constants: a tile's 32 to 64 products are past what the compiler unrolls
template <int... I, class F> __device__ __forceinline__ void each(std::integer_sequence<int, I...>, F&& f) {
  (f(std::integral_constant<int, I>{}), ...);
}

// Documents seen from either side (row_range)
struct DocView {
  int Sq, Sk;
  const int* q_starts; const int* k_starts;
  int docs;
  static constexpr int causal = 0;
  static constexpr const int* prefix = nullptr;
};

// What dq is divided by for its row's total of P.  lse is the forward's total of rounded weights; P sums to 1 but for that.  It would
// be a third of what dq is off beside its own roundings (f32 dq over 226 keys 0.00179 from the exact one, so 0.00173); the sums cost 3 % (65,520
// over 512: 1,226 and 1,258 us).  A total far from 1 is no rounding's: a row of nothing, or of what is not finite.
__device__ __forceinline__ float row_total(float sum) { return sum > 0.5f && sum < 2.f ? sum : 1.f; }

template <int D> constexpr int ab_lds() { return 4 * BTile<D>::kBytes + 2 * 512 + AB_WAVES * AB_SCRATCH_WAVE + AB_CTL_BYTES; }

}  // namespace

// FINE: P and dS as two bf16 each, where the queries are one block or the keys a few
template <int D, bool KV, bool FINE>
__global__ void __launch_bounds__(AB_THREADS, FINE ? (D == 64 && !KV ? 2 : 1) : D == 64 ? 3 : 2) icsa_attn_bwd_kernel(AttnBwdParams p) {
  typedef BTile<D> T;
  constexpr int kSteps = D / 16, kSub = D / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* const rowv = smem + 4 * T::kBytes;                       // KV: lse and D of the tile's rows, two buffers
  unsigned char* const scratch_all = rowv + 2 * 512;
  int* const ctl = reinterpret_cast<int*>(scratch_all + AB_WAVES * AB_SCRATCH_WAVE);   // the waves' ranges; rows cleared
  const int lane = threadIdx.x & 63, li = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = p.by_g.d, n_q = p.Sq * G, n_st = KV ? p.Sk : n_q, n_sm = KV ? n_q : p.Sk;   // rows held, rows walked
  const FastDiv& by_blk = KV ? p.by_kblk : p.by_qblk;
  const int n_blk = by_blk.d, n_split = KV ? p.k_split : p.q_split, BH = p.B * p.Hk;
  const int w = xcd_remap(blockIdx.x, BH * n_split * n_blk);             // neighbours: blocks that walk the same rows
  if (w < 0) return;
  const int ws = by_blk.div(w), blk = w - ws * n_blk, bh = ws / n_split, split = ws - bh * n_split;
  const int b = p.by_hk.div(bh), hk = p.by_hk.mod(bh);
  const int r0 = blk * AB_ROWS + 32 * wave;                          // the wave's first row
  const int rows_valid = min(32, n_st - r0);

  // ---- the held rows: operands of S (b1) and dP (b2) ----
  const int r = r0 + li, rc = min(r, n_st - 1);
  bf16x8 b1[kSteps], b2[kSteps];
  float lse = 0.f, dd = 0.f;                                              // query-major: the row's
  {
    const bf16 *s1, *s2;
    if constexpr (KV) {
      s1 = p.k + (int64_t)b * p.k_sb + (int64_t)rc * p.k_ss + (int64_t)hk * p.k_sh + 8 * hl;
      s2 = p.v + (int64_t)b * p.v_sb + (int64_t)rc * p.v_ss + (int64_t)hk * p.v_sh + 8 * hl;
    } else {
      s1 = p.q + row_at(p.q_sb, p.q_ss, p.q_sh, b, hk, p.by_g, rc) + 8 * hl;
      s2 = p.dout + row_at(p.do_sb, p.do_ss, p.do_sh, b, hk, p.by_g, rc) + 8 * hl;
    }
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk) {
      b1[kk] = *reinterpret_cast<const bf16x8*>(s1 + 16 * kk);
      b2[kk] = *reinterpret_cast<const bf16x8*>(s2 + 16 * kk);
    }
  }
  if constexpr (!KV) {                                                    // D = rowsum(dO * O), f32
    const bf16* so = p.o + row_at(p.o_sb, p.o_ss, p.o_sh, b, hk, p.by_g, rc) + 8 * hl;
    lse = p.lse[(int64_t)bh * n_q + rc];
    u32x4 rest[kSteps / 2];                                               // 16 bytes: two steps' (rest_at)
    if (p.rest != nullptr) {
      const unsigned char* sr = p.rest + row_at((int64_t)p.Sq * p.H * D, (int64_t)p.H * D, D, b, hk, p.by_g, rc) + hl * (D / 2);
#pragma unroll
      for (int i = 0; i < kSteps / 2; ++i) rest[i] = *reinterpret_cast<const u32x4*>(sr + 16 * i);
    } else {
#pragma unroll
      for (int i = 0; i < kSteps / 2; ++i) rest[i] = u32x4{0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u};
    }
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk) {
      const bf16x8 o = *reinterpret_cast<const bf16x8*>(so + 16 * kk);
      const int at = (kk & 1) * (kSteps / 2) + (kk >> 1);                 // its eight bytes
#pragma unroll
      for (int e = 0; e < 8; ++e) dd = fmaf((float)b2[kk][e], with_rest(o[e], rest[at >> 1][2 * (at & 1) + (e >> 2)], e & 3), dd);
    }
    dd = xhalf_sum(dd);
    if (split == 0 && hl == 0 && r < n_st) {                              // what the key-major kernel's accumulators start with
      p.rowv[(int64_t)bh * n_q + r] = -lse / (p.scale * AB_LOG2E);
      p.rowv[(int64_t)(BH + bh) * n_q + r] = -dd;
    }
  }
  if (!KV && p.dq.p == nullptr) return;                                   // only D was wanted

  // ---- what the rows see ----
  const DocView view = KV ? DocView{p.Sk, p.Sq, p.k_starts, p.q_starts, p.docs} : DocView{p.Sq, p.Sk, p.q_starts, p.k_starts, p.docs};
  RowRange rr = row_range(view, b, KV || G == 1 ? r : (int)p.by_g.div(r));
  if constexpr (KV) { rr.lo *= G; rr.hi *= G; }
  if (r >= n_st) rr = RowRange{0, 0, 0};
  const bool some = rr.hi > rr.lo;
  {
    const int lo = wave_min(some ? rr.lo : 0x7fffffff), hi = wave_max(some ? rr.hi : 0);
    const int in_lo = wave_max(some ? rr.lo : 0), in_hi = wave_min(some ? rr.hi : 0x7fffffff);
    if (lane == 0) { ctl[wave] = lo; ctl[4 + wave] = hi; ctl[8 + wave] = in_lo; ctl[12 + wave] = in_hi; }
  }
  // what only tiles seen in part need of a row: its range, and whether it gets NaN (key-major); the wave's own LDS
  int* const seen = reinterpret_cast<int*>(scratch_all + wave * AB_SCRATCH_WAVE) + lane;
  seen[0] = rr.lo;
  seen[64] = rr.hi;
  seen[128] = 0;
  __syncthreads();
  // walked rows that some row sees, [u_lo, u_hi), and those that every row (that sees any) sees, [a_lo, a_hi)
  auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  const int u_lo = uni(min(min(ctl[0], ctl[1]), min(ctl[2], ctl[3]))), u_hi = uni(max(max(ctl[4], ctl[5]), max(ctl[6], ctl[7])));
  const int a_lo = uni(max(max(ctl[8], ctl[9]), max(ctl[10], ctl[11]))), a_hi = uni(min(min(ctl[12], ctl[13]), min(ctl[14], ctl[15])));
  int t0 = 0, t1 = 0;                                                     // tiles from row u_lo on, this part's
  if (u_hi > u_lo) {
    const int tiles = (u_hi - u_lo + ATT_BN - 1) / ATT_BN, q = tiles / n_split, more = tiles - q * n_split;
    t0 = q * split + min(split, more);
    t1 = t0 + q + (split < more);
  }

  // ---- loads ----
  const bf16* const xb = KV ? p.q + (int64_t)b * p.q_sb + (int64_t)hk * G * p.q_sh : p.k + (int64_t)b * p.k_sb + (int64_t)hk * p.k_sh;
  const bf16* const yb = KV ? p.dout + (int64_t)b * p.do_sb + (int64_t)hk * G * p.do_sh : p.v + (int64_t)b * p.v_sb + (int64_t)hk * p.v_sh;
  const int64_t x_ss = KV ? p.q_ss : p.k_ss, y_ss = KV ? p.do_ss : p.v_ss;
  const int x_sh = KV ? (int)p.q_sh : 0, y_sh = KV ? (int)p.do_sh : 0;
  const bool grouped = KV && G > 1;
  const unsigned lds0 = lds_u32(smem);
  auto load_tile = [&](int t) __attribute__((always_inline)) {
    const int j0 = u_lo + t * ATT_BN, rows = min(ATT_BN, n_sm - j0);
    const unsigned at = lds0 + (t & 1) * 2 * T::kBytes + wave * T::kRows16;
    int ln = lane;
    asm volatile("" : "+v"(ln));                                          // offsets worked out here, not kept in registers
    // this lane's row of the wave's first load (+ kRowsPerLoad i of load i), and its chunk's byte
    const int lane_row = (ln >> 2) % T::kRowsPerLoad, row0 = 16 * wave + lane_row;
    const int ch = (ln / (4 * T::kRowsPerLoad) * 4 + ((ln & 3) ^ T::flip(lane_row))) << 4;
    if (!grouped) {
      const u32x4 xr = dma_rsrc(xb + (int64_t)j0 * x_ss, (int64_t)(rows - 1) * x_ss * 2 + 2 * D);
      const u32x4 yr = dma_rsrc(yb + (int64_t)j0 * y_ss, (int64_t)(rows - 1) * y_ss * 2 + 2 * D);
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i) {
        const int r = row0 + T::kRowsPerLoad * i;
        lds_dma16(at + T::kLoad * i, r * (int)x_ss * 2 + ch, xr);
        lds_dma16(at + T::kBytes + T::kLoad * i, r * (int)y_ss * 2 + ch, yr);
      }
    } else {                                                              // rows (query, head): each its own offset
      const int i0 = p.by_g.div(j0);
      const u32x4 xr = dma_rsrc(xb + (int64_t)i0 * x_ss, 0x7fffffff), yr = dma_rsrc(yb + (int64_t)i0 * y_ss, 0x7fffffff);
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i) {
        const int lr = row0 + T::kRowsPerLoad * i, r = j0 + lr, qi = p.by_g.div(r), g = r - qi * G;
        const bool in = lr < rows;                                        // past the last row: out of the buffer's range
        lds_dma16(at + T::kLoad * i, in ? ((qi - i0) * (int)x_ss + g * x_sh) * 2 + ch : 0x7fffffff, xr);
        lds_dma16(at + T::kBytes + T::kLoad * i, in ? ((qi - i0) * (int)y_ss + g * y_sh) * 2 + ch : 0x7fffffff, yr);
      }
    }
    if (KV && wave < 2)
      lds_dma4(lds0 + 4 * T::kBytes + (t & 1) * 512 + wave * 256, lane * 4,
               dma_rsrc(p.rowv + (int64_t)(wave * BH + bh) * n_q + j0, rows * 4));
  };
#pragma unroll
  for (int kk = 0; kk < kSteps; ++kk) {                                   // in registers before the first tile is requested
    u32x4 x = __builtin_bit_cast(u32x4, b1[kk]), y = __builtin_bit_cast(u32x4, b2[kk]);
    asm volatile("" : "+v"(x), "+v"(y));
    b1[kk] = __builtin_bit_cast(bf16x8, x);
    b2[kk] = __builtin_bit_cast(bf16x8, y);
  }
  if constexpr (!KV) asm volatile("" : "+v"(lse), "+v"(dd));
  // Key-major with 128 dims the registers are two operands short; what the compiler spills it reloads behind a wait for all loads
  // in flight, the next tile's too.  Both sides' first operand lies in the wave's LDS instead.
  constexpr bool kLent = KV && D == 128 && !FINE;
  bf16x8* const lent = reinterpret_cast<bf16x8*>(scratch_all + wave * AB_SCRATCH_WAVE + 1024) + lane;
  if constexpr (kLent) { lent[0] = b1[0]; lent[64] = b2[0]; }
  if (t0 < t1) load_tile(t0);

  const int ro = T::at(li, hl);                                           // chunk 2 kk + hl of row li: + kPiece (kk / 2) + 32 (kk % 2)
  int tro;                                                                // transposing reads, dims 32 d: + kPiece d; 8 rows on: + kRows16 / 2
  {
    const int g = lane >> 4, s = lane & 15;
    tro = T::at(4 * (g >> 1) + (s >> 2), 2 * (g & 1) + ((s & 3) >> 1)) + (s & 1) * 8;
  }
  const float c = p.scale * AB_LOG2E;
  floatx16 acc1[kSub] = {};                                               // dq or dk
  floatx16 acc2[KV ? kSub : 1] = {};                                      // dv
  float total[2] = {};                                                    // query-major: of the row's P

  for (int t = t0; t < t1; ++t) {
    const int j0 = u_lo + t * ATT_BN;
    unsigned char* const xs = smem + (t & 1) * 2 * T::kBytes;
    unsigned char* const ys = xs + T::kBytes;
    const float* const lse_l = reinterpret_cast<const float*>(rowv + (t & 1) * 512);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const bool wg_partial = j0 < a_lo || j0 + ATT_BN > a_hi;              // for some row of the workgroup
    if (wg_partial) {
      // this wave's 16 rows of the tile: cleared where no row sees them, or where they hold something that is not finite
      const int row = 16 * wave + (lane >> 2), c0 = (lane & 3) * (T::kChunks / 4);
      const bool past = j0 + row >= u_hi;
      unsigned bad = 0;
#pragma unroll
      for (int e = 0; e < T::kChunks / 4; ++e) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(xs + T::at(row, c0 + e));
        bad |= not_finite2(x[0]) | not_finite2(x[1]) | not_finite2(x[2]) | not_finite2(x[3]);
        if constexpr (KV) {
          const u32x4 y = *reinterpret_cast<const u32x4*>(ys + T::at(row, c0 + e));
          bad |= not_finite2(y[0]) | not_finite2(y[1]) | not_finite2(y[2]) | not_finite2(y[3]);
        }
      }
      const unsigned long long any = __ballot(bad != 0u && !past);
      if (past || ((any >> (lane & ~3)) & 15ull) != 0ull) {
#pragma unroll
        for (int e = 0; e < T::kChunks / 4; ++e) {
          *reinterpret_cast<u32x4*>(xs + T::at(row, c0 + e)) = u32x4{0u, 0u, 0u, 0u};
          if constexpr (KV) *reinterpret_cast<u32x4*>(ys + T::at(row, c0 + e)) = u32x4{0u, 0u, 0u, 0u};
        }
      }
      const unsigned long long rows16 = __ballot(lane < 16 && ((any >> (4 * (lane & 15))) & 15ull) != 0ull);
      if (lane == 0) ctl[16 + (t & 1) * 4 + wave] = (int)rows16;
    }
    ATT_BARRIER();
    if (t + 1 < t1) load_tile(t + 1);
    // the tile's rows that hold something not finite, and those that this lane's row sees
    auto cleared = [&]() __attribute__((always_inline)) {
      const int* w = ctl + 16 + (t & 1) * 4;
      return (unsigned long long)(unsigned)(uni(w[0]) | uni(w[1]) << 16) | (unsigned long long)(unsigned)(uni(w[2]) | uni(w[3]) << 16) << 32;
    };
    auto visible = [&]() __attribute__((always_inline)) {
      const int lo = min(max(seen[0] - j0, 0), 64), hi = min(max(seen[64] - j0, 0), 64);
      return (hi >= 64 ? ~0ull : (1ull << hi) - 1) & ~(lo >= 64 ? ~0ull : (1ull << lo) - 1);
    };
    bool partial = false;
    if (wg_partial) {
      const unsigned long long bad = cleared(), vis = visible();
      // a row that sees nothing asks for no mask: what it sums is not used
      partial = __ballot(bad != 0ull || (some && ~vis != 0ull)) != 0ull;
      if (__ballot(vis != 0ull) == 0ull) continue;                        // none of the wave's rows sees any of the tile
      if (KV && bad != 0ull) {
#pragma unroll 1
        for (int x = 0; x < 64; ++x) {
          const float l = lse_l[x], d = lse_l[64 + x];                    // -lse / c, -D
          if (((bad >> x) & (vis >> x) & 1ull) != 0ull && (l != l || !__builtin_isfinite(d))) seen[128] = 1;
        }
      }
    }
    // The tile's products in one stream of phases of kSteps each, an operand read kAhead products ahead of its use; query-major, the
    // elementwise work of one phase between the products of the next (key-major has no registers for that):
    //   key-major     S, dP | P, dS | dv, dk of either 32 rows in turn
    //   query-major   S0, dP0 | P0, S1 | dS0, dP1 | P1, dq0 | dS1, dq1
    // Key-major with 64 dims: spread out too, and operands three ahead, it takes 184 registers instead of 168, and a third workgroup on
    // the CU is worth more (65,520 queries over 512 keys, 40 heads: 693 us, 682 with three, 649 with parts for three).
    constexpr int kAhead = KV && D == 64 ? 2 : 3;
    constexpr int kPhases = KV ? 8 : 6, kOps = kPhases * kSteps, kEl = 16 / kSteps;
    static constexpr int kWhat[8] = {0, 1, KV ? 2 : 0, KV ? 3 : 1, KV ? 0 : 3, KV ? 1 : 3, 2, 3};      // S, dP, dv, dk (dq)
    static constexpr int kOf[8] = {0, 0, KV ? 0 : 1, KV ? 0 : 1, KV ? 1 : 0, 1, 1, 1};                  // which 32 rows
    floatx16 s[2], dp[2];
    bf16x8 first[2], second[2];
    bf16x8 pf[2][2], df[2][2];
    bf16x8 pl[2][2], dl[2][2];                                            // FINE: what the roundings leave
    bf16x8 a[kOps];
    auto op = [&](int x) __attribute__((always_inline)) {
      const int what = kWhat[x / kSteps], sub = kOf[x / kSteps], i = x % kSteps;
      const unsigned char* tile = what == 1 || what == 2 ? ys : xs;
      if (what < 2) {                                                     // chunk 2 i + hl of a row
        a[x] = *reinterpret_cast<const bf16x8*>(tile + ro + sub * 2 * T::kRows16 + (i >> 1) * T::kPiece + (i & 1) * 32);
      } else {                                                            // dims 32 (i % kSub) of 16 rows, transposed
        const unsigned char* at = tile + tro + (2 * sub + i / kSub) * T::kRows16 + i % kSub * T::kPiece;
        const rt_v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((rt_lds_v4s)at);
        const rt_v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((rt_lds_v4s)(at + T::kRows16 / 2));
        const short __attribute__((ext_vector_type(8))) a8 = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        a[x] = __builtin_bit_cast(bf16x8, a8);
      }
    };
    // P and dS rounded to bf16, the matrix instruction's type (2^-8 of a weight at most), as in the forward: over many queries
    // that is as much again as the results' own rounding leaves.  Over a few, one weight's error can be most of a
    // result's, and the products are no time at all: FINE adds what the rounding left.
    auto weights = [&](int sub, int e) __attribute__((always_inline)) {
      s[sub][e] = __builtin_amdgcn_exp2f(KV ? s[sub][e] * c : fmaf(s[sub][e], c, -lse));
      if constexpr (KV) {
        pf[sub][e >> 3][e & 7] = (bf16)s[sub][e];
        if constexpr (FINE) pl[sub][e >> 3][e & 7] = (bf16)(s[sub][e] - (float)pf[sub][e >> 3][e & 7]);
      }
    };
    auto slopes = [&](int sub, int e) __attribute__((always_inline)) {
      const float x = s[sub][e] * (KV ? dp[sub][e] : dp[sub][e] - dd);
      df[sub][e >> 3][e & 7] = (bf16)x;
      if constexpr (FINE) dl[sub][e >> 3][e & 7] = (bf16)(x - (float)df[sub][e >> 3][e & 7]);
    };
    auto clear = [&](bf16x8 (&w)[2], int sub) __attribute__((always_inline)) {
      const int wd = (int)(unsigned)((visible() & ~cleared()) >> (32 * sub + 4 * hl));
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        u32x4 d = __builtin_bit_cast(u32x4, w[m]);
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const int i = 8 * m + e, bit = 8 * (i >> 2) + (i & 3);          // element i is row bit (+ 4 hl) of the 32
          d[e >> 1] &= bit_select(0xffffu, (unsigned)__builtin_amdgcn_sbfe(wd, bit, 1), (unsigned)__builtin_amdgcn_sbfe(wd, bit + 1, 1));
        }
        w[m] = __builtin_bit_cast(bf16x8, d);
      }
    };
    auto start = [&](int sub) __attribute__((always_inline)) {
      s[sub] = dp[sub] = floatx16{};
      first[sub] = kLent ? lent[0] : b1[0];
      if constexpr (KV) {                                                 // element 4 g + y is row 8 g + 4 hl + y
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const floatx4 l4 = *reinterpret_cast<const floatx4*>(lse_l + 32 * sub + 8 * g + 4 * hl);
          const floatx4 d4 = *reinterpret_cast<const floatx4*>(lse_l + 64 + 32 * sub + 8 * g + 4 * hl);
#pragma unroll
          for (int y = 0; y < 4; ++y) { s[sub][4 * g + y] = l4[y]; dp[sub][4 * g + y] = d4[y]; }
        }
      }
    };
    start(0);
    if (!KV) start(1);
#pragma unroll
    for (int x = 0; x < kAhead; ++x) op(x);
    each(std::make_integer_sequence<int, kOps>{}, [&](auto number) __attribute__((always_inline)) {
      constexpr int x = decltype(number)::value, ph = x / kSteps, what = kWhat[ph], sub = kOf[ph], i = x % kSteps;
      if (KV && x == 4 * kSteps) start(1);
      if (x + kAhead < kOps) op(x + kAhead);
      if (what == 0 && i == kSteps - kAhead) second[sub] = kLent ? lent[64] : b2[0];
      if (what == 0) s[sub] = mfma32x32x16(a[x], i == 0 ? first[sub] : b1[i], s[sub]);
      else if (what == 1) dp[sub] = mfma32x32x16(a[x], i == 0 ? second[sub] : b2[i], dp[sub]);
      else if (what == 2) acc2[i % kSub] = mfma32x32x16(a[x], pf[sub][i / kSub], acc2[i % kSub]);
      else acc1[i % kSub] = mfma32x32x16(a[x], df[sub][i / kSub], acc1[i % kSub]);
      if constexpr (FINE) {
        if (what == 2) acc2[i % kSub] = mfma32x32x16(a[x], pl[sub][i / kSub], acc2[i % kSub]);
        if (what == 3) acc1[i % kSub] = mfma32x32x16(a[x], dl[sub][i / kSub], acc1[i % kSub]);
      }
      if constexpr (KV) {
        if (what == 1 && i == kSteps - 1) {
#pragma unroll
          for (int e = 0; e < 16; ++e) { weights(sub, e); slopes(sub, e); }
          if (partial) {
            clear(pf[sub], sub);
            clear(df[sub], sub);
            if (FINE) { clear(pl[sub], sub); clear(dl[sub], sub); }
          }
        }
      } else {
#pragma unroll
        for (int e = i * kEl; e < (i + 1) * kEl; ++e) {
          if (ph == 1) weights(0, e);
          else if (ph == 2) slopes(0, e);
          else if (ph == 3) weights(1, e);
          else if (ph == 4) slopes(1, e);
        }
        if (i == kSteps - 1 && (ph == 1 || ph == 3)) {
          const int wd = partial ? (int)(unsigned)((visible() & ~cleared()) >> (16 * (ph - 1) + 4 * hl)) : -1;
          if (partial) {
#pragma unroll
            for (int e = 0; e < 16; ++e) total[e & 1] += wd >> (8 * (e >> 2) + (e & 3)) & 1 ? s[ph / 2][e] : 0.f;
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) total[e & 1] += s[ph / 2][e];
          }
        }
        if (i == kSteps - 1 && partial && (ph == 2 || ph == 4)) {
          clear(df[ph / 4], ph / 4);
          if (FINE) clear(dl[ph / 4], ph / 4);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  }

  // ---- results ----
  if (rows_valid <= 0) return;
  unsigned char* const scratch = scratch_all + wave * AB_SCRATCH_WAVE;
  float f1 = p.scale, f2 = 1.f;
  if (!some) {                                                            // whatever it holds of tiles that others see whole
#pragma unroll
    for (int d = 0; d < kSub; ++d) {
      acc1[d] = floatx16{};
      if constexpr (KV) acc2[d] = floatx16{};
    }
  } else if constexpr (KV) {
    if (seen[128] != 0) f1 = f2 = NAN;
  } else if (lse != lse || !__builtin_isfinite(dd)) {
    f1 = NAN;
  } else if (n_split == 1) {
    f1 /= row_total(xhalf_sum(total[0] + total[1]));
  }
  if constexpr (!KV) {                                                    // of parts: divided by where they are joined
    if (n_split > 1) {
      const float sum = xhalf_sum(total[0] + total[1]);
      if (hl == 0 && li < rows_valid) p.dq_total[((int64_t)split * BH + bh) * n_st + r] = sum;
    }
  }
  auto finish = [&](const floatx16* acc, float f, const OutView& out, float* part) {
    if (n_split == 1) {
      if (out.p != nullptr) store_wave<D>(out, KV ? FastDiv{1u, 0u, 1u, 0u} : p.by_g, scratch, acc, f, b, hk, r0, rows_valid);
    } else if (li < rows_valid) {
      float* dst = part + (((int64_t)split * BH + bh) * n_st + r) * D + 4 * hl;
#pragma unroll
      for (int d = 0; d < kSub; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<floatx4*>(dst + 32 * d + 8 * g) =
              floatx4{acc[d][4 * g] * f, acc[d][4 * g + 1] * f, acc[d][4 * g + 2] * f, acc[d][4 * g + 3] * f};
    }
  };
  if constexpr (KV) {
    finish(acc1, f1, p.dk, p.dk_part);
    finish(acc2, f2, p.dv, p.dv_part);
  } else {
    finish(acc1, f1, p.dq, p.dq_part);
  }
}

// Joins the parts of every row in their order.  D / 4 threads a row, 4 dims each.  blockIdx.y: dk or dv.
template <int D, bool KV>
__global__ void __launch_bounds__(256) icsa_attn_bwd_join_kernel(AttnBwdParams p) {
  constexpr int kPer = D / 4;
  const int n_st = KV ? p.Sk : p.Sq * (int)p.by_g.d, n_split = KV ? p.k_split : p.q_split;
  const int64_t rows = (int64_t)p.B * p.Hk * n_st, row = (int64_t)blockIdx.x * (256 / kPer) + threadIdx.x / kPer;
  const OutView out = !KV ? p.dq : blockIdx.y ? p.dv : p.dk;
  if (row >= rows || out.p == nullptr) return;
  const int d = threadIdx.x % kPer * 4;
  const float* src = (!KV ? p.dq_part : blockIdx.y ? p.dv_part : p.dk_part) + row * D + d;
  floatx4 s = *reinterpret_cast<const floatx4*>(src);
  float total = KV ? 1.f : p.dq_total[row];
#pragma unroll 4
  for (int i = 1; i < n_split; ++i) {
    const floatx4 v = *reinterpret_cast<const floatx4*>(src + (int64_t)i * rows * D);
    if constexpr (!KV) total += p.dq_total[i * rows + row];
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += v[e];
  }
  if constexpr (!KV) {
    total = row_total(total);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] /= total;
  }
  const int bh = (int)((unsigned)row / (unsigned)n_st), r = (int)row - bh * n_st;   // query rows: under 2^28 (check_masked_sizes); key rows: 2^32 of dk are 512 GiB
  const int64_t off = row_at(out.sb, out.ss, out.sh, p.by_hk.div(bh), p.by_hk.mod(bh), KV ? FastDiv{1u, 0u, 1u, 0u} : p.by_g, r) + d;
  if (out.dtype == ICSA_DT_BF16) {
    bf16x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (bf16)s[e];
    *reinterpret_cast<bf16x4*>(reinterpret_cast<bf16*>(out.p) + off) = y;
  } else {
    *reinterpret_cast<floatx4*>(reinterpret_cast<float*>(out.p) + off) = s;
  }
}

#define AB_CUS 256
#define AB_MAX_SPLIT 64
// P and dS as two bf16 (FINE): up to this many queries of a key head's group, where a call is all start and end; and this many keys,
// where the one bf16's error shows beside the result's own rounding (600 queries over 2 to 8: dq 1.47 to 1.54 of that rounding, dk 1.49 to 1.57;
// FINE 1.07 to 1.14 and 1.09 to 1.17) at a price where queries are many (65,520 of 40 heads: dq 785 us and 1,020, dk and dv 288 and 585).
#define AB_FINE AB_ROWS
#define AB_FINE_KEYS 8
#define AB_MIN_TILES 8                                // of the walked side that a part is worth

namespace {

// Parts of an item's walk (tiles, over all documents): as many as make the rounds of workgroups come out shortest, beside the parts'
// sums on their way through memory: 256 KB written and read an item and part at some 4.5 TB/s, in the time of an item's tiles at
// 3.8 us (65,520 queries over 512 keys of 40 heads: 160 items, 3 parts).  Documents differ in length, and blocks with rows of two
// walk both: there, where rounds are few, four parts at least and two rounds of workgroups (dk and dv: 4 clips of 1,500 to 17,600
// tokens over 320 to 370 keys, 440 items, 1,274 us in one part, 878 in two, 766 in four, 762 in eight; of 8,190 tokens each 794, 700,
// 698 in one, two, four; 5 of 30,000 tokens together over 512 keys, 160 items, 624 in four, 531 in seven; 2 of 20,000 over 1,000,
// 96 items, 251 in four, 229 in eleven).  With heads of 64 a CU holds three workgroups, of which one alone makes about 0.6 of the
// rate and two 0.93: a round of one or two a CU takes that much less time (8,192 x 8,192, 8 heads: 270 in one part, 282 in three;
// 65,520 over 512, 40 heads: 889 in eight, 907 in nine, 935 in three, with the row sums' 260).
int parts(int64_t items, int64_t tiles, int docs, int D) {
  const int slots = AB_CUS * (D == 64 ? 3 : 2);
  auto rounds = [&](int64_t n) {
    const int64_t last = n % slots, cu = (last + AB_CUS - 1) / AB_CUS;
    return (double)(n / slots) + (cu == 0 ? 0. : D != 64 || cu == 3 ? 1. : cu == 2 ? 0.72 : 0.56);
  };
  int best = 1;
  double time = 0.;
  const int64_t walk = tiles / docs > 0 ? tiles / docs : 1;
  for (int n = 1; n <= AB_MAX_SPLIT && (n == 1 || walk / n >= AB_MIN_TILES); ++n) {
    const double t = rounds(items * n) / n + (n > 1 ? items * n / (65. * walk) : 0.);
    if (n == 1 || t < time) { time = t; best = n; }
  }
  if (docs > 1 && items <= 2 * slots)
    best = std::max(best, (int)std::min<int64_t>({AB_MAX_SPLIT, walk / AB_MIN_TILES, std::max<int64_t>(4, (2 * slots + items - 1) / items)}));
  return best;
}

int64_t blocks(int64_t rows) { return (rows + AB_ROWS - 1) / AB_ROWS; }

template <int D, bool FINE>
hipError_t run_bwd(const AttnBwdParams& p, hipStream_t stream) {
  static std::atomic<unsigned> set_q{0u}, set_k{0u};
  hipError_t e = ensure_lds_limit(reinterpret_cast<const void*>(icsa_attn_bwd_kernel<D, false, FINE>), ab_lds<D>(), &set_q);
  if (e != hipSuccess) return e;
  e = ensure_lds_limit(reinterpret_cast<const void*>(icsa_attn_bwd_kernel<D, true, FINE>), ab_lds<D>(), &set_k);
  if (e != hipSuccess) return e;
  const int64_t BH = (int64_t)p.B * p.Hk, n_q = (int64_t)p.Sq * (p.H / p.Hk);
  const int64_t wq = BH * blocks(n_q) * p.q_split, wk = BH * blocks(p.Sk) * p.k_split;
  const int64_t jq = (BH * n_q * D + 1023) / 1024, jk = (BH * p.Sk * D + 1023) / 1024;
  if (wq > 0x3fffffffLL || wk > 0x3fffffffLL || (p.q_split > 1 && jq > 0x7fffffffLL) || (p.k_split > 1 && jk > 0x7fffffffLL))
    return hipErrorInvalidValue;
  if (wq > 0) {                                       // without queries dk and dv are zeros, which the key-major kernel writes
    hipLaunchKernelGGL((icsa_attn_bwd_kernel<D, false, FINE>), dim3(xcd_grid((int)wq)), dim3(AB_THREADS), ab_lds<D>(), stream, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (p.q_split > 1 && p.dq.p != nullptr) {
    hipLaunchKernelGGL((icsa_attn_bwd_join_kernel<D, false>), dim3((unsigned)jq), dim3(256), 0, stream, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (p.dk.p == nullptr && p.dv.p == nullptr) return hipSuccess;
  hipLaunchKernelGGL((icsa_attn_bwd_kernel<D, true, FINE>), dim3(xcd_grid((int)wk)), dim3(AB_THREADS), ab_lds<D>(), stream, p);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  if (p.k_split > 1) hipLaunchKernelGGL((icsa_attn_bwd_join_kernel<D, true>), dim3((unsigned)jk, 2), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

AttnBwdPlan attn_bwd_plan(int B, int Sq, int Sk, int H, int Hk, int D, int docs) {
  const int64_t BH = (int64_t)B * Hk, n_q = (int64_t)Sq * (H / Hk);
  return AttnBwdPlan{parts(BH * blocks(n_q), (Sk + ATT_BN - 1) / ATT_BN, docs, D),
                     parts(BH * blocks(Sk), (n_q + ATT_BN - 1) / ATT_BN, docs, D)};
}

hipError_t launch_attn_bwd(AttnBwdParams p, hipStream_t stream) {
  const int G = p.H / p.Hk;
  p.by_g = fast_div(G);
  p.by_hk = fast_div(p.Hk);
  p.by_qblk = fast_div((unsigned)std::max<int64_t>(1, blocks((int64_t)p.Sq * G)));
  p.by_kblk = fast_div((unsigned)std::max<int64_t>(1, blocks(p.Sk)));
  if ((int64_t)p.Sq * G <= AB_FINE || p.Sk <= AB_FINE_KEYS) return p.D == 128 ? run_bwd<128, true>(p, stream) : run_bwd<64, true>(p, stream);
  return p.D == 128 ? run_bwd<128, false>(p, stream) : run_bwd<64, false>(p, stream);
}
