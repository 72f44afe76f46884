// Backward of attention over documents (the cross attention's): with P = exp2(c q.k - lse), c = scale log2 e, and
// D = rowsum(dO * O),
//   dS = P * (dO V^T - D);  dq = scale dS K;  dk = scale dS^T Q;  dv = P^T dO.
//
// Two kernels of one body, without atomics, so that the same inputs give the same bits: query-major (dq, and D on the way)
// and key-major (dk, dv), which compute S and dP each.  A workgroup of 4 waves holds 64 NS rows of one side in registers
// a wave, 32 a sub-block (queries with dO, or keys with values), and walks the other side in tiles of 64 rows, whose two
// row-major arrays arrive by direct global->LDS loads, two buffers, one barrier a tile.  Products by
// v_mfma_f32_32x32x16_bf16: S and dP with the tile's rows as the first operand and the registers' rows as the second, so that a lane holds
// one of its wave's rows; P and dS go from there to the second products, whose first operand is read transposed from the same tile.
// Each operand read from LDS serves NS products.
//
// A row of the query side is a (query, head) pair; the H / Hk heads of a key head's group are consecutive rows, and the
// key-major walk goes over all of them: dk and dv are summed over the group in the accumulators.
//
// What a row sees of the other side is one range in either direction, its document's.  Only tiles that some row sees in part are masked:
// P and dS of unseen pairs are cleared by bits.  There, rows of the tile that hold a NaN or an infinity are cleared too, as
// 0 times such a value would reach rows that do not see it; the rows that do get NaN at the end, as they would have:
// from a NaN of lse or a D that is not finite, which every such row has unless its weight there is 0.
#include <algorithm>

#include "attn_rows.h"

#define AB_THREADS 256
#define AB_WAVES 4
#define AB_AHEAD 4                                    // operands read ahead of their products
#define AB_SCRATCH_WAVE 2048
#define AB_CTL_BYTES 256
#define AB_LOG2E 1.4426950408889634f

namespace {

// A tile: 64 rows, 16-byte chunk c of row r at c ^ swz(r): 16 rows' reads of one chunk touch every bank once, and the
// transposing reads of four rows fall into different bank quarters.  swz has a period of 16 rows and swz(r + 8) = swz(r) ^ 2.
template <int D> struct BTile {
  static constexpr int kRow = D * 2, kBytes = ATT_BN * kRow, kChunks = D / 8;
  static constexpr int kRowsPerLoad = 1024 / kRow, kLoads = 16 / kRowsPerLoad;   // of a wave's 16 rows
  static __device__ __forceinline__ int swz(int r) {
    return D == 128 ? rt_swz(r) : ((((r >> 1) & 1) << 2) | ((r >> 2) & 3));
  }
};

// Documents seen from either side (row_range)
struct DocView {
  int Sq, Sk;
  const int* q_starts; const int* k_starts;
  int docs;
  static constexpr int causal = 0;
  static constexpr const int* prefix = nullptr;
};

__host__ __device__ constexpr int ab_lds(int D) { return 4 * ATT_BN * D * 2 + 2 * 512 + AB_WAVES * AB_SCRATCH_WAVE + AB_CTL_BYTES; }

}  // namespace

template <int D, bool KV, int NS>
__global__ void __launch_bounds__(AB_THREADS, NS == 2 ? 1 : 2) icsa_attn_bwd_kernel(AttnBwdParams p) {
  typedef BTile<D> T;
  constexpr int kSteps = D / 16, kSub = D / 32, kWaveRows = 32 * NS, kRows = AB_WAVES * kWaveRows;
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
  const int r0 = blk * kRows + wave * kWaveRows;                          // the wave's first row
  const int rows_valid = min(kWaveRows, n_st - r0);

  // ---- the held rows: operands of S (b1) and dP (b2) ----
  bf16x8 b1[NS][kSteps], b2[NS][kSteps];
  float lse[NS], dd[NS];                                                  // query-major: the row's
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const int r = min(r0 + 32 * n + li, n_st - 1);
    const bf16 *s1, *s2;
    if constexpr (KV) {
      s1 = p.k + (int64_t)b * p.k_sb + (int64_t)r * p.k_ss + (int64_t)hk * p.k_sh + 8 * hl;
      s2 = p.v + (int64_t)b * p.v_sb + (int64_t)r * p.v_ss + (int64_t)hk * p.v_sh + 8 * hl;
    } else {
      s1 = p.q + row_at(p.q_sb, p.q_ss, p.q_sh, b, hk, p.by_g, r) + 8 * hl;
      s2 = p.dout + row_at(p.do_sb, p.do_ss, p.do_sh, b, hk, p.by_g, r) + 8 * hl;
    }
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk) {
      b1[n][kk] = *reinterpret_cast<const bf16x8*>(s1 + 16 * kk);
      b2[n][kk] = *reinterpret_cast<const bf16x8*>(s2 + 16 * kk);
    }
    if constexpr (!KV) {                                                  // D = rowsum(dO * O), f32
      const bf16* so = p.o + row_at(p.o_sb, p.o_ss, p.o_sh, b, hk, p.by_g, r) + 8 * hl;
      float d = 0.f;
#pragma unroll
      for (int kk = 0; kk < kSteps; ++kk) {
        const bf16x8 o = *reinterpret_cast<const bf16x8*>(so + 16 * kk);
#pragma unroll
        for (int e = 0; e < 8; ++e) d = fmaf((float)b2[n][kk][e], (float)o[e], d);
      }
      dd[n] = xhalf_sum(d);
      lse[n] = p.lse[(int64_t)bh * n_q + r];
      if (split == 0 && hl == 0 && r0 + 32 * n + li < n_st) p.dvec[(int64_t)bh * n_q + r] = dd[n];
    }
  }
  if (!KV && p.dq.p == nullptr) return;                                   // only D was wanted

  // ---- what the rows see ----
  const DocView view = KV ? DocView{p.Sk, p.Sq, p.k_starts, p.q_starts, p.docs} : DocView{p.Sq, p.Sk, p.q_starts, p.k_starts, p.docs};
  RowRange rr[NS];
  {
    int lo = 0x7fffffff, hi = 0, in_lo = 0, in_hi = 0x7fffffff;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const int r = r0 + 32 * n + li;
      rr[n] = row_range(view, b, KV || G == 1 ? r : (int)p.by_g.div(r));
      if constexpr (KV) { rr[n].lo *= G; rr[n].hi *= G; }
      if (r >= n_st) rr[n] = RowRange{0, 0, 0};
      if (rr[n].hi > rr[n].lo) {
        lo = min(lo, rr[n].lo); hi = max(hi, rr[n].hi);
        in_lo = max(in_lo, rr[n].lo); in_hi = min(in_hi, rr[n].hi);
      }
    }
    lo = wave_min(lo); hi = wave_max(hi); in_lo = wave_max(in_lo); in_hi = wave_min(in_hi);
    if (lane == 0) { ctl[wave] = lo; ctl[4 + wave] = hi; ctl[8 + wave] = in_lo; ctl[12 + wave] = in_hi; }
  }
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
  int lrow[T::kLoads], lchunk[T::kLoads];                                 // this lane's row of each load, and its chunk's byte
#pragma unroll
  for (int i = 0; i < T::kLoads; ++i) {
    lrow[i] = 16 * wave + T::kRowsPerLoad * i + lane / T::kChunks;
    lchunk[i] = ((lane % T::kChunks) ^ T::swz(lrow[i])) << 4;
  }
  const unsigned lds0 = lds_u32(smem);
  auto load_tile = [&](int t) __attribute__((always_inline)) {
    const int j0 = u_lo + t * ATT_BN, rows = min(ATT_BN, n_sm - j0);
    const unsigned at = lds0 + (t & 1) * 2 * T::kBytes + wave * 16 * T::kRow;
    if (!grouped) {
      const u32x4 xr = dma_rsrc(xb + (int64_t)j0 * x_ss, (int64_t)(rows - 1) * x_ss * 2 + 2 * D);
      const u32x4 yr = dma_rsrc(yb + (int64_t)j0 * y_ss, (int64_t)(rows - 1) * y_ss * 2 + 2 * D);
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i) lds_dma16(at + 1024 * i, lrow[i] * (int)x_ss * 2 + lchunk[i], xr);
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i) lds_dma16(at + T::kBytes + 1024 * i, lrow[i] * (int)y_ss * 2 + lchunk[i], yr);
    } else {                                                              // rows (query, head): each its own offset
      const int i0 = p.by_g.div(j0);
      const u32x4 xr = dma_rsrc(xb + (int64_t)i0 * x_ss, 0x7fffffff), yr = dma_rsrc(yb + (int64_t)i0 * y_ss, 0x7fffffff);
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i) {
        const int r = j0 + lrow[i], qi = p.by_g.div(r), g = r - qi * G;
        const bool in = lrow[i] < rows;                                   // past the last row: out of the buffer's range
        lds_dma16(at + 1024 * i, in ? ((qi - i0) * (int)x_ss + g * x_sh) * 2 + lchunk[i] : 0x7fffffff, xr);
        lds_dma16(at + T::kBytes + 1024 * i, in ? ((qi - i0) * (int)y_ss + g * y_sh) * 2 + lchunk[i] : 0x7fffffff, yr);
      }
    }
    if (KV && wave < 2)
      lds_dma4(lds0 + 4 * T::kBytes + (t & 1) * 512 + wave * 256, lane * 4,
               dma_rsrc((wave == 0 ? p.lse : p.dvec) + (int64_t)bh * n_q + j0, rows * 4));
  };
#pragma unroll
  for (int n = 0; n < NS; ++n)
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk) {                                 // in registers before the first tile is requested
      u32x4 x = __builtin_bit_cast(u32x4, b1[n][kk]), y = __builtin_bit_cast(u32x4, b2[n][kk]);
      asm volatile("" : "+v"(x), "+v"(y));
      b1[n][kk] = __builtin_bit_cast(bf16x8, x);
      b2[n][kk] = __builtin_bit_cast(bf16x8, y);
    }
  if constexpr (!KV) {
#pragma unroll
    for (int n = 0; n < NS; ++n) asm volatile("" : "+v"(lse[n]), "+v"(dd[n]));
  }
  if (t0 < t1) load_tile(t0);

  const int ro = li * T::kRow + ((hl ^ T::swz(li)) << 4);                 // chunk 2 kk + hl of row li: ro ^ (kk << 5)
  int tro;                                                                // transposing reads: dims 32 d at tro ^ (d << 6)
  {
    const int g = lane >> 4, s = lane & 15, row = 4 * (g >> 1) + (s >> 2), col = 16 * (g & 1) + 4 * (s & 3);
    tro = row * T::kRow + (((col >> 3) ^ T::swz(row)) << 4) + (col & 7) * 2;
  }
  const float c = p.scale * AB_LOG2E;
  floatx16 acc1[NS][kSub] = {};                                           // dq or dk
  floatx16 acc2[KV ? NS : 1][kSub] = {};                                  // dv
  float poison[NS] = {};

  for (int t = t0; t < t1; ++t) {
    const int j0 = u_lo + t * ATT_BN;
    unsigned char* const xs = smem + (t & 1) * 2 * T::kBytes;
    unsigned char* const ys = xs + T::kBytes;
    const float* const lse_l = reinterpret_cast<const float*>(rowv + (t & 1) * 512);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const bool wg_partial = j0 < a_lo || j0 + ATT_BN > a_hi;              // for some row of the workgroup
    if (wg_partial) {
      // this wave's 16 rows of the tile: cleared where no row sees them, or where they hold something that is not finite
      const int row = 16 * wave + (lane >> 2), at = row * T::kRow + (lane & 3) * (T::kRow / 4);
      u32x4* const x = reinterpret_cast<u32x4*>(xs + at);
      u32x4* const y = reinterpret_cast<u32x4*>(ys + at);
      const bool past = j0 + row >= u_hi;
      unsigned bad = 0;
#pragma unroll
      for (int e = 0; e < T::kRow / 64; ++e) {
        bad |= not_finite2(x[e][0]) | not_finite2(x[e][1]) | not_finite2(x[e][2]) | not_finite2(x[e][3]);
        if constexpr (KV) bad |= not_finite2(y[e][0]) | not_finite2(y[e][1]) | not_finite2(y[e][2]) | not_finite2(y[e][3]);
      }
      const unsigned long long any = __ballot(bad != 0u && !past);
      if (past || ((any >> (lane & ~3)) & 15ull) != 0ull) {
#pragma unroll
        for (int e = 0; e < T::kRow / 64; ++e) {
          x[e] = u32x4{0u, 0u, 0u, 0u};
          if constexpr (KV) y[e] = u32x4{0u, 0u, 0u, 0u};
        }
      }
      const unsigned long long rows16 = __ballot(lane < 16 && ((any >> (4 * (lane & 15))) & 15ull) != 0ull);
      if (lane == 0) ctl[16 + (t & 1) * 4 + wave] = (int)rows16;
    }
    ATT_BARRIER();
    if (t + 1 < t1) load_tile(t + 1);
    if (rows_valid <= 0) continue;                                        // a wave without rows moves tiles only
    unsigned long long vis[NS];
    bool partial = false;
    if (wg_partial) {
      const int* bw = ctl + 16 + (t & 1) * 4;
      const unsigned long long bad = (unsigned long long)(unsigned)(uni(bw[0]) | uni(bw[1]) << 16) |
                                     (unsigned long long)(unsigned)(uni(bw[2]) | uni(bw[3]) << 16) << 32;
      bool cutoff = bad != 0ull;
#pragma unroll
      for (int n = 0; n < NS; ++n) {
        // the tile's rows that this lane's row sees; one that sees nothing asks for no mask (what it sums is not used)
        const int a = min(max(rr[n].lo - j0, 0), 64), z = min(max(rr[n].hi - j0, 0), 64);
        const unsigned long long below_a = a >= 64 ? ~0ull : (1ull << a) - 1, below_z = z >= 64 ? ~0ull : (1ull << z) - 1;
        vis[n] = below_z & ~below_a;
        cutoff = cutoff || (rr[n].hi > rr[n].lo && ~vis[n] != 0ull);
        if constexpr (KV) {
          if (bad != 0ull) {
            for (int x = 0; x < 64; ++x)
              if ((bad >> x) & (vis[n] >> x) & 1ull) {
                const float l = lse_l[x], d = lse_l[64 + x];
                if (l != l || !__builtin_isfinite(d)) poison[n] = NAN;
              }
          }
        }
        vis[n] = (vis[n] & ~bad) >> (4 * hl);
      }
      partial = __ballot(cutoff) != 0ull;
    }

#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      // S and dP of 32 rows of the tile
      floatx16 s[NS] = {}, dp[NS] = {};
      {
        bf16x8 a[2 * kSteps];
        auto op = [&](int x) __attribute__((always_inline)) {
          a[x] = *reinterpret_cast<const bf16x8*>(((x & 1) ? ys : xs) + sub * 32 * T::kRow + (ro ^ ((x >> 1) << 5)));
        };
#pragma unroll
        for (int x = 0; x < AB_AHEAD; ++x) op(x);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < 2 * kSteps; ++x) {
          if (x + AB_AHEAD < 2 * kSteps) op(x + AB_AHEAD);
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            if (x & 1) dp[n] = mfma32x32x16(a[x], b2[n][x >> 1], dp[n]);
            else s[n] = mfma32x32x16(a[x], b1[n][x >> 1], s[n]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      // P and dS, rounded to bf16, the matrix instruction's type (2^-9 of a weight), as in the forward
      bf16x8 pf[NS][2], df[NS][2];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        floatx4 l4, d4;
        if constexpr (KV) {
          l4 = *reinterpret_cast<const floatx4*>(lse_l + 32 * sub + 8 * g + 4 * hl);
          d4 = *reinterpret_cast<const floatx4*>(lse_l + 64 + 32 * sub + 8 * g + 4 * hl);
        }
#pragma unroll
        for (int n = 0; n < NS; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int e = 4 * g + x;
            const float pr = __builtin_amdgcn_exp2f(fmaf(s[n][e], c, KV ? -l4[x] : -lse[n]));
            if constexpr (KV) pf[n][e >> 3][e & 7] = (bf16)pr;
            df[n][e >> 3][e & 7] = (bf16)(pr * (dp[n][e] - (KV ? d4[x] : dd[n])));
          }
      }
      if (partial) {
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          const int wd = (int)(unsigned)(vis[n] >> (32 * sub));
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            u32x4 d = __builtin_bit_cast(u32x4, df[n][m]), pp = d;
            if constexpr (KV) pp = __builtin_bit_cast(u32x4, pf[n][m]);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
              const int i = 8 * m + e, bit = 8 * (i >> 2) + (i & 3);      // element i is row bit (+ 4 hl) of the 32
              const unsigned keep = bit_select(0xffffu, (unsigned)__builtin_amdgcn_sbfe(wd, bit, 1),
                                               (unsigned)__builtin_amdgcn_sbfe(wd, bit + 1, 1));
              d[e >> 1] &= keep;
              if constexpr (KV) pp[e >> 1] &= keep;
            }
            df[n][m] = __builtin_bit_cast(bf16x8, d);
            if constexpr (KV) pf[n][m] = __builtin_bit_cast(bf16x8, pp);
          }
        }
      }
      // dq^T (dk^T) += X^T dS, dv^T += Y^T P
      {
        constexpr int kOps = 2 * kSub * (KV ? 2 : 1);
        bf16x8 a[kOps];
        auto op = [&](int x) __attribute__((always_inline)) {
          const int d = (KV ? x >> 1 : x) % kSub, m = (KV ? x >> 1 : x) / kSub;
          const unsigned char* at = (KV && (x & 1) ? ys : xs) + (32 * sub + 16 * m) * T::kRow;
          const rt_v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((rt_lds_v4s)(at + (tro ^ (d << 6))));
          const rt_v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((rt_lds_v4s)(at + (tro ^ (d << 6) ^ 32) + 8 * T::kRow));
          const short __attribute__((ext_vector_type(8))) a8 = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          a[x] = __builtin_bit_cast(bf16x8, a8);
        };
#pragma unroll
        for (int x = 0; x < AB_AHEAD; ++x) op(x);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < kOps; ++x) {
          if (x + AB_AHEAD < kOps) op(x + AB_AHEAD);
          const int d = (KV ? x >> 1 : x) % kSub, m = (KV ? x >> 1 : x) / kSub;
#pragma unroll
          for (int n = 0; n < NS; ++n) {
            if (KV && (x & 1)) acc2[n][d] = mfma32x32x16(a[x], pf[n][m], acc2[n][d]);
            else acc1[n][d] = mfma32x32x16(a[x], df[n][m], acc1[n][d]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }

  // ---- results ----
  if (rows_valid <= 0) return;
  unsigned char* const scratch = scratch_all + wave * AB_SCRATCH_WAVE;
#pragma unroll
  for (int n = 0; n < NS; ++n) {
    const int valid = min(32, n_st - r0 - 32 * n), rn = r0 + 32 * n;
    if (valid <= 0) break;
    float f1 = p.scale, f2 = 1.f;
    if (rr[n].hi <= rr[n].lo) {                                           // whatever it holds of tiles that others see whole
#pragma unroll
      for (int d = 0; d < kSub; ++d) {
        acc1[n][d] = floatx16{};
        if constexpr (KV) acc2[n][d] = floatx16{};
      }
    } else if constexpr (KV) {
      f1 += poison[n];
      f2 += poison[n];
    } else if (lse[n] != lse[n] || !__builtin_isfinite(dd[n])) {
      f1 = NAN;
    }
    auto finish = [&](const floatx16* acc, float f, const OutView& out, float* part) {
      if (n_split == 1) {
        if (out.p != nullptr) store_wave<D>(out, KV ? FastDiv{1u, 0u, 1u, 0u} : p.by_g, scratch, acc, f, b, hk, rn, valid);
      } else if (part != nullptr && li < valid) {
        float* dst = part + (((int64_t)split * BH + bh) * n_st + rn + li) * D + 4 * hl;
#pragma unroll
        for (int d = 0; d < kSub; ++d)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<floatx4*>(dst + 32 * d + 8 * g) =
                floatx4{acc[d][4 * g] * f, acc[d][4 * g + 1] * f, acc[d][4 * g + 2] * f, acc[d][4 * g + 3] * f};
      }
    };
    if constexpr (KV) {
      finish(acc1[n], f1, p.dk, p.dk_part);
      finish(acc2[n], f2, p.dv, p.dv_part);
    } else {
      finish(acc1[n], f1, p.dq, p.dq_part);
    }
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
#pragma unroll 4
  for (int i = 1; i < n_split; ++i) {
    const floatx4 v = *reinterpret_cast<const floatx4*>(src + (int64_t)i * rows * D);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += v[e];
  }
  const int bh = (int)(row / n_st), r = (int)(row - (int64_t)bh * n_st);
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
#define AB_MIN_TILES 8                                // of the walked side that a part is worth

namespace {

// Parts: as many as make the rounds of workgroups come out shortest, each part's sums costing a few per cent of a round
int parts(int64_t items, int64_t tiles, int slots) {
  int best = 1;
  double time = 0.;
  for (int n = 1; n <= AB_MAX_SPLIT && (n == 1 || tiles / n >= AB_MIN_TILES); ++n) {
    if (n > 1 && items * n > 8 * slots) break;
    const double t = (double)((items * n + slots - 1) / slots) / n + 0.01 * n;
    if (n == 1 || t < time) { time = t; best = n; }
  }
  return best;
}

constexpr int kNS = 2;
constexpr int kBlockRows = 32 * kNS * AB_WAVES;

int64_t blocks(int64_t rows) { return (rows + kBlockRows - 1) / kBlockRows; }

template <int D>
hipError_t run_bwd(const AttnBwdParams& p, hipStream_t stream) {
  static std::atomic<unsigned> set_q{0u}, set_k{0u};
  hipError_t e = ensure_lds_limit(reinterpret_cast<const void*>(icsa_attn_bwd_kernel<D, false, kNS>), ab_lds(D), &set_q);
  if (e != hipSuccess) return e;
  e = ensure_lds_limit(reinterpret_cast<const void*>(icsa_attn_bwd_kernel<D, true, kNS>), ab_lds(D), &set_k);
  if (e != hipSuccess) return e;
  const int64_t BH = (int64_t)p.B * p.Hk, n_q = (int64_t)p.Sq * (p.H / p.Hk);
  const int64_t wq = BH * blocks(n_q) * p.q_split, wk = BH * blocks(p.Sk) * p.k_split;
  const int64_t jq = (BH * n_q * D + 1023) / 1024, jk = (BH * p.Sk * D + 1023) / 1024;
  if (wq > 0x3fffffffLL || wk > 0x3fffffffLL || (p.q_split > 1 && jq > 0x7fffffffLL) || (p.k_split > 1 && jk > 0x7fffffffLL))
    return hipErrorInvalidValue;
  if (wq > 0) {                                       // without queries dk and dv are zeros, which the key-major kernel writes
    hipLaunchKernelGGL((icsa_attn_bwd_kernel<D, false, kNS>), dim3(xcd_grid((int)wq)), dim3(AB_THREADS), ab_lds(D), stream, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (p.q_split > 1 && p.dq.p != nullptr) {
    hipLaunchKernelGGL((icsa_attn_bwd_join_kernel<D, false>), dim3((unsigned)jq), dim3(256), 0, stream, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  if (p.dk.p == nullptr && p.dv.p == nullptr) return hipSuccess;
  hipLaunchKernelGGL((icsa_attn_bwd_kernel<D, true, kNS>), dim3(xcd_grid((int)wk)), dim3(AB_THREADS), ab_lds(D), stream, p);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  if (p.k_split > 1) hipLaunchKernelGGL((icsa_attn_bwd_join_kernel<D, true>), dim3((unsigned)jk, 2), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

AttnBwdPlan attn_bwd_plan(int B, int Sq, int Sk, int H, int Hk, int D) {
  (void)D;
  const int64_t BH = (int64_t)B * Hk, n_q = (int64_t)Sq * (H / Hk);
  return AttnBwdPlan{parts(BH * blocks(n_q), (Sk + ATT_BN - 1) / ATT_BN, AB_CUS), parts(BH * blocks(Sk), (n_q + ATT_BN - 1) / ATT_BN, AB_CUS)};
}

hipError_t launch_attn_bwd(AttnBwdParams p, hipStream_t stream) {
  const int G = p.H / p.Hk;
  p.by_g = fast_div(G);
  p.by_hk = fast_div(p.Hk);
  p.by_qblk = fast_div((unsigned)std::max<int64_t>(1, blocks((int64_t)p.Sq * G)));
  p.by_kblk = fast_div((unsigned)std::max<int64_t>(1, blocks(p.Sk)));
  return p.D == 128 ? run_bwd<128>(p, stream) : run_bwd<64>(p, stream);
}
