// Attention under masks: softmax over the visible keys of cap tanh(scale q.k / cap) + bias(distance).
//
// Which keys a query sees is one range [lo, hi) of the sequence: its document's keys, cut at the
// query's own position (causal, aligned at the document's end) or at the document's prefix, whichever is
// further.  A row of work is a (query, head) pair; the H / Hk heads that share a key head are consecutive rows, so
// a tile of keys serves them all (one query token of a group is one tile of rows).
//
// A workgroup of 4 waves takes 128 rows of one (batch, key head) over the 64-key tiles of the union of
// their ranges, or over one of n_split equal parts of it (icsa_masked_combine_kernel joins the parts): where rows are few, and
// for the items of a last, incomplete round.  Only tiles that some row sees in part are masked.  Scores are
// computed transposed, S^T = K Q^T: a lane holds one row and 32 of a tile's 64 keys, the other 32 are in lane ^ 32
// (attn_tile.h).  P goes to the second product from its registers; V is read transposed from its row-major tile.
//
// K and V tiles arrive by direct global->LDS loads, two buffers, one barrier a tile: behind it the next tile is
// requested into the buffer that everybody has left.  Two workgroups share a CU, three with heads of 64: one's exponentials run
// beside another's products.  Products read their operands from LDS four ahead of their use, with raised priority.
//
// Values in masked places: scores are replaced, not added to, so a NaN of a masked key does not
// matter; V rows that no row of the workgroup sees are cleared in LDS; and where a partly visible tile holds
// a V that is not finite, 0 * V would reach rows that do not see it: such values are cleared too, and added at
// the end to the rows that see them.
//
// What bounds it (two waves a SIMD with heads of 128, three with 64): the vector instructions and the products of a tile side by
// side, 550 to 800 and 1,024 cycles a wave with heads of 128, and the clock, 1.7 to 2.1 GHz under them; capped scores add two
// transcendentals an element.  9,373 tokens, 12 heads of 128: dense 525 us (1.03 PFLOP/s in two rounds of workgroups, the second 73 %
// full), causal 282 (0.96), a prefix and capped scores 375 to 415 (matrix pipe busy 36 %, vector pipe 54 %: neither is full, a
// SIMD's waves do not keep to opposite phases by themselves); 32,760 tokens, 5 heads 2.41 ms (1.14); 9,373 tokens, 12 heads
// of 64 301 us (0.90).  One query of 40 heads over 8 key heads of 65,536 keys: 43 us for 268 MB and 6 for joining 64 parts.  Short
// documents (packed prompts of 350 keys, 40 heads, 32,760 queries: 314 to 346 us) add the way of Q and the output
// through memory, 140 us at the copy rate, and each workgroup's start, which two workgroups a CU do not hide.
// Tried and slower: the next tile's scores between the exponentials of the one at hand (dense 541 -> 564 us; heads of 64 310 -> 357);
// several items a workgroup; tanh as a polynomial where x is small (prefix 415 -> 429).  A second way through the loop for
// values that are not finite made the compiler copy O every tile: dense 605 us.
#include "attn_rows.h"

#define MA_THREADS 256
#define MA_WAVES 4
#define MA_SCRATCH_WAVE 2048                          // per wave: staged output rows
#define MA_CTL_BYTES 256                              // per-wave ranges, a flag
#define MA_PSUM_MAX 18446744073709551616.0f           // as in the dense kernel: the reference max is raised past it
#define MA_M_NONE (-3.4028234663852886e38f)           // finite: a tile without visible keys leaves O = l = 0
#define MA_LOG2E 1.4426950408889634f
#define MA_CUS 256
#define MA_MAX_SPLIT 256
#define MA_FEW_PARTS 16                               // from so many parts on a row's are shared by thread groups
#define MA_TAIL_ROUNDS 8                              // up to so many rounds a last, incomplete one is cut in parts
#define MA_TAIL_TILES 32                              // from so many key tiles on
#define MA_MIN_SPLIT_TILES 4                          // key tiles a split part is worth
#define MA_BIAS_MARGIN ATT_BN
#define MA_AHEAD 4                                    // operands read ahead; 2, 3 and 5 measured alike or up to 3 % slower
#define MA_LDS_MAX (160 * 1024)

namespace {

template <int D> struct Tile {
  static constexpr int kRow = D * 2, kBytes = ATT_BN * kRow, kChunks = D / 8;
  static constexpr int kRowsPerLoad = 1024 / kRow, kLoads = 16 / kRowsPerLoad;   // of a wave's 16 rows
  // 16-byte chunk c of row r sits at c ^ kswz(r) in a K tile: 16 rows' reads of one chunk touch
  // every bank once; at c ^ vswz(r) in a V tile, for the transposing reads
  static __device__ __forceinline__ int kswz(int r) { return D == 128 ? (r & 15) : ((r >> 1) & 7); }
  static __device__ __forceinline__ int vswz(int r) { return D == 128 ? (r & 3) << 2 : ((r >> 1) & 1) << 2; }
};

// Workgroups a CU holds: registers for three with heads of 64 (4 x 512 tokens of 64 heads with bias and documents 42.5 us with
// two, 40.0 with three)
__host__ __device__ constexpr int ma_wg_per_cu(int D) { return D == 64 ? 3 : 2; }

__host__ __device__ __forceinline__ int ma_fixed_lds(int D) { return 4 * ATT_BN * D * 2 + MA_WAVES * MA_SCRATCH_WAVE + MA_CTL_BYTES; }

// Sum of a lane's 32 probabilities as they go into the second product.  They are rounded to bf16, the matrix instruction's type, as
// in the framework's other attention kernels (2^-8 of a weight at most; 0.0023 of the outputs in the 2-norm with the outputs' own
// rounding, 0.0017 without): where few keys carry a row, what their rounding adds to the product it adds to the sum, and the
// quotient does not see it.  Two values an instruction.
__device__ __forceinline__ float sum_p(const bf16x8 pf[4]) {
  const bf16x2 one = {(bf16)1.f, (bf16)1.f};
  float r[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    r[m] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e += 2) r[m] = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{pf[m][e], pf[m][e + 1]}, one, r[m], false);
  }
  return (r[0] + r[1]) + (r[2] + r[3]);
}

}  // namespace

template <int D, bool kCap, bool kBias>
__global__ void __launch_bounds__(MA_THREADS, ma_wg_per_cu(D)) icsa_masked_attn_kernel(MaskedAttnParams p) {
  typedef Tile<D> T;
  constexpr int kSteps = D / 16, kSub = D / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* const scratch_all = smem + 4 * T::kBytes;
  int* const ctl = reinterpret_cast<int*>(scratch_all + MA_WAVES * MA_SCRATCH_WAVE);   // ranges of the 4 waves, a flag
  float* const bias_lds = reinterpret_cast<float*>(scratch_all + MA_WAVES * MA_SCRATCH_WAVE + MA_CTL_BYTES);
  const int lane = threadIdx.x & 63, li = lane & 31, hl = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = p.by_g.d, n_rows = p.Sq * G, n_blk = p.by_blk.d;
  // Whole items, then parts of items.  Alike ones: each list dealt to the XCDs in runs, a head's items side by side.  Under a causal
  // mask: the longest rows of every head first, so that the last items to start are short ones; workgroups go round the
  // XCDs, so an XCD has the same few heads all the way.
  const int BH = p.B * p.Hk, n_parts = (BH * n_blk - p.n_whole) * p.n_split, whole_wg = xcd_grid(p.n_whole);
  const bool cut = (int)blockIdx.x >= whole_wg;
  int w = cut ? blockIdx.x - whole_wg : blockIdx.x;
  if (!p.causal) w = xcd_remap(w, cut ? n_parts : p.n_whole);
  if (w < 0 || w >= (cut ? n_parts : p.n_whole)) return;
  const int item = cut ? p.n_whole + (int)p.by_split.div(w) : w, split = cut ? (int)p.by_split.mod(w) : 0;
  const int blk = n_blk - 1 - (int)(p.causal ? p.by_bh.div(item) : p.by_blk.mod(item)), bh = p.causal ? p.by_bh.mod(item) : p.by_blk.div(item);
  const int b = p.by_hk.div(bh), hk = p.by_hk.mod(bh);
  const int r0 = blk * MA_ROWS + 32 * wave;
  const int rows_valid = min(32, n_rows - r0);

  bf16x8 qf[kSteps];
  {
    const bf16* src = p.q + row_at(p.q_sb, p.q_ss, p.q_sh, b, hk, p.by_g, min(r0 + li, n_rows - 1)) + 8 * hl;
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk) qf[kk] = *reinterpret_cast<const bf16x8*>(src + 16 * kk);
  }

  // the heads' bias tables, their ends repeated over a tile's width: the first values requested here, with the rows' borders
  const int bias_width = 2 * p.radius + 1, bias_row = bias_width + 2 * MA_BIAS_MARGIN;
  auto bias_value = [&](int x) {
    const int h = G == 1 ? 0 : x / bias_row, at = x - h * bias_row;
    return p.bias[(int64_t)(hk * G + h) * bias_width + min(max(at - MA_BIAS_MARGIN, 0), bias_width - 1)];
  };
  float bias_first[2] = {0.f, 0.f};
  if constexpr (kBias) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (threadIdx.x + MA_THREADS * i < (unsigned)(G * bias_row)) bias_first[i] = bias_value(threadIdx.x + MA_THREADS * i);
  }

  // ---- what the rows see ----
  RowRange rr = row_range(p, b, G == 1 ? r0 + li : p.by_g.div(r0 + li));
  if (li >= rows_valid) rr = RowRange{0, 0, 0};
  {
    const bool any = rr.hi > rr.lo;
    int lo = any ? rr.lo : 0x7fffffff, hi = any ? rr.hi : 0, in_lo = any ? rr.lo : 0, in_hi = any ? rr.hi : 0x7fffffff;
    if (__ballot(rr.lo != __builtin_amdgcn_readfirstlane(rr.lo) || rr.hi != __builtin_amdgcn_readfirstlane(rr.hi)) != 0ull) {
      lo = wave_min(lo);                               // unless all rows see the same
      hi = wave_max(hi);
      in_lo = wave_max(in_lo);
      in_hi = wave_min(in_hi);
    }
    if (lane == 0) { ctl[wave] = lo; ctl[4 + wave] = hi; ctl[8 + wave] = in_lo; ctl[12 + wave] = in_hi; }
    if (threadIdx.x == 0) ctl[16] = 0;
  }
  const float c = p.scale * MA_LOG2E;
  if constexpr (kBias) {
    int i = 0;
    for (int x = threadIdx.x; x < G * bias_row; x += MA_THREADS, ++i) {
      const float f = i == 0 ? bias_first[0] : i == 1 ? bias_first[1] : bias_value(x);
      // a type's lowest value stays finite in units of log2 (biases past 2^128 / log2(e) = 2.36e38 are one); infinities and
      // NaN are kept
      bias_lds[x] = !__builtin_isfinite(f) ? f : fminf(fmaxf(f * MA_LOG2E, -3.4028234663852886e38f), 3.4028234663852886e38f);
    }
  }
  __syncthreads();
  // keys that some row sees, [u_lo, u_hi), and keys that every row (that sees any) sees, [a_lo, a_hi)
  auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  const int u_lo = uni(min(min(ctl[0], ctl[1]), min(ctl[2], ctl[3]))), u_hi = uni(max(max(ctl[4], ctl[5]), max(ctl[6], ctl[7])));
  const int a_lo = uni(max(max(ctl[8], ctl[9]), max(ctl[10], ctl[11]))), a_hi = uni(min(min(ctl[12], ctl[13]), min(ctl[14], ctl[15])));
  int t0 = 0, t1 = 0;                                  // tiles from key u_lo on
  if (u_hi > u_lo) {
    t1 = (u_hi - u_lo + ATT_BN - 1) / ATT_BN;
    if (cut) {                                         // equal parts, the first ones a tile longer
      const int q = p.by_split.div(t1), more = t1 - q * p.n_split;
      t0 = q * split + min(split, more);
      t1 = t0 + q + (split < more);
    }
  }
  const int key0 = u_lo + t0 * ATT_BN;

  // ---- loads ----
  const bf16* kb = p.k + (int64_t)b * p.k_sb + (int64_t)hk * p.k_sh;
  const bf16* vb = p.v + (int64_t)b * p.v_sb + (int64_t)hk * p.v_sh;
  int kofs[T::kLoads], vofs[T::kLoads];
#pragma unroll
  for (int i = 0; i < T::kLoads; ++i) {
    const int r = 16 * wave + T::kRowsPerLoad * i + lane / T::kChunks, ch = lane % T::kChunks;
    kofs[i] = (int)((r * p.k_ss + 8 * (ch ^ T::kswz(r))) * 2);
    vofs[i] = (int)((r * p.v_ss + 8 * (ch ^ T::vswz(r))) * 2);
  }
  const unsigned lds0 = lds_u32(smem);
  auto kbuf = [&](int t) { return smem + (t & 1) * T::kBytes; };
  auto vbuf = [&](int t) { return smem + (2 + (t & 1)) * T::kBytes; };
  // the next tile's: addresses and lengths move on by a tile (64-bit products would take 60 scalar instructions)
  const int k_row = (int)p.k_ss * 2, v_row = (int)p.v_ss * 2;
  unsigned long long k_at = (unsigned long long)(kb + (int64_t)key0 * p.k_ss), v_at = (unsigned long long)(vb + (int64_t)key0 * p.v_ss);
  int left = p.Sk - key0;
  auto load_tile = [&](int t) __attribute__((always_inline)) {
    const int rows = min(ATT_BN, left) - 1;
    const u32x4 krs = {(unsigned)k_at, (unsigned)(k_at >> 32) & 0xffffu, (unsigned)(rows * k_row + 2 * D), 0x00020000u};
    const u32x4 vrs = {(unsigned)v_at, (unsigned)(v_at >> 32) & 0xffffu, (unsigned)(rows * v_row + 2 * D), 0x00020000u};
    const unsigned at = lds0 + (t & 1) * T::kBytes + wave * 16 * T::kRow;
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) lds_dma16(at + 1024 * i, kofs[i], krs);
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) lds_dma16(at + 2 * T::kBytes + 1024 * i, vofs[i], vrs);
    k_at += (unsigned)(ATT_BN * k_row);
    v_at += (unsigned)(ATT_BN * v_row);
    left -= ATT_BN;
  };
  if (t0 < t1) load_tile(t0);

  int kro[kSteps], vro[kSub];                        // operand read offsets (bytes); + 32 rows a sub-tile
#pragma unroll
  for (int kk = 0; kk < kSteps; ++kk) kro[kk] = li * T::kRow + (((2 * kk + hl) ^ T::kswz(li)) << 4);
#pragma unroll
  for (int ds = 0; ds < kSub; ++ds) {
    const int g = lane >> 4, s = lane & 15, row = 4 * (g >> 1) + (s >> 2), col = 32 * ds + 16 * (g & 1) + 4 * (s & 3);
    vro[ds] = row * T::kRow + (((col >> 3) ^ T::vswz(row)) << 4) + (col & 7) * 2;
  }
  unsigned char* const scratch = scratch_all + wave * MA_SCRATCH_WAVE;
  const float* const my_bias = kBias ? bias_lds + (G == 1 ? 0 : p.by_g.mod(r0 + li)) * bias_row + MA_BIAS_MARGIN + p.radius : nullptr;

  floatx16 o[kSub] = {};
  float m_ref = MA_M_NONE, l_run = 0.f;
  bool first = true;
  // a row that sees nothing, or does not exist, asks for no mask of its own: its scores are masked
  // whenever the others' are, and what it holds is not used
  const bool some = rr.hi > rr.lo;
  const int see_lo = some ? rr.lo : 0, see_hi = some ? rr.hi : 0x7fffffff;

  for (int t = t0; t < t1; ++t) {
    const int j0 = u_lo + t * ATT_BN;
    unsigned char* const ks = kbuf(t);
    unsigned char* const vs = vbuf(t);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const bool wg_partial = j0 < a_lo || j0 + ATT_BN > a_hi;            // for some row of the workgroup
    if (wg_partial) {
      // this wave's 16 V rows: those that no row sees cleared, the others looked at
      const int row = 16 * wave + (lane >> 2), key = j0 + row;
      u32x4* own = reinterpret_cast<u32x4*>(vs + row * T::kRow + (lane & 3) * (T::kRow / 4));
      unsigned bad = 0;
      if (key >= u_hi) {
#pragma unroll
        for (int e = 0; e < T::kRow / 64; ++e) own[e] = u32x4{0u, 0u, 0u, 0u};
      } else {
#pragma unroll
        for (int e = 0; e < T::kRow / 64; ++e) bad |= not_finite2(own[e][0]) | not_finite2(own[e][1]) | not_finite2(own[e][2]) | not_finite2(own[e][3]);
      }
      if (__ballot(bad != 0u) != 0ull) {
        if (lane == 0) ctl[16] = 1;
        if (bad != 0u) {
#pragma unroll 1
          for (int e = 0; e < T::kRow / 4; e += 4) {
            unsigned short* const x = reinterpret_cast<unsigned short*>(own) + e / 2;
            const unsigned y = *reinterpret_cast<const unsigned*>(x), m = not_finite2(y);
            if (m & 0x8000u) x[0] = 0;
            if (m & 0x80000000u) x[1] = 0;
          }
        }
      }
    }
    ATT_BARRIER();
    if (t + 1 < t1) load_tile(t + 1);
    if (rows_valid <= 0) continue;                                     // a wave without rows moves tiles only
    const bool partial = wg_partial && __ballot(j0 < see_lo || j0 + ATT_BN > see_hi) != 0ull;   // for some row of the wave

    // operands are read MA_AHEAD products ahead of their use
    floatx16 s[2] = {};
    {
      bf16x8 ka[2 * kSteps];
      auto k_op = [&](int x) __attribute__((always_inline)) { ka[x] = *reinterpret_cast<const bf16x8*>(ks + kro[x >> 1] + (x & 1) * 32 * T::kRow); };
#pragma unroll
      for (int x = 0; x < MA_AHEAD; ++x) k_op(x);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int x = 0; x < 2 * kSteps; ++x) {
        if (x + MA_AHEAD < 2 * kSteps) k_op(x + MA_AHEAD);
        s[x & 1] = mfma32x32x16(ka[x], qf[x >> 1], s[x & 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
    }
    // Scores in units of log2, as base + mul * s.  Capped: cap tanh(x) = cap - 2 cap r with r = 1 / (1 + exp(2 x)), so
    // s becomes r; with a bias s becomes the score itself.
    const float in = kCap ? 2.f * MA_LOG2E * p.scale / p.softcap : 0.f, top = kCap ? p.softcap * MA_LOG2E : 0.f;
    if constexpr (kCap) {
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[sub][i] = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s[sub][i] * in));
    }
    if constexpr (kBias) {
      const int d0 = j0 - rr.at + 4 * hl, R = p.radius;
      const float f = kCap ? -2.f * top : c;
      if (__ballot(!(d0 >= R || d0 + ATT_BN <= -R)) == 0ull) {           // the whole tile past the table's ends
        const float end = my_bias[d0 > 0 ? R : -R], x = kCap ? end + top : end;
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[sub][i] = fmaf(s[sub][i], f, x);
      } else {
        // a row's 64 distances lie inside the table and its margins, or are past one end alike
        const float* t = my_bias + min(max(d0, -R - MA_BIAS_MARGIN + 4 * hl), R + 4 * hl);
#pragma unroll
        for (int sub = 0; sub < 2; ++sub)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float x = t[32 * sub + 8 * (i >> 2) + (i & 3)];
            s[sub][i] = fmaf(s[sub][i], f, kCap ? x + top : x);
          }
      }
    }
    const float base = kBias || !kCap ? 0.f : top, mul = kBias ? 1.f : kCap ? -2.f * top : c;
    if (partial) {
      // keys outside [lo, hi) as one 64-bit word: element i of sub-tile sub is key 32 sub + 8 (i / 4) + 4 hl + i % 4
      const int a = min(max(rr.lo - j0, 0), 64), z = min(max(rr.hi - j0, 0), 64);
      const unsigned long long below_a = a >= 64 ? ~0ull : (1ull << a) - 1, below_z = z >= 64 ? ~0ull : (1ull << z) - 1;
      const unsigned long long mw = ~(below_z & ~below_a) >> (4 * hl);
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const unsigned wd = (unsigned)(mw >> (32 * sub));
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int kbit = 8 * (i >> 2) + (i & 3);
          const unsigned all = (unsigned)__builtin_amdgcn_sbfe((int)wd, kbit, 1);    // the bit, over the whole word
          // score -inf: s is -inf, or +inf where the factor is negative
          s[sub][i] = __uint_as_float(bit_select(all, kCap && !kBias ? 0x7f800000u : 0xff800000u, __float_as_uint(s[sub][i])));
        }
      }
    }
    bf16x8 pf[4];
    float rs = 0.f;
    if (!first) {
      const float off = base - m_ref;
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int i = 0; i < 16; ++i) pf[2 * sub + (i >> 3)][i & 7] = (bf16)__builtin_amdgcn_exp2f(fmaf(s[sub][i], mul, off));
      rs = sum_p(pf);
    }
    if (first || __ballot(!(rs <= MA_PSUM_MAX)) != 0ull) {
      float mx = -INFINITY;
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, kCap && !kBias ? -s[sub][i] : s[sub][i]);
      mx = fmaf(xhalf_max(mx), fabsf(mul), base);
      const float mn = mx > m_ref ? mx : m_ref;
      const float al = __builtin_amdgcn_exp2f(m_ref - mn);
#pragma unroll
      for (int ds = 0; ds < kSub; ++ds)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[ds][i] *= al;
      l_run *= al;
      m_ref = mn;
      const float off = base - m_ref;
#pragma unroll
      for (int sub = 0; sub < 2; ++sub)
#pragma unroll
        for (int i = 0; i < 16; ++i) pf[2 * sub + (i >> 3)][i & 7] = (bf16)__builtin_amdgcn_exp2f(fmaf(s[sub][i], mul, off));
      rs = sum_p(pf);
      first = false;
    }
    l_run += rs;

    {
      bf16x8 va[4 * kSub];
      auto v_op = [&](int x) __attribute__((always_inline)) {
        const unsigned char* at = vs + vro[x % kSub] + x / kSub * 16 * T::kRow;
        const rt_v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((rt_lds_v4s)at);
        const rt_v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((rt_lds_v4s)(at + 8 * T::kRow));
        const short __attribute__((ext_vector_type(8))) a8 = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        va[x] = __builtin_bit_cast(bf16x8, a8);
      };
#pragma unroll
      for (int x = 0; x < MA_AHEAD; ++x) v_op(x);
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int x = 0; x < 4 * kSub; ++x) {
        if (x + MA_AHEAD < 4 * kSub) v_op(x + MA_AHEAD);
        o[x % kSub] = mfma32x32x16(va[x], pf[x / kSub], o[x % kSub]);
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
    }
  }

  if (rows_valid <= 0) return;
  if (uni(ctl[16]) != 0) {                             // what was cleared, from memory, to the rows that see it
    for (int t = t0; t < t1; ++t) {
      const int j0 = u_lo + t * ATT_BN;
      if (j0 >= a_lo && j0 + ATT_BN <= a_hi) continue;
#pragma unroll 1
      for (int key = j0; key < min(j0 + ATT_BN, u_hi); ++key) {
        const bool vis = key >= rr.lo && key < rr.hi;
#pragma unroll
        for (int ds = 0; ds < kSub; ++ds)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const bf16x4 v4 = *reinterpret_cast<const bf16x4*>(vb + (int64_t)key * p.v_ss + 32 * ds + 8 * g + 4 * hl);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float v = (float)v4[e];
              o[ds][4 * g + e] += vis && !__builtin_isfinite(v) ? v : 0.f;
            }
          }
      }
    }
  }
  const float l = xhalf_sum(l_run);
  if (!some) {                                         // whatever it holds of tiles that others see whole
#pragma unroll
    for (int ds = 0; ds < kSub; ++ds) o[ds] = floatx16{};
  }
  if (!cut) {
    if (p.lse != nullptr && hl == 0 && li < rows_valid) p.lse[(int64_t)bh * n_rows + r0 + li] = row_lse(m_ref, some ? l : 0.f);
    store_wave<D>(p.out, p.by_g, scratch, o, !some || l == 0.f ? 0.f : __builtin_amdgcn_rcpf(l), b, hk, r0, rows_valid,
                  p.rest, p.Sq, p.H);
  } else if (li < rows_valid) {
    // a row's raw O, reference max and sum: [part][row][D], then [part][2][row]
    float* dst = p.part + ((int64_t)w * MA_ROWS + 32 * wave + li) * D + 4 * hl;
#pragma unroll
    for (int ds = 0; ds < kSub; ++ds)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<floatx4*>(dst + 32 * ds + 8 * g) = floatx4{o[ds][4 * g], o[ds][4 * g + 1], o[ds][4 * g + 2], o[ds][4 * g + 3]};
    if (hl == 0) {
      float* ml = p.part + (int64_t)n_parts * MA_ROWS * D + (int64_t)w * 2 * MA_ROWS + 32 * wave + li;
      ml[0] = some ? m_ref : MA_M_NONE;
      ml[MA_ROWS] = some ? l : 0.f;
    }
  }
}

// Joins the parts of every row, in a fixed order (bitwise reproducible).  256 threads, D / 4 for each of their rows (4 dims a
// thread); kFew, where parts are many and rows few: one row, whose parts the 1024 / D thread groups share.
template <int D, bool kFew>
__global__ void __launch_bounds__(256) icsa_masked_combine_kernel(MaskedAttnParams p) {
  constexpr int kPer = D / 4, kGroups = 256 / kPer, kRows = kFew ? 1 : kGroups;
  __shared__ float wt[MA_MAX_SPLIT][kRows];
  __shared__ __attribute__((aligned(16))) float acc[kFew ? kGroups : 1][D];
  const int G = p.by_g.d, n_rows = p.Sq * G, n_blk = p.by_blk.d, n = p.n_split;
  const int t = threadIdx.x % kPer, grp = threadIdx.x / kPer, x = kFew ? 0 : grp;
  const int x_item = blockIdx.x / (MA_ROWS / kRows), row = blockIdx.x % (MA_ROWS / kRows) * kRows + x, item = p.n_whole + x_item;
  const int BH = p.B * p.Hk, blk = n_blk - 1 - (int)(p.causal ? p.by_bh.div(item) : p.by_blk.mod(item)),
            bh = p.causal ? p.by_bh.mod(item) : p.by_blk.div(item);
  const int r = blk * MA_ROWS + row;
  if (r - x >= n_rows) return;                        // uniform: the block's first row
  const bool on = r < n_rows;
  const int64_t part0 = (int64_t)x_item * n;
  const float* ml = p.part + (int64_t)(BH * n_blk - p.n_whole) * n * MA_ROWS * D + part0 * 2 * MA_ROWS + row;
  // every part's weight 2^(m_s - max), and the sum of the row, by the row's first threads
  float m = MA_M_NONE, l = 0.f;
  for (int s = t; s < n; s += kPer) m = fmaxf(m, on ? ml[(int64_t)s * 2 * MA_ROWS] : MA_M_NONE);
#pragma unroll
  for (int o = kPer / 2; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, kPer));
  for (int s = t; s < n; s += kPer) {
    const float w = on ? __builtin_amdgcn_exp2f(ml[(int64_t)s * 2 * MA_ROWS] - m) : 0.f;
    if (on) l = fmaf(ml[(int64_t)s * 2 * MA_ROWS + MA_ROWS], w, l);
    if (!kFew || grp == 0) wt[s][x] = w;
  }
#pragma unroll
  for (int o = kPer / 2; o >= 1; o >>= 1) l += __shfl_xor(l, o, kPer);
  __syncthreads();
  floatx4 o = {};
  if (on) {
    const float* src = p.part + (part0 * MA_ROWS + row) * D + 4 * t;
    const int s1 = kFew ? n * (grp + 1) / kGroups : n;
#pragma unroll 8
    for (int s = kFew ? n * grp / kGroups : 0; s < s1; ++s) {
      const floatx4 v = *reinterpret_cast<const floatx4*>(src + (int64_t)s * MA_ROWS * D);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(v[e], wt[s][x], o[e]);
    }
  }
  if constexpr (kFew) {
    *reinterpret_cast<floatx4*>(&acc[grp][4 * t]) = o;
    __syncthreads();
    if (grp > 0) return;
#pragma unroll
    for (int y = 1; y < kGroups; ++y)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] += acc[y][4 * t + e];
  }
  if (!on) return;
  if (p.lse != nullptr && t == 0) p.lse[(int64_t)bh * n_rows + r] = row_lse(m, l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t off = row_at(p.out.sb, p.out.ss, p.out.sh, p.by_hk.div(bh), p.by_hk.mod(bh), p.by_g, r) + 4 * t;
  if (p.rest != nullptr) {
    const float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
    *reinterpret_cast<unsigned*>(p.rest + row_at((int64_t)p.Sq * p.H * D, (int64_t)p.H * D, D, p.by_hk.div(bh), p.by_hk.mod(bh), p.by_g, r) +
                                 rest_at<D>(4 * t)) = rest_bytes(v);
  }
  if (p.out.dtype == ICSA_DT_BF16) {
    bf16x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (bf16)(o[e] * inv);
    *reinterpret_cast<bf16x4*>(reinterpret_cast<bf16*>(p.out.p) + off) = y;
  } else {
    *reinterpret_cast<floatx4*>(reinterpret_cast<float*>(p.out.p) + off) = floatx4{o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  }
}

// Which items are whole, and how many parts the others' keys are cut into.  Few items: all in parts, enough to fill the chip
// with workgroups of a few tiles each (rows of a block at most read keys from memory: two workgroups a CU, which leave fewer sums to
// join; one token, 65,536 keys of 8 heads of 64: 32.4 us, with three 36.4).  Some rounds of alike items (no causal mask, no
// documents; else the hardware fills the gaps as items end): the last, incomplete round's items in parts, as many as make the
// rounds come out shortest, where a part is long against its sums' way through memory; rounds of two or three workgroups a CU, which share its
// rate (heads of 64: 16 x 9,373 tokens 381 us by two, 402 by three; 24 x 4,000 over 8,000 keys 228 and 216).
MaskedPlan masked_attn_plan(int B, int Sq, int Sk, int H, int Hk, int D, bool alike) {
  const int64_t rows = (int64_t)Sq * (H / Hk), items = (int64_t)B * Hk * ((rows + MA_ROWS - 1) / MA_ROWS);
  const int tiles = (Sk + ATT_BN - 1) / ATT_BN;
  MaskedPlan f = {(int)items, 1};
  if (items <= 0) return f;
  const int most = MA_CUS * ma_wg_per_cu(D), fill = rows <= MA_ROWS ? 2 * MA_CUS : most;
  if (items * 2 <= fill) {
    int64_t n = (fill + items - 1) / items;
    n = n < tiles / MA_MIN_SPLIT_TILES ? n : tiles / MA_MIN_SPLIT_TILES;
    if (n > 1) { f.n_whole = 0; f.n_split = n > MA_MAX_SPLIT ? MA_MAX_SPLIT : (int)n; }
    return f;
  }
  if (!alike || items > MA_TAIL_ROUNDS * 2 * MA_CUS || tiles < MA_TAIL_TILES) return f;
  double best = 0.;
  for (int slots = 2 * MA_CUS; slots <= most; slots += MA_CUS) {
    const int64_t tail = items % slots;
    for (int n = 1; n <= 8 && (n == 1 || tiles / n >= MA_TAIL_TILES / 4); ++n) {
      const double last = (double)((tail * n + slots - 1) / slots) / n + (n > 1 ? 0.03 * n : 0.), time = slots * (items / slots + last);
      if (best != 0. && time >= best) continue;
      best = time;
      f.n_split = n;
      f.n_whole = (int)(n > 1 ? items - tail : items);
    }
  }
  return f;
}

int64_t masked_attn_part_floats(int B, int Sq, int H, int Hk, int D, MaskedPlan f) {
  const int64_t rows = (int64_t)Sq * (H / Hk), items = (int64_t)B * Hk * ((rows + MA_ROWS - 1) / MA_ROWS);
  return (items - f.n_whole) * f.n_split * MA_ROWS * (D + 2);
}

bool masked_attn_bias_fits(int H, int Hk, int D, int radius) {
  return (int64_t)(H / Hk) * (2 * (int64_t)radius + 1 + 2 * MA_BIAS_MARGIN) * 4 <= MA_LDS_MAX - ma_fixed_lds(D);
}

namespace {

template <int D, bool kCap, bool kBias>
hipError_t run_masked(const MaskedAttnParams& p, hipStream_t stream) {
  static std::atomic<unsigned> lds_set{0u};
  const int G = p.H / p.Hk;
  const int lds = ma_fixed_lds(D) + (kBias ? G * (2 * p.radius + 1 + 2 * MA_BIAS_MARGIN) * 4 : 0);
  const hipError_t a = ensure_lds_limit(reinterpret_cast<const void*>(icsa_masked_attn_kernel<D, kCap, kBias>), MA_LDS_MAX, &lds_set);
  if (a != hipSuccess) return a;
  const int64_t items = (int64_t)p.B * p.Hk * (((int64_t)p.Sq * G + MA_ROWS - 1) / MA_ROWS), cut = items - p.n_whole;
  if (items > 0x3fffffffLL || cut * p.n_split > 0x3fffffffLL) return hipErrorInvalidValue;
  const int grid = xcd_grid(p.n_whole) + xcd_grid((int)(cut * p.n_split));
  hipLaunchKernelGGL((icsa_masked_attn_kernel<D, kCap, kBias>), dim3(grid), dim3(MA_THREADS), lds, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || cut == 0) return e;
  if (p.n_split >= MA_FEW_PARTS)
    hipLaunchKernelGGL((icsa_masked_combine_kernel<D, true>), dim3((unsigned)(cut * MA_ROWS)), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL((icsa_masked_combine_kernel<D, false>), dim3((unsigned)(cut * (MA_ROWS * D / 1024))), dim3(256), 0, stream, p);
  return hipGetLastError();
}

template <int D>
hipError_t pick_masked(const MaskedAttnParams& p, hipStream_t stream) {
  const bool cap = p.softcap > 0.f, bias = p.bias != nullptr;
  if (cap) return bias ? run_masked<D, true, true>(p, stream) : run_masked<D, true, false>(p, stream);
  return bias ? run_masked<D, false, true>(p, stream) : run_masked<D, false, false>(p, stream);
}

}  // namespace

hipError_t launch_masked_attn(MaskedAttnParams p, hipStream_t stream) {
  const int G = p.H / p.Hk;
  p.by_g = fast_div(G);
  p.by_blk = fast_div((unsigned)(((int64_t)p.Sq * G + MA_ROWS - 1) / MA_ROWS));
  p.by_hk = fast_div(p.Hk);
  p.by_bh = fast_div(p.B * p.Hk);
  p.by_split = fast_div(p.n_split);
  return p.D == 128 ? pick_masked<128>(p, stream) : pick_masked<64>(p, stream);
}
