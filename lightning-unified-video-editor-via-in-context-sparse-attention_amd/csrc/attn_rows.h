// Rows of attention under document borders: what a row sees, its address, its way to the output.  Shared by the
// forward (masked_attn.hip) and the backward (attn_bwd.hip).
#pragma once

#include "attn_tile.h"
#include "icsa_kernels.h"

namespace {

// What a row sees: keys [lo, hi); at: the key position its own query is aligned with.
struct RowRange { int lo, hi, at; };

template <class P>
__device__ __forceinline__ RowRange doc_range(const P& p, int i, int q1, int k0, int k1, int prefix) {
  RowRange r = {0, 0, 0};
  k0 = min(max(k0, 0), p.Sk);
  k1 = min(max(k1, 0), p.Sk);
  const int64_t at = (int64_t)i + k1 - min(q1, p.Sq);
  r.at = (int)max((int64_t)-0x40000000, min((int64_t)0x40000000, at));
  int64_t end = k1;
  if (p.causal) end = min(end, max(at + 1, (int64_t)k0 + prefix));
  if (end > k0) { r.lo = k0; r.hi = (int)end; }
  return r;
}

// Of query i (this lane's).  P has Sq, Sk, q_starts, k_starts, docs, causal and prefix.  Up to 63 documents: the lanes hold
// their borders, requested together, and a document is found by counting; more: a search in memory.  Called by whole waves.
template <class P>
__device__ __forceinline__ RowRange row_range(const P& p, int b, int i) {
  const int lane = threadIdx.x & 63, docs = p.docs;
  const int* pre = p.prefix != nullptr ? p.prefix + (int64_t)b * docs : nullptr;
  if (p.q_starts == nullptr) return doc_range(p, i, p.Sq, 0, p.Sk, pre ? pre[0] : 0);
  const int* qs = p.q_starts + (int64_t)b * (docs + 1);
  const int* ks = p.k_starts + (int64_t)b * (docs + 1);
  int n, q1, k0, k1, px = 0;
  if (docs < 64) {
    const int own_q = lane <= docs ? qs[lane] : 0x7fffffff, own_k = lane <= docs ? ks[lane] : 0;
    const int own_p = pre != nullptr && lane < docs ? pre[lane] : 0;
    n = -1;                                           // the count of starts <= i, less one
    for (int x = 0; x <= docs; ++x) n += __builtin_amdgcn_readlane(own_q, x) <= i;
    const int c = min(max(n, 0), docs - 1);
    q1 = __shfl(own_q, c + 1, 64);
    k0 = __shfl(own_k, c, 64);
    k1 = __shfl(own_k, c + 1, 64);
    px = __shfl(own_p, c, 64);
  } else {
    int lo = 0, hi = docs + 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (qs[mid] <= i) lo = mid + 1; else hi = mid;
    }
    n = lo - 1;
    const int c = min(max(n, 0), docs - 1);
    q1 = qs[c + 1];
    k0 = ks[c];
    k1 = ks[c + 1];
    if (pre != nullptr) px = pre[c];
  }
  if (n < 0 || n >= docs) return RowRange{0, 0, 0};   // in front of the first document, or behind the last
  return doc_range(p, i, q1, k0, k1, px);
}

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x = min(x, __shfl_xor(x, o, 64));
  return x;
}
__device__ __forceinline__ int wave_max(int x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x = max(x, __shfl_xor(x, o, 64));
  return x;
}

// a where the mask's bits are set, b elsewhere (the compiler makes a comparison and a select of the C form, three
// instructions with the mask's instead of two)
__device__ __forceinline__ unsigned bit_select(unsigned mask, unsigned a, unsigned b) {
  unsigned r;
  asm("v_bfi_b32 %0, %1, %2, %3" : "=v"(r) : "v"(mask), "v"(a), "v"(b));
  return r;
}

// The sign bits of those of two bf16 that are infinite or NaN: a full exponent carries into them
__device__ __forceinline__ unsigned not_finite2(unsigned x) { return ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u; }

// One wave's 32 rows of 32 dims to the output: through 2 KB of the wave's LDS, so that bf16
// stores are 64-byte segments.  v: this lane's 16 values (dims 8 (e / 4) + 4 hl + e % 4 of row li).
template <int kB16>
__device__ __forceinline__ void store_dims32(unsigned char* stage, const float v[16], int rows_valid, int64_t row_off[2],
                                             int64_t own_off, void* out, int d0) {
  const int lane = threadIdx.x & 63, li = lane & 31, hl = lane >> 5;
  if constexpr (kB16) {
    const int wx = (li >> 2) & 3;
#pragma unroll
    for (int pr = 0; pr < 2; ++pr) {
      bf16x4 lo, hi;
#pragma unroll
      for (int e = 0; e < 4; ++e) { lo[e] = (bf16)v[8 * pr + e]; hi[e] = (bf16)v[8 * pr + 4 + e]; }
      const u32x2 x = __builtin_bit_cast(u32x2, lo), y = __builtin_bit_cast(u32x2, hi);
      const auto w0 = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false);
      const auto w1 = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
      *reinterpret_cast<u32x4*>(stage + li * 64 + (((2 * pr + hl) ^ wx) << 4)) = u32x4{w0[0], w1[0], w0[1], w1[1]};
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 16 * i + (lane >> 2);
      const u32x4 x = *reinterpret_cast<const u32x4*>(stage + r * 64 + (((lane & 3) ^ ((r >> 2) & 3)) << 4));
      if (r < rows_valid) *reinterpret_cast<u32x4*>(reinterpret_cast<bf16*>(out) + row_off[i] + d0 + 8 * (lane & 3)) = x;
    }
  } else if (li < rows_valid) {
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<floatx4*>(reinterpret_cast<float*>(out) + own_off + d0 + 8 * g + 4 * hl) =
          floatx4{v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3]};
  }
}

// What the backward takes of a row: log2 of its sum of 2^score; +inf, with which every weight is 0, where it has none
__device__ __forceinline__ float row_lse(float m, float l) { return l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l); }

// What rounding o to bf16 (b) leaves, in a byte: (o - b) in 1/256 of b's last place, + 128.  The backward's D = rowsum(dO * O) takes O
// from both: from the rounded O alone D's error, a row's common shift of dP, is as large as dS's own rounding where a row's weight
// lies on few keys (77 keys: dq 0.0026 from the exact one in the 2-norm, 0.0024 with the byte, 0.0017 is the results' rounding alone; 8 keys:
// 0.0029 and 0.0025; 3 keys: 0.0036 and 0.0025).
// A row's bytes lie in the order in which the backward's lanes read them: rest_at of a dim.
__device__ __forceinline__ unsigned rest_bytes(const float o[4]) {
  unsigned w = 0u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float f = (float)(bf16)o[e];
    // 2^15 over f's power of two; what this is not for (values under 2^-112, infinities) has a byte that moves nothing
    const float up = __uint_as_float(0x86800000u - (__float_as_uint(f) & 0x7f800000u));
    w = __builtin_amdgcn_cvt_pk_u8_f32(fmaf(o[e] - f, up, 128.f), e, w);  // to a whole number, 0 to 255
  }
  return w;
}
// and back: byte e of w beside b
__device__ __forceinline__ float with_rest(bf16 b, unsigned w, int e) {
  const float f = (float)b, power = __uint_as_float(__float_as_uint(f) & 0x7f800000u), t = (float)((w >> (8 * e)) & 255u);
  return fmaf(fmaf(t, 0x1p-15f, -0x1p-8f), power, f);
}
template <int D> __device__ __forceinline__ int rest_at(int dim) {
  return ((dim >> 3) & 1) * (D / 2) + ((dim >> 4) & 1) * (D / 4) + (dim >> 5) * 8 + (dim & 7);
}

// element offset of row r (query r / G, head hk G + r % G) in a [B, S, H, D] tensor
__device__ __forceinline__ int64_t row_at(int64_t sb, int64_t ss, int64_t sh, int b, int hk, const FastDiv& g, int r) {
  const unsigned i = g.d == 1 ? r : g.div(r);
  return (int64_t)b * sb + (int64_t)i * ss + (int64_t)(hk * g.d + r - i * g.d) * sh;
}

// rest: [B, S, H, D] bytes like a contiguous output, or null
template <int D>
__device__ __forceinline__ void store_wave(const OutView& out, const FastDiv& by_g, unsigned char* stage, const floatx16 o[D / 32],
                                           float inv_l, int b, int hk, int r0, int rows_valid,
                                           unsigned char* rest = nullptr, int Sq = 0, int H = 0) {
  const int lane = threadIdx.x & 63, li = lane & 31;
  int64_t off[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) off[i] = row_at(out.sb, out.ss, out.sh, b, hk, by_g, r0 + 16 * i + (lane >> 2));
  const int64_t own = row_at(out.sb, out.ss, out.sh, b, hk, by_g, r0 + li);
#pragma unroll
  for (int ds = 0; ds < D / 32; ++ds) {
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = o[ds][e] * inv_l;
    if (out.dtype == ICSA_DT_BF16) store_dims32<1>(stage, v, rows_valid, off, own, out.p, 32 * ds);
    else store_dims32<0>(stage, v, rows_valid, off, own, out.p, 32 * ds);
  }
  if (rest == nullptr) return;
  // dims 32 ds + 16 hl .. + 15 of row li in a lane: eight bytes for either half of the backward's lanes
  const int hl = lane >> 5;
  u32x2 first[D / 32], second[D / 32];
#pragma unroll
  for (int ds = 0; ds < D / 32; ++ds) {
    unsigned w[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float v[4] = {o[ds][4 * g] * inv_l, o[ds][4 * g + 1] * inv_l, o[ds][4 * g + 2] * inv_l, o[ds][4 * g + 3] * inv_l};
      w[g] = rest_bytes(v);
    }
    const auto x = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    const auto y = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    first[ds] = u32x2{x[0], x[1]};
    second[ds] = u32x2{y[0], y[1]};
  }
  if (li >= rows_valid) return;
  unsigned char* dst = rest + row_at((int64_t)Sq * H * D, (int64_t)H * D, D, b, hk, by_g, r0 + li) + hl * (D / 4);
#pragma unroll
  for (int ds = 0; ds < D / 32; ds += 2) {
    *reinterpret_cast<u32x4*>(dst + 8 * ds) = u32x4{first[ds][0], first[ds][1], first[ds + 1][0], first[ds + 1][1]};
    *reinterpret_cast<u32x4*>(dst + D / 2 + 8 * ds) = u32x4{second[ds][0], second[ds][1], second[ds + 1][0], second[ds + 1][1]};
  }
}

}  // namespace
