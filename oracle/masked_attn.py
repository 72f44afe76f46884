"""Attention under masks on the CPU in float64, from its definition, and a bound on a bf16
kernel's distance from it."""
import math

import torch


def visible(B, Sq, Sk, q_starts=None, k_starts=None, causal=False, prefix=None):
    """([B, Sq, Sk] truth values, [B, Sq] aligned key positions), row by row."""
    see = torch.zeros(B, Sq, Sk, dtype=torch.bool)
    at = torch.zeros(B, Sq, dtype=torch.long)
    for b in range(B):
        qs = [0, Sq] if q_starts is None else q_starts[b].tolist()
        ks = [0, Sk] if k_starts is None else k_starts[b].tolist()
        for n in range(len(qs) - 1):
            pre = 0 if prefix is None else int(prefix.reshape(B, -1)[b, n])
            for i in range(max(qs[n], 0), min(qs[n + 1], Sq)):
                at[b, i] = i + ks[n + 1] - qs[n + 1]
                hi = ks[n + 1]
                if causal:
                    hi = min(hi, max(int(at[b, i]) + 1, ks[n] + pre))
                see[b, i, max(ks[n], 0):max(hi, 0)] = True
    return see, at


def attention(q, k, v, *, q_starts=None, k_starts=None, causal=False, prefix=None, softcap=0.0, bias=None, scale=None):
    """(out, bound) float64 [B, Sq, H, D].  Values of keys that no query sees play no part, and a
    value that is not finite reaches the queries that see it.

    bound, for f32 scores, P rounded to bf16 and f32 sums: a score is off by at most
    2^-23 (D scale sum |q k| + 8 (|s| + cap + |bias|) + 8) = e (its additions, the roundings of its
    products, tanh and the exponential, each a few steps), so a probability by a factor exp(+-2 e)
    (its own and the total's), which moves the output o by 2.5 e sum p |v| at most.  Rounded weights
    p (1 + d), |d| <= 2^-8, stand in the product and in the total that divides it:
    sum p (1 + d) v / sum p (1 + d) - o = sum p d (v - o) / (1 + sum p d), at most
    2^-8 / (1 - 2^-8) sum p |v - o| <= 1.004 2^-8 (sum p |v| + |o|).  (Two keys, p = 0.9 at v = 0 and 0.1 at
    v = 1, rounded in opposite directions: 0.18 2^-8, past 2^-8 sum p |v|.)"""
    q, k, v = q.double(), k.double(), v.double()
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1:3]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    see, at = visible(B, Sq, Sk, q_starts, k_starts, causal, prefix)
    out = torch.zeros(B, Sq, H, D, dtype=torch.float64)
    bound = torch.zeros_like(out)
    if Sk == 0:
        return out, bound
    dist = torch.arange(Sk)[None, None] - at[:, :, None]
    for b in range(B):
        for h in range(H):
            s = scale * q[b, :, h] @ k[b, :, h // G].t()
            mass = scale * q[b, :, h].abs() @ k[b, :, h // G].abs().t()
            size = s.abs()
            if softcap:
                s = softcap * torch.tanh(s / softcap)
                size = size.clamp(max=8 * softcap) + softcap
            if bias is not None:
                R = bias.shape[1] // 2
                x = bias[h].double()[dist[b].clamp(-R, R) + R]
                s = s + x
                size = size + torch.where(torch.isfinite(x) & (x.abs() < 1e30), x.abs(), torch.zeros_like(x))
            s = torch.where(see[b], s, torch.full_like(s, -math.inf))
            none = ~(s > -math.inf).any(-1) & ~torch.isnan(s).any(-1)
            m = torch.where(none, 0.0, s.amax(-1))
            p = torch.exp(s - m[:, None])
            p = p / torch.where(none, 1.0, p.sum(-1))[:, None]
            vv = v[b, :, h // G]
            fine = torch.isfinite(vv)
            o = p @ torch.where(fine, vv, 0.0)
            if not fine.all():
                for j in (~fine).any(1).nonzero().flatten().tolist():
                    rows = see[b, :, j]
                    o[rows] += torch.where(fine[j], 0.0, p[rows, j, None] * vv[j])
            out[b, :, h] = torch.where(none[:, None], 0.0, o)
            e = 2.0 ** -23 * (D * torch.where(see[b], mass, 0.0).amax(-1) + 8 * torch.where(see[b], size, 0.0).amax(-1) + 8)
            size = p @ torch.where(fine, vv.abs(), 0.0)
            own = torch.where(none[:, None], 0.0, p @ torch.where(fine, vv, 0.0)).abs()
            bound[b, :, h] = 1.004 * 2.0 ** -8 * (size + own) + 2.5 * e[:, None] * size + 1e-30
    return out, bound


def one_head(q, k, v, lo, hi, at, *, scale, softcap=0.0, bias=None):
    """(out, bound) float64 of one head, on its inputs' device: q [R, D], k, v [Sk, D], row i sees the keys [lo_i, hi_i) and
    stands at key at_i (all [R]); bias [2 R + 1].  The bound is :func:`attention`'s.  Values have to be finite."""
    q, k, v = q.double(), k.double(), v.double()
    kt = k.t().contiguous()
    s = scale * (q @ kt)
    mass = scale * (q.abs() @ kt.abs())
    size = s.abs()
    if softcap:
        s = softcap * torch.tanh(s / softcap)
        size = size.clamp(max=8 * softcap) + softcap
    j = torch.arange(k.shape[0], device=q.device)[None]
    if bias is not None:
        R = bias.shape[0] // 2
        x = bias.double()[(j - at[:, None]).clamp(-R, R) + R]
        s = s + x
        size = size + x.abs()
    see = (j >= lo[:, None]) & (j < hi[:, None])
    none = ~see.any(-1)
    s = s.masked_fill(~see, -math.inf)
    p = torch.exp(s - torch.where(none, 0.0, s.amax(-1))[:, None])
    p = p / torch.where(none, 1.0, p.sum(-1))[:, None]
    e = 2.0 ** -23 * (q.shape[1] * torch.where(see, mass, 0.0).amax(-1) + 8 * torch.where(see, size, 0.0).amax(-1) + 8)
    out, size = p @ v, p @ v.abs()
    return out, 1.004 * 2.0 ** -8 * (size + out.abs()) + 2.5 * e[:, None] * size + 1e-30
