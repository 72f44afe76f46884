"""Attention over documents and its gradients on the CPU in float64, from their definition, with a bound on a
bf16 kernel's distance from each."""
import math

import torch

U = 2.0 ** -24               # half a step of float32
W = 2.0 ** -8                # of bfloat16


def documents(B, Sq, Sk, q_starts=None, k_starts=None):
    """(batch row, first and last query, first and last key) of every document, clamped to the lengths."""
    for b in range(B):
        qs = [0, Sq] if q_starts is None else q_starts[b].tolist()
        ks = [0, Sk] if k_starts is None else k_starts[b].tolist()
        for n in range(len(qs) - 1):
            i0, i1, j0, j1 = (min(max(x, 0), top) for x, top in ((qs[n], Sq), (qs[n + 1], Sq), (ks[n], Sk), (ks[n + 1], Sk)))
            if i1 > i0 and j1 > j0:
                yield b, i0, i1, j0, j1


def cross_attention(q, k, v, dout, *, q_starts=None, k_starts=None, scale=None, rest=True):
    """({name: value}, {name: bound}) for out, dq, dk, dv, float64.

    Bounds, element by element, for f32 scores and sums, P and dS rounded to bf16 (W each), and a total of rounded weights.  A score is off by e <= 2 U (D sum |q k| scale + 8 |s| + 8), so
    exp(score) by a factor 1 + 2 e; the total by W more, so a weight of the backward by f = 4 e + 1.01 W of itself, and its
    rounded form by f + W.
      out   1.01 (2.5 e sum p |v| + W sum p |v - o|), as in masked attention; D reads it with a byte of what its rounding left, in
            256ths of the last place (2^-7 of a value at most), clamped by one: 2^-15 |o|; without that byte (rest) rounded: W |o|
      D     sum |dout| (o's) + 2 U D sum |dout o|
      dP    2 U D sum |dout v|
      dS    p (f |dP - D| + (1 + f) (dP's + D's)), and W of |dS| + that
      dq    scale sum_j (dS's |k_j| + n U |dS k_j|) for a sum of n terms; dk alike over queries and heads
      dv    sum_i ((f + W) p |dout_i| + n U |p dout_i|)"""
    q, k, v, dout = (t.double() for t in (q, k, v, dout))
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1:3]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    val = {n: torch.zeros_like(t) for n, t in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    tol = {n: torch.zeros_like(t) for n, t in val.items()}
    for b, i0, i1, j0, j1 in documents(B, Sq, Sk, q_starts, k_starts):
        for h in range(H):
            g = h // G
            Q, K, V, dO = q[b, i0:i1, h], k[b, j0:j1, g], v[b, j0:j1, g], dout[b, i0:i1, h]
            s = scale * Q @ K.t()
            p = torch.softmax(s, 1)
            o = p @ V
            dP = dO @ V.t()
            Dr = (dO * o).sum(1, keepdim=True)
            dS = p * (dP - Dr)
            val["out"][b, i0:i1, h] = o
            val["dq"][b, i0:i1, h] = scale * dS @ K
            val["dk"][b, j0:j1, g] += scale * dS.t() @ Q
            val["dv"][b, j0:j1, g] += p.t() @ dO

            e = 2 * U * (D * scale * Q.abs() @ K.abs().t() + 8 * s.abs() + 8)
            em = e.amax(1, keepdim=True)
            f = 4 * em + 1.01 * W
            to = 1.01 * (2.5 * em * (p @ V.abs()) + W * (p @ V.abs() + o.abs()))
            tD = (dO.abs() * (to + (2.0 ** -15 if rest else W) * (o.abs() + to))).sum(1, keepdim=True) + 2 * U * D * (dO * o).abs().sum(1, keepdim=True)
            tP = 2 * U * D * dO.abs() @ V.abs().t()
            tS = p * (f * (dP - Dr).abs() + (1 + f) * (tP + tD))
            tS = tS + W * (dS.abs() + tS)
            n_k, n_q = j1 - j0 + 64, (i1 - i0) * G + 64
            tol["out"][b, i0:i1, h] = to
            tol["dq"][b, i0:i1, h] = scale * (tS @ K.abs() + n_k * U * (dS.abs() + tS) @ K.abs())
            tol["dk"][b, j0:j1, g] += scale * (tS.t() @ Q.abs() + n_q * U * (dS.abs() + tS).t() @ Q.abs())
            tol["dv"][b, j0:j1, g] += ((f + W + n_q * U) * 1.01 * p).t() @ dO.abs()
    return val, tol
