"""Layer norm, RMS norm and rotary positions with their gradients on the CPU in float64, from their definitions, with
a bound on a float32 kernel's distance from each (before its result's own rounding)."""
import torch

U = 2.0 ** -24               # half a step of float32


def norm(x, dy, gain=None, shift=None, *, rms=False, eps=1e-6):
    """({name: value}, {name: bound}) of y, dx, da, db for x, dy [G, rows, dim], gain and shift [G, dim] (gain: the whole
    factor, 1 + scale where it is one).  float64.

    Bounds: a sum over a row adds at most 32 values in a lane and 12 more in the lanes' tree, so it is off by 48 U of its absolute
    terms' sum, and one over n rows by n U.  mean: 48 U mean|x|, which moves the variance by its square alone; the centred values'
    rounding and the sum: 52 U; rstd: 30 U.  xh: rstd (mean's + 33 U |x - mean|).  y: |a| xh's + 3 U (|a xh| + |b|).
    dx: rstd (4 U (|u| + |m0| + |xh m1|) + 50 U mean|u| + |xh| m1's + |m1| xh's) + 31 U |dx|, m1's = mean(|u| xh's) + 52 U mean|u xh|."""
    x, dy = x.double(), dy.double()
    G, rows, dim = x.shape
    a = torch.ones(G, 1, dim, dtype=torch.float64) if gain is None else gain.double().reshape(G, 1, dim)
    b = torch.zeros(G, 1, dim, dtype=torch.float64) if shift is None else shift.double().reshape(G, 1, dim)
    mean = torch.zeros(G, rows, 1, dtype=torch.float64) if rms else x.mean(-1, keepdim=True)
    v = x - mean
    r = 1 / (v.square().mean(-1, keepdim=True) + eps).sqrt()
    xh = v * r
    u = dy * a
    m1 = (u * xh).mean(-1, keepdim=True)
    m0 = 0 * m1 if rms else u.mean(-1, keepdim=True)
    val = dict(y=xh * a + b, dx=r * (u - m0 - xh * m1), da=(dy * xh).sum(1), db=dy.sum(1))

    t_mean = 0 * mean if rms else 48 * U * x.abs().mean(-1, keepdim=True)
    t_xh = r * (t_mean * (1 + t_mean * r * xh.abs()) + 33 * U * v.abs())
    t_m1 = (u.abs() * t_xh).mean(-1, keepdim=True) + 52 * U * (u * xh).abs().mean(-1, keepdim=True)
    tol = dict(y=a.abs() * t_xh + 3 * U * ((a * xh).abs() + b.abs()),
               dx=r * (4 * U * (u.abs() + m0.abs() + (xh * m1).abs()) + 50 * U * u.abs().mean(-1, keepdim=True)
                       + xh.abs() * t_m1 + m1.abs() * t_xh) + 31 * U * val["dx"].abs(),
               da=(dy.abs() * t_xh).sum(1) + (rows + 2) * U * (dy * xh).abs().sum(1), db=rows * U * dy.abs().sum(1))
    return val, tol


def rotary(x, cos, sin, positions, sections, interleaved=True, backward=False):
    """(value, bound) float64 [B, S, H, D], token by token; positions [B, S, A].  Two products and a sum in float32:
    2 U (|x0 c| + |x1 s|)."""
    B, S, H, D = x.shape
    n = cos.shape[1]
    axis = [a for a, pairs in enumerate(sections) for _ in range(pairs)]
    y, t = x.double().clone(), torch.zeros(B, S, H, D, dtype=torch.float64)
    for j in range(n):
        d0, d1 = (2 * j, 2 * j + 1) if interleaved else (j, j + n)
        pos = positions[..., axis[j]].long()
        ok = (pos >= 0) & (pos < cos.shape[0])
        at = pos.clamp(0, cos.shape[0] - 1)
        c = torch.where(ok, cos.double()[at, j], 1.0)[:, :, None]
        s = torch.where(ok, sin.double()[at, j], 0.0)[:, :, None] * (-1 if backward else 1)
        x0, x1 = x.double()[..., d0], x.double()[..., d1]
        y[..., d0], y[..., d1] = x0 * c - x1 * s, x0 * s + x1 * c
        t[..., d0] = 2 * U * ((x0 * c).abs() + (x1 * s).abs())
        t[..., d1] = 2 * U * ((x0 * s).abs() + (x1 * c).abs())
    return y, t
