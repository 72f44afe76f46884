"""Microscaled 4-bit floating point on the CPU, from its definition: blocks of 32 e2m1 values
with a power of two, quantisation to it, and products of such rows in float64."""
import math

import torch

E2M1 = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
GROUP, BLOCK = 256, 32


def padded(k: int) -> int:
    return -(-k // GROUP) * GROUP


def quantize(x: torch.Tensor):
    """(codes uint8 [M, Kp/2], scales uint8 [Kp/256, M, 8]) of x [M, K]: scale 2^(floor(log2
    max|x|) - 2) with the byte kept at 0 or more, nearest table entry (ties: the even code), 255
    and zero codes for a block with a NaN or an infinity."""
    M, K = x.shape
    Kp = padded(K)
    b = torch.zeros(M, Kp, dtype=torch.float64)
    b[:, :K] = x.double()
    b = b.view(M, Kp // BLOCK, BLOCK)
    bad = ~torch.isfinite(b).all(-1)
    b = torch.where(bad[..., None], torch.zeros_like(b), b)
    amax = b.abs().amax(-1)
    e = torch.frexp(amax).exponent.long() - 1 - 2
    byte = torch.where(amax > 0, (e + 127).clamp(min=0), torch.zeros_like(e))
    a = b.abs() / torch.exp2(byte.double() - 127)[..., None]
    d = (a[..., None] - E2M1).abs()
    best = d.amin(-1, keepdim=True)
    near = d == best                                       # two entries at a tie: take the even code
    code = torch.arange(8).expand_as(near)
    pick = torch.where(near, torch.where(near.sum(-1, keepdim=True) > 1, code % 2, torch.zeros_like(code)) * 100 + code,
                       torch.full_like(code, 1000)).amin(-1) % 100
    code = (pick | (torch.signbit(b).long() << 3)).to(torch.uint8).view(M, Kp)
    byte = torch.where(bad, torch.full_like(byte, 255), byte).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte.view(M, Kp // GROUP, 8).permute(1, 0, 2).contiguous()


def values(codes: torch.Tensor, scales: torch.Tensor, K: int) -> torch.Tensor:
    """float64 [M, K] of codes and scales (any device; computed on the CPU)."""
    codes, scales = codes.cpu().long(), scales.cpu()
    M = codes.shape[0]
    c = torch.stack([codes & 15, codes >> 4], -1).view(M, -1)
    v = torch.where(c >= 8, -1.0, 1.0).double() * E2M1[c & 7]
    s = scales.permute(1, 0, 2).reshape(M, -1).double()
    s = torch.where(s == 255, torch.full_like(s, math.nan), torch.exp2(s - 127))
    return (v * s.repeat_interleave(BLOCK, 1))[:, :K]


def gelu_tanh(t: torch.Tensor) -> torch.Tensor:
    return 0.5 * t * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3)))
