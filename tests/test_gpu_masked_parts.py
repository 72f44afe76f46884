"""Attention under masks where whole items come first and the last round's items are cut in parts of
their keys: every row of the first head (whole), of the head in which the parts begin and of the last
one against float64, under the oracle's bound (roundings of P, 2^-8 (sum p |v| + |o|): a lost or
wrongly weighted part is past it in every row, test_mx_masked_plan.py).  That each size is dealt out as it says is checked there too."""
import math

import pytest
import torch

from icsa_hip import masked_attn_func
from oracle import masked_attn as O

pytestmark = pytest.mark.gpu
BF = torch.bfloat16

# B, Sq, Sk, H, Hk, D, whole items, parts of each of the others
MIXED = [
    (1, 9373, 9373, 16, 16, 64, 1024, 3),        # two workgroups a CU
    (1, 6650, 2100, 20, 20, 64, 768, 2),         # three workgroups a CU
    (1, 6600, 2133, 20, 10, 64, 768, 2),         # two heads a key head, the last block not full
    (2, 3300, 2100, 24, 12, 64, 1024, 2),        # the parts begin in the second batch row
    (1, 8300, 8300, 9, 9, 128, 512, 6),
    (1, 6200, 2111, 12, 12, 128, 512, 4),
    (1, 4150, 2100, 18, 9, 128, 512, 4),
]


def first_cut_head(B, Sq, H, Hk, n_whole):
    """Batch row and head of the first item in parts: a head's row blocks are consecutive items."""
    blocks = -(-Sq * (H // Hk) // 128)
    b, hk = divmod(n_whole // blocks, Hk)
    return b, hk * (H // Hk)


def _check(gpu, case, out_dtype, softcap=0.0, radius=None, borders=None, seed=0):
    B, Sq, Sk, H, Hk, D, n_whole, _ = case
    g = torch.Generator(device=gpu).manual_seed(seed)
    q = (1.5 * torch.randn(B, Sq, H, D, generator=g, device=gpu)).to(BF)
    k, v = (torch.randn(B, Sk, Hk, D, generator=g, device=gpu).to(BF) for _ in range(2))
    bias = None if radius is None else torch.randn(H, 2 * radius + 1, generator=g, device=gpu)
    (q0, q1), (k0, k1) = borders or ((0, Sq), (0, Sk))
    starts = {}
    if borders:
        starts = {n: torch.tensor([x] * B, dtype=torch.int32, device=gpu) for n, x in (("q_starts", (q0, q1)), ("k_starts", (k0, k1)))}
    out = masked_attn_func(q, k, v, softcap=softcap, bias=bias, out_dtype=out_dtype, **starts)
    assert out.dtype == out_dtype
    i = torch.arange(Sq, device=gpu)
    inside = (i >= q0) & (i < q1)
    lo, hi, at = torch.full_like(i, k0), torch.where(inside, k1, k0), i + k1 - q1
    for b, h in {(0, 0), first_cut_head(B, Sq, H, Hk, n_whole), (B - 1, H - 1)}:
        hk = h * Hk // H
        ref, bound = O.one_head(q[b, :, h], k[b, :, hk], v[b, :, hk], lo, hi, at, scale=D ** -0.5, softcap=softcap,
                                bias=None if bias is None else bias[h])
        d = (out[b, :, h].double() - ref).abs()
        tol = bound + (2.0 ** -8 if out_dtype == BF else 2.0 ** -22) * ref.abs()
        assert (d <= tol).all(), f"row {b}, head {h}: {(d / tol).max().item():.2f} of the tolerance"
    assert torch.equal(out, masked_attn_func(q, k, v, softcap=softcap, bias=bias, out_dtype=out_dtype, **starts))


@pytest.mark.parametrize("case", range(len(MIXED)))
def test_plain(gpu, case):
    print(f"[masked parts] {MIXED[case]}", flush=True)
    _check(gpu, MIXED[case], BF if case % 2 else torch.float32, seed=case)


@pytest.mark.parametrize("case", [1, 2, 5, 6])
@pytest.mark.parametrize("softcap,radius", [(10.0, None), (0.0, 64), (10.0, 64)])
def test_caps_and_biases(gpu, case, softcap, radius):
    print(f"[masked parts] {MIXED[case]} cap={softcap} R={radius}", flush=True)
    _check(gpu, MIXED[case], torch.float32 if case % 2 else BF, softcap, radius, seed=20 + case)


@pytest.mark.parametrize("case", [1, 5])
def test_one_document_inside(gpu, case):
    """Rows in front of and behind the document see nothing; its keys begin and end inside tiles."""
    _, Sq, Sk = MIXED[case][:3]
    print(f"[masked parts] {MIXED[case]} inside", flush=True)
    _check(gpu, MIXED[case], BF, radius=8, borders=((130, Sq - 77), (67, Sk - 101)), seed=40 + case)


@pytest.mark.parametrize("case", [1, 5])
def test_values_that_are_not_finite(gpu, case):
    """Behind the last key of the document they reach nobody; seen by every query, each of them."""
    B, Sq, Sk, H, Hk, D, _, _ = MIXED[case]
    print(f"[masked parts] {MIXED[case]} not finite", flush=True)
    q, k, v = (torch.randn(B, n, h, D, device=gpu).to(BF) for n, h in ((Sq, H), (Sk, Hk), (Sk, Hk)))
    starts = dict(q_starts=torch.tensor([[0, Sq]] * B, dtype=torch.int32, device=gpu),
                  k_starts=torch.tensor([[0, Sk - 33]] * B, dtype=torch.int32, device=gpu))
    want = masked_attn_func(q, k, v, **starts)
    v[:, Sk - 33:] = math.nan
    k[:, Sk - 30:] = math.inf
    assert torch.equal(masked_attn_func(q, k, v, **starts), want)
    v[0, Sk - 40, 0, 5], v[0, 70, 0, 6] = math.inf, -math.inf
    got = masked_attn_func(q, k, v, **starts)
    group = range(H // Hk)                                   # the heads of key head 0
    for d, x in ((5, math.inf), (6, -math.inf)):
        for h in group:
            assert (got[0, :, h, d] == x).all()
            want[0, :, h, d] = x
    assert torch.equal(got, want)
