"""CPU checks behind test_gpu_masked_parts.py: its sizes are dealt out as they say, its reference is the oracle's, and its
tolerance sees a lost or wrongly weighted part."""
import pytest
import torch

from icsa_hip import _lib
from oracle import masked_attn as O
from test_gpu_masked_parts import MIXED, first_cut_head

pytestmark = pytest.mark.cpu
BF = torch.bfloat16


@pytest.mark.parametrize("B,Sq,Sk,H,Hk,D,n_whole,n_split", MIXED)
def test_sizes_of_the_gpu_tests_are_mixed(B, Sq, Sk, H, Hk, D, n_whole, n_split):
    """The workspace holds 128 (D + 2) f32 for each part of an item that is not whole."""
    items = B * Hk * -(-Sq * (H // Hk) // 128)
    assert 0 < n_whole < items and n_split > 1
    size = (items - n_whole) * n_split * 128 * (D + 2) * 4
    assert _lib.lib().icsa_masked_attn_workspace_size(B, Sq, Sk, H, Hk, D, 1, 0) == -(-size // 256) * 256
    b, h = first_cut_head(B, Sq, H, Hk, n_whole)
    assert 0 <= b < B and 0 <= h < H


@pytest.mark.parametrize("causal", [False, True])
def test_one_head_is_the_oracle(causal):
    q, k, v = (torch.randn(1, n, h, 64).to(BF) for n, h in ((50, 2), (70, 1), (70, 1)))
    qs, ks, bias = torch.tensor([[3, 45]]), torch.tensor([[5, 66]]), torch.randn(2, 9)
    ref, bound = O.attention(q, k, v, q_starts=qs, k_starts=ks, causal=causal, softcap=3.0, bias=bias)
    see, _ = O.visible(1, 50, 70, qs, ks, causal)
    lo = torch.where(see[0].any(1), see[0].int().argmax(1), 0)
    hi = lo + see[0].sum(1)
    for h in range(2):
        out, b = O.one_head(q[0, :, h], k[0, :, 0], v[0, :, 0], lo, hi, torch.arange(50) + 66 - 45, scale=64 ** -0.5,
                            softcap=3.0, bias=bias[h])
        assert torch.allclose(out, ref[0, :, h], rtol=1e-12, atol=1e-12)
        assert torch.allclose(b[lo < hi], bound[0, :, h][lo < hi], rtol=1e-9, atol=0)


@pytest.mark.parametrize("D,Sk,n", [(64, 9373, 3), (64, 2100, 2), (128, 8300, 6), (128, 2111, 4)])
@pytest.mark.parametrize("mistake", ["lost", "weight"])
def test_tolerance_sees_a_wrong_part(D, Sk, n, mistake):
    """One of the n parts left out, or with half its weight: past the tolerance in every row."""
    g = torch.Generator().manual_seed(Sk)
    q, k, v = ((s * torch.randn(m, D, generator=g)).to(BF) for m, s in ((40, 1.5), (Sk, 1.0), (Sk, 1.0)))
    whole = [torch.full((40,), x) for x in (0, Sk, 0)]
    ref, bound = O.one_head(q, k, v, *whole, scale=D ** -0.5)
    tol = bound + 2.0 ** -8 * ref.abs()
    p = torch.exp(D ** -0.5 * q.double() @ k.double().t())
    assert ((p @ v.double() / p.sum(1, keepdim=True) - ref).abs() <= tol).all()
    for part in range(n):
        wrong = p.clone()
        wrong[:, Sk * part // n:Sk * (part + 1) // n] *= 0.0 if mistake == "lost" else 0.5
        d = (wrong @ v.double() / wrong.sum(1, keepdim=True) - ref).abs()
        assert (d > tol).any(1).all()


def test_bound_counts_the_rounding_of_the_total():
    """Two weights, near 0.9 and 0.1, rounded to bf16 in opposite directions, in the product and in the total: the result is past
    2^-8 sum p |v| and within the bound."""
    d = 2.0 ** -8 * 0.99
    p = torch.tensor([[0.9, 0.1]], dtype=torch.float64)
    q, k, v = torch.ones(1, 64).double(), torch.log(p).t() / 8 * torch.ones(2, 64), torch.tensor([[0.0], [1.0]]).double().expand(2, 64)
    one = torch.ones(1, dtype=torch.long)
    ref, bound = O.one_head(q, k, v, 0 * one, 2 * one, one, scale=64 ** -0.5)
    assert torch.allclose(ref, torch.full_like(ref, 0.1), atol=1e-12)
    w = p * torch.tensor([[1 - d, 1 + d]])
    off = (w @ v / w.sum() - ref).abs()
    assert (off > 2.0 ** -8 * (p @ v.abs())).all() and (off <= bound).all()
