"""Rows of the attention under masks: strides of dimensions of length one do not count, whatever torch holds there."""
import pytest
import torch

from icsa_hip import masked_attn_func
from icsa_hip.hip_host import _rows16

BF = torch.bfloat16


def _aligned(t):
    return all(s % 8 == 0 for s, n in zip(t.stride()[:3], t.shape) if n > 1) and t.stride(3) == 1 and t.data_ptr() % 16 == 0


def _views(device="cpu"):
    """[B, S, H, 64] views with odd strides in dimensions of length one and, some of them, in others too."""
    g = torch.Generator().manual_seed(0)
    base = torch.randn(2, 5, 3, 65, generator=g).to(BF).to(device)
    one = torch.randn(2, 5, 1, 65, generator=g).to(BF).to(device)
    return {"one token, one head": one[0:1, 0:1, :, :64], "one token": base[:, 0:1, :, :64], "one head": base[:, :, 1:2, :64],
            "odd everywhere": base[..., :64], "odd start": one[0:1, 1:2, :, 1:], "odd batch": torch.empty(
                2 * 64 + 3, dtype=BF, device=device).copy_(base.flatten()[:131]).as_strided((1, 2, 1, 64), (131, 64, 7, 1))}


@pytest.mark.cpu
@pytest.mark.parametrize("name", list(_views()))
def test_rows16_gives_strides_that_the_library_takes(name):
    t = _views()[name]
    r, (p, *strides) = _rows16(t)
    assert torch.equal(r, t) and p == r.data_ptr() and p % 16 == 0
    assert all(s % 8 == 0 for s in strides), strides
    assert all(s == u for s, u, n in zip(strides, r.stride(), r.shape) if n > 1)
    if _aligned(t):
        assert r is t                                        # rows that are in place are not copied


@pytest.mark.cpu
def test_aligned_rows_are_taken_as_they_are():
    t = torch.zeros(2, 5, 3, 128, dtype=BF)[..., :64]
    r, a = _rows16(t)
    assert r is t and a == (t.data_ptr(), *t.stride()[:3])


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(_views()))
def test_attention_of_such_views(gpu, name):
    t = _views(gpu)[name]
    ref = masked_attn_func(*(t.clone(memory_format=torch.contiguous_format) for _ in range(3)), causal=True)
    assert torch.equal(masked_attn_func(t, t, t, causal=True), ref)
