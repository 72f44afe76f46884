"""Attention under masks at the ends of what its arguments may hold."""
import pytest
import torch

from icsa_hip import masked_attn_func

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("D", [64, 128])
def test_biases_past_the_exponentials_range(gpu, D, softcap):
    """Finite biases from -2.36e38 (the float32 range over log2 e) down count as one: such keys weigh alike where a row sees no others, and nothing beside
    others.  Tolerance: P and the result are rounded to bf16 (2^-8 each, of the mean |v| and of the value), f32 sums."""
    g = torch.Generator().manual_seed(D)
    q, k, v = (torch.randn(1, n, 1, D, generator=g).to(BF) for n in (1, 90, 90))
    low = torch.full((1, 201), -2.5e38)
    low[0, ::3] = -3.3e38
    run = lambda bias: masked_attn_func(q.to(gpu), k.to(gpu), v.to(gpu), bias=bias.to(gpu), softcap=softcap).double().cpu()
    mean, size = v.double().mean(1, keepdim=True), v.double().abs().mean(1, keepdim=True)
    assert ((run(low) - mean).abs() <= 2.0 ** -8 * 1.01 * size + 2.0 ** -8 * mean.abs()).all()
    low[0, 100] = 0.0                                        # the last key, on which the query stands
    assert torch.equal(run(low), v[:, -1:].double())
