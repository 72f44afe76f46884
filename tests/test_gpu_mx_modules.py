"""Types of the 4-bit layers in the modules: results in the input's type also where an input is quantised once for several layers."""
import pytest
import torch
import torch.nn as nn

from icsa_hip import MXLinear, mx_linear, wan
from oracle import wan_glue as W

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


class _Alone(nn.Module):
    """An MXLinear that quantises its own input, whatever stands beside it."""

    def __init__(self, linear):
        super().__init__()
        self.m = MXLinear(linear)

    def forward(self, x, activation=None):
        return self.m(x, activation)


def _replace(module, names, kind):
    for n in names:
        setattr(module, n, kind(getattr(module, n)))
    return module


@torch.no_grad()
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_self_attention_keeps_the_input_type(gpu, dtype):
    """Quantised once for q, k and v, or by each of them: the same projections, in x's type."""
    torch.manual_seed(0)
    a = wan.WanSelfAttention(256, 2).to(gpu).to(dtype)
    b = wan.WanSelfAttention(256, 2).to(gpu).to(dtype)
    b.load_state_dict(a.state_dict())
    grid = [(2, 16, 16)]
    x = torch.randn(1, 1024, 256, device=gpu).to(dtype)
    args = (torch.tensor([1024]), grid, grid, 1, W.wan_freqs(128))
    _replace(a, "qkv", MXLinear)
    _replace(b, "qkv", _Alone)
    seen = []
    for n in "qkv":
        getattr(a, n).register_forward_hook(lambda m, i, y: seen.append(y.dtype))
    y, z = a(x, *args), b(x, *args)
    assert seen == [dtype] * 3
    assert y.dtype == dtype and torch.equal(y, z)


@torch.no_grad()
@pytest.mark.parametrize("dtype", [BF, torch.float32])
@pytest.mark.parametrize("lens", [None, [24]])
def test_cross_attention_keeps_the_input_type(gpu, dtype, lens):
    torch.manual_seed(1)
    a = wan.WanT2VCrossAttention(256, 2).to(gpu).to(dtype)
    b = wan.WanT2VCrossAttention(256, 2).to(gpu).to(dtype)
    b.load_state_dict(a.state_dict())
    _replace(a, "kv", MXLinear)
    _replace(b, "kv", _Alone)
    x, ctx = (torch.randn(1, n, 256, device=gpu).to(dtype) for n in (70, 40))
    assert torch.equal(a(x, ctx, lens), b(x, ctx, lens))


@torch.no_grad()
@pytest.mark.parametrize("dtype", [BF, torch.float32])
def test_ffn_keeps_the_input_type(gpu, dtype):
    blk = wan.WanAttentionBlock("t2v_cross_attn", 256, 512, 2).to(gpu).to(dtype)
    h = torch.randn(1, 130, 256, device=gpu).to(dtype)
    l0, l2 = blk.ffn[0], blk.ffn[2] = MXLinear(blk.ffn[0]), MXLinear(blk.ffn[2])
    y = blk._ffn(h)
    assert y.dtype == dtype
    assert torch.equal(y, mx_linear(l0(h, "gelu_tanh", "mxfp4"), l2.weight, l2.bias, out_dtype=dtype))
