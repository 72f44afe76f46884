"""Types and places of the 4-bit layers in the modules: results in the input's type also where an input is quantised once for
several layers, MXLinear in the model's text and time layers and its head, and what the layers' containers read as."""
import math

import pytest
import torch
import torch.nn as nn

from icsa_hip import MXFP4Tensor, MXLinear, mx_linear, wan
from oracle import mxfp4 as O
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


@torch.no_grad()
@pytest.mark.parametrize("text", [(0,), (2,), (0, 2)])
def test_text_and_time_layers_of_the_model(gpu, text):
    """MXLinear in the place of a Linear of the text embedding, the time embedding, the time projection and the head: each is
    called once; the time layers and the head in float32, the text layers in the weights' type."""
    torch.manual_seed(2)
    m = wan.WanModel(in_dim=4, dim=256, ffn_dim=512, freq_dim=32, text_dim=64, out_dim=4, num_heads=2, num_layers=1, text_len=16)
    m.init_weights()
    nn.init.normal_(m.head.head.weight, std=0.02)
    m = m.to(gpu).to(BF)
    lat, ctx = torch.randn(4, 2, 32, 32, device=gpu).to(BF), [torch.randn(12, 64, device=gpu).to(BF)]
    args = ([lat], torch.tensor([637.0], device=gpu), ctx, 1024, [lat])
    plain = m(*args)[0]
    calls = {}
    for name, seq, i in [("time0", m.time_embedding, 0), ("time2", m.time_embedding, 2), ("proj", m.time_projection, 1),
                         *((f"text{i}", m.text_embedding, i) for i in text)]:
        seq[i] = MXLinear(seq[i])
        seq[i].register_forward_hook(lambda mod, x, y, name=name: calls.setdefault(name, []).append(y))
    m.head.head = MXLinear(m.head.head)
    m.head.head.register_forward_hook(lambda mod, x, y: calls.setdefault("head", []).append(y))
    out = m(*args)[0]
    assert torch.isfinite(out).all() and out.shape == plain.shape and out.dtype == plain.dtype
    assert torch.equal(out, m(*args)[0])
    assert sorted(calls) == sorted(["time0", "time2", "proj", "head", *(f"text{i}" for i in text)])
    for name, ys in calls.items():
        assert len(ys) == 2
        if not name.startswith("text"):
            assert ys[0].dtype == torch.float32
    # the text embedding: GELU between its layers, whichever of them are in 4 bits
    t0, t2 = m.text_embedding[0], m.text_embedding[2]
    padded = torch.zeros(1, 16, 64, dtype=BF, device=gpu)
    padded[0, :12] = ctx[0]
    if text == (0, 2):
        assert torch.equal(calls["text2"][0], mx_linear(mx_linear(padded, t0.weight, t0.bias, "gelu_tanh", "mxfp4"), t2.weight, t2.bias))
    elif text == (0,):
        assert torch.equal(calls["text0"][0], mx_linear(padded, t0.weight, t0.bias, "gelu_tanh"))
    else:
        hidden = nn.functional.gelu(t0(padded), approximate="tanh")
        assert torch.equal(calls["text2"][0], mx_linear(hidden, t2.weight, t2.bias))


def test_values_past_the_types(gpu):
    """Scale bytes over 252, which mx_quantize does not write: values from 2^128 on, which neither type holds, read as
    infinities; all others exactly."""
    codes = torch.arange(16, dtype=torch.uint8).repeat(16).view(1, 256)
    codes = codes[:, 0::2] | (codes[:, 1::2] << 4)
    scales = torch.tensor([252, 253, 254, 255, 0, 1, 127, 200], dtype=torch.uint8).view(1, 1, 8)
    t = MXFP4Tensor(codes.to(gpu), scales.to(gpu), (1, 256))
    ref = O.values(codes, scales, 256)
    ref = torch.where(ref.abs() >= 2.0 ** 128, torch.sign(ref) * math.inf, ref)
    for dt in (BF, torch.float32):
        got = t.dequantize(dt).cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(torch.nan_to_num(got, nan=0.0, posinf=1e300, neginf=-1e300),
                           torch.nan_to_num(ref, nan=0.0, posinf=1e300, neginf=-1e300))


@pytest.mark.parametrize("lens", [None, [24]])
def test_cross_attention_carries_no_gradient(gpu, lens):
    """With lengths as without: the output projection alone learns."""
    ca = wan.WanT2VCrossAttention(256, 2).to(gpu).to(BF)
    x, ctx = torch.randn(1, 70, 256, device=gpu).to(BF), torch.randn(1, 40, 256, device=gpu).to(BF)
    ca(x, ctx, lens).float().sum().backward()
    assert ca.o.weight.grad is not None
    assert all(m.weight.grad is None for m in (ca.q, ca.k, ca.v, ca.norm_q, ca.norm_k))


@torch.no_grad()
@pytest.mark.parametrize("text", [(0,), (2,), (0, 2)])
def test_text_layers_of_another_type_than_the_model(gpu, text):
    """A float32 text embedding in a bf16 model works in float32, its layers in 4 bits or not."""
    m = wan.WanModel(in_dim=4, dim=256, ffn_dim=512, freq_dim=32, text_dim=64, out_dim=4, num_heads=2, num_layers=1, text_len=16)
    m.init_weights()
    m = m.to(gpu).to(BF)
    m.text_embedding.float()
    for i in text:
        m.text_embedding[i] = MXLinear(m.text_embedding[i])
    seen = []
    m.text_embedding[2].register_forward_hook(lambda mod, x, y: seen.append(y.dtype))
    lat, ctx = torch.randn(4, 2, 32, 32, device=gpu).to(BF), [torch.randn(12, 64, device=gpu).to(BF)]
    out = m([lat], torch.tensor([637.0], device=gpu), ctx, 1024, [lat])[0]
    assert torch.isfinite(out).all() and seen == [torch.float32]
