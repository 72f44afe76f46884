"""The 4-bit layers and the attention under masks as the block calls them, in runs together, on other
streams and in captured graphs."""
import math

import pytest
import torch
import torch.nn as nn

from icsa_hip import MXLinear, masked_attn_func, mx_linear, mx_quantize, wan
from oracle import wan_glue as W
from test_wan_block_oracle import _params

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


class _Apart(nn.Module):
    """A linear layer that quantises its own input in its own call."""

    def __init__(self, linear):
        super().__init__()
        self.w, self.b = mx_quantize(linear.weight.detach()), linear.bias.detach()

    def forward(self, x, activation=None):
        return mx_linear(x, self.w, self.b, activation=activation)


def _block(gpu, dim, ffn, H):
    blk = wan.WanAttentionBlock("t2v_cross_attn", dim, ffn, H, cross_attn_norm=True)
    blk.load_state_dict({k: v.float() for k, v in _params(dim, ffn, 3).items()}, strict=True)
    return blk.to(gpu).to(BF)


@pytest.mark.parametrize("lens", [None, [24], [5]])
def test_block_with_quantized_layers(gpu, lens):
    """quantize_linears changes the layers alone: the block equals, bit for bit, one whose layers each
    quantise their own input, with the hidden row of the FFN quantised from f32."""
    dim, ffn, H, grid = 256, 512, 2, (2, 16, 16)
    print(f"[mx block] lens={lens}", flush=True)
    a, b = _block(gpu, dim, ffn, H), _block(gpu, dim, ffn, H)
    S = 2 * math.prod(grid)
    g = torch.Generator().manual_seed(11)
    x, e = torch.randn(1, S, dim, generator=g).to(gpu), (torch.randn(1, 6, dim, generator=g) * 0.1).to(gpu)
    ctx = torch.randn(1, 24, dim, generator=g).to(BF).to(gpu)
    args = (e, torch.tensor([S]), [grid], W.wan_freqs(128), ctx, lens, [grid], 1)
    before = a(x, *args)
    assert wan.quantize_linears(a) is a and isinstance(a.ffn[2], MXLinear) and isinstance(a.cross_attn.o, MXLinear)
    wan.quantize_linears(a)                                   # a second call changes nothing
    ffn0, ffn2 = _Apart(b.ffn[0]), _Apart(b.ffn[2])
    for att in (b.self_attn, b.cross_attn):
        for n in ("q", "k", "v", "o"):
            setattr(att, n, _Apart(getattr(att, n)))
    b._ffn = lambda h: ffn2(mx_linear(h, ffn0.w, ffn0.b, activation="gelu_tanh", out_dtype=torch.float32))
    out, ref = a(x, *args), b(x, *args)
    assert torch.isfinite(out).all() and torch.equal(out, ref)
    assert not torch.equal(out, before)


@torch.no_grad()
def test_one_quantized_ffn_layer(gpu):
    """Either FFN layer alone in 4 bits: the other takes its bf16 results, or gives it bf16."""
    h = torch.randn(1, 130, 256, device=gpu).to(BF)
    for i in (0, 2):
        blk = _block(gpu, 256, 512, 2)
        blk.ffn[i] = MXLinear(blk.ffn[i])
        l0, l2 = blk.ffn[0], blk.ffn[2]
        if i == 0:
            ref = nn.functional.linear(l0(h, activation="gelu_tanh"), l2.weight, l2.bias)
        else:
            ref = l2(torch._addmm_activation(l0.bias, h[0], l0.weight.t(), use_gelu=True))[None]
        assert torch.equal(blk._ffn(h), ref)


def test_model_quantizes_every_block(gpu):
    m = wan.WanModel(in_dim=4, dim=256, ffn_dim=512, freq_dim=32, text_dim=64, out_dim=4, num_heads=2, num_layers=2, text_len=16)
    m.init_weights()
    nn.init.normal_(m.head.head.weight, std=0.02)
    m = m.to(gpu).to(BF)
    assert m.quantize_linears() is m
    assert sum(isinstance(x, MXLinear) for x in m.modules()) == 2 * 10
    lat = torch.randn(4, 2, 32, 32, device=gpu).to(BF)
    ctx = [torch.randn(12, 64, device=gpu).to(BF)]
    with torch.no_grad():
        out = [m([lat], torch.tensor([637.0], device=gpu), ctx, 1024, [lat])[0] for _ in range(2)]
    assert torch.isfinite(out[0]).all() and torch.equal(*out)
    assert "blocks.1.ffn.0.codes" in m.state_dict()


def test_cross_attention_text_lengths(gpu):
    """context_lens against the dense path on the rows' real tokens alone.  Both are within (2^-8 of P +
    2^-8 of the output, and the scores' few 2^-20) max |v| of the exact value."""
    B, S, L, dim, H = 3, 70, 40, 256, 2
    ca = wan.WanT2VCrossAttention(dim, H).to(gpu).to(BF)
    ca.o = nn.Identity()
    x, ctx = torch.randn(B, S, dim, device=gpu).to(BF), torch.randn(B, L, dim, device=gpu).to(BF)
    ctx[1, 17:] = math.nan                                    # a buffer's unused end
    lens = [40, 17, 0]
    for given in (lens, torch.tensor(lens), torch.tensor(lens, device=gpu)):
        with torch.no_grad():
            y = ca(x, ctx, given)
            for b, n in enumerate(lens):
                if n == 0:
                    assert (y[b] == 0).all()
                    continue
                ref = ca(x[b:b + 1], ctx[b:b + 1, :n].contiguous())[0]
                top = ca.v(ctx[b, :n]).abs().max().item()
                assert (y[b].float() - ref.float()).abs().max().item() <= 2.0 ** -6 * 1.05 * top
    with pytest.raises(ValueError):
        ca(x, ctx, [1, 2])


@torch.no_grad()
@pytest.mark.parametrize("quantized", [False, True])
def test_text_lengths_change_under_a_captured_graph(gpu, quantized):
    B, S, L, dim, H = 3, 70, 40, 256, 2
    ca = wan.WanT2VCrossAttention(dim, H).to(gpu).to(BF)
    if quantized:
        for n in ("q", "k", "v", "o"):
            setattr(ca, n, MXLinear(getattr(ca, n)))
    x, ctx = torch.randn(B, S, dim, device=gpu).to(BF), torch.randn(B, L, dim, device=gpu).to(BF)
    lens = torch.tensor([40, 17, 0], device=gpu)
    all_lens = [lens.clone(), torch.tensor([1, 40, 39], device=gpu), torch.tensor([0, 0, 8], device=gpu)]
    refs = [ca(x, ctx, n) for n in all_lens]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ca(x, ctx, lens)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ca(x, ctx, lens)
    for _ in range(2):
        for n, r in zip(all_lens, refs):
            lens.copy_(n)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, r)
            assert torch.equal(ca(x, ctx, n), r)


def _together(x, w1, b1, w2, k, v, starts):
    """A layer into 4 bits, a layer out of them, attention of its result under documents."""
    h = mx_linear(x, w1, b1, activation="gelu_tanh", out_dtype="mxfp4")
    y = mx_linear(h, w2)
    q = y.view(1, x.shape[0], 4, 64)
    return masked_attn_func(q, k, v, q_starts=starts, k_starts=starts, causal=True, softcap=20.0)


def _inputs(gpu, seed, rows=200):
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn(rows, 320, generator=g)).to(BF).to(gpu), mx_quantize((torch.randn(520, 320, generator=g) / 18).to(gpu)),
            torch.randn(520, generator=g).to(gpu), mx_quantize((torch.randn(256, 520, generator=g) / 23).to(gpu)),
            torch.randn(1, rows, 2, 64, generator=g).to(BF).to(gpu), torch.randn(1, rows, 2, 64, generator=g).to(BF).to(gpu),
            torch.tensor([[0, 30, rows - 50]], dtype=torch.int32, device=gpu))


@torch.no_grad()
def test_other_streams_give_the_same(gpu):
    args = [_inputs(gpu, s) for s in (0, 1)]
    ref = [_together(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    outs = []
    for s, a in zip(streams, args):
        with torch.cuda.stream(s):
            outs.append([_together(*a) for _ in range(3)])
    torch.cuda.synchronize()
    for r, os in zip(ref, outs):
        assert all(torch.equal(r, o) for o in os)


@torch.no_grad()
@pytest.mark.parametrize("rows", [1, 3, 200, 5000])
def test_captured_and_replayed(gpu, rows):
    """Replays with eager work between them, and on new data (documents among it) in the captured inputs."""
    print(f"[mx graph] rows={rows}", flush=True)

    def ins(seed):
        x, w1, b1, w2, k, v, st = _inputs(gpu, seed, max(rows, 100))
        return (x[:rows], w1, b1, w2, k[:, :rows].contiguous(), v[:, :rows].contiguous(), st.clamp(max=rows))

    a, new = list(ins(2)), ins(3)
    ref, ref_new = _together(*a).clone(), _together(new[0], *a[1:4], *new[4:]).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _together(*a)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = _together(*a)
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
        assert torch.equal(_together(*a), ref)
    for i in (0, 4, 5, 6):
        a[i].copy_(new[i])
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ref_new)


@torch.no_grad()
def test_one_query_at_a_time(gpu):
    """Tokens one by one over a growing sequence equal the causal call over all of it, within both bounds."""
    q, k, v = (torch.randn(1, 90, h, 128, device=gpu).to(BF) for h in (4, 2, 2))
    whole = masked_attn_func(q, k, v, causal=True)
    top = v.abs().max().item()
    for i in (0, 1, 63, 64, 89):
        one = masked_attn_func(q[:, i:i + 1], k[:, :i + 1], v[:, :i + 1], causal=True)
        assert (one[:, 0].float() - whole[:, i].float()).abs().max().item() <= 2.0 ** -6 * 1.05 * top


def test_gradients_are_refused(gpu):
    x = torch.randn(4, 256, device=gpu, requires_grad=True)
    w = mx_quantize(torch.randn(8, 256, device=gpu))
    q = torch.randn(1, 4, 2, 64, device=gpu).to(BF).requires_grad_()
    for call in (lambda: mx_quantize(x), lambda: mx_linear(x, w), lambda: mx_linear(x.detach(), w, torch.zeros(8, device=gpu, requires_grad=True)),
                 lambda: masked_attn_func(q, q.detach(), q.detach())):
        with pytest.raises(ValueError, match="backward"):
            call()
    with torch.no_grad():
        assert mx_linear(x, w).shape == (4, 8) and masked_attn_func(q, q, q).shape == q.shape


def test_gpu_refusals(gpu):
    w = mx_quantize(torch.randn(8, 256, device=gpu))
    x = torch.randn(4, 256, device=gpu)
    q = torch.randn(2, 4, 2, 64, device=gpu).to(BF)
    st = torch.zeros(2, 3, dtype=torch.int32, device=gpu)
    for call in (lambda: mx_linear(x[:, :255], w), lambda: mx_linear(x, w, torch.zeros(7, device=gpu)),
                 lambda: mx_linear(x, w, torch.zeros(8)), lambda: mx_linear(x.cpu(), w), lambda: mx_linear(x, w.codes),
                 lambda: masked_attn_func(q, q, q, q_starts=st), lambda: masked_attn_func(q, q, q, q_starts=st, k_starts=st[:, :2]),
                 lambda: masked_attn_func(q, q, q, q_starts=st.long(), k_starts=st.long()),
                 lambda: masked_attn_func(q, q, q, q_starts=st.cpu(), k_starts=st.cpu()),
                 lambda: masked_attn_func(q, q, q, prefix=st[:, :1].contiguous()),
                 lambda: masked_attn_func(q, q, q, causal=True, prefix=st),
                 lambda: masked_attn_func(q, q, q, softcap=-1.0), lambda: masked_attn_func(q, q[:, :, :1], q),
                 lambda: masked_attn_func(q, q, q, bias=torch.zeros(2, 4, device=gpu)),
                 lambda: masked_attn_func(q, q, q, bias=torch.zeros(3, 5, device=gpu)),
                 lambda: masked_attn_func(q, q, q, out_dtype=torch.half),
                 lambda: masked_attn_func(q[..., :32], q[..., :32], q[..., :32])):
        with pytest.raises((ValueError, TypeError)):
            call()
    with pytest.raises(TypeError):
        mx_quantize(x.half())
