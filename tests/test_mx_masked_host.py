"""Host-side checks of the 4-bit linear operators and of the attention under masks: argument errors
come back before any device work, the containers check what they are given, and the oracles agree
with independent forms."""
import ctypes
import math

import pytest
import torch
import torch.nn.functional as F

from icsa_hip import MXFP4Tensor, MXLinear, _lib, masked_attn_func, mx_linear, mx_quantize
from icsa_hip.hip_host import IcsaArgumentError
from oracle import masked_attn as A
from oracle import mxfp4 as O

pytestmark = pytest.mark.cpu
BF = torch.bfloat16
PTR = 1 << 20                # a 16-byte aligned address that no check may follow


def test_sizes():
    L = _lib.lib()
    for M, K in ((1, 1), (5, 256), (7, 257), (65520, 13824)):
        Kp = -(-K // 256) * 256
        assert L.icsa_mx_codes_size(M, K) == M * Kp // 2 and L.icsa_mx_scales_size(M, K) == M * Kp // 32
        assert L.icsa_mx_linear_workspace_size(M, 8, K, _lib.MXFP4) == 0
        # one or two rows are quantised inside the product
        assert L.icsa_mx_linear_workspace_size(M, 8, K, _lib.BF16) >= (M * Kp * 17 // 32 if M > 2 else 0)
    assert L.icsa_mx_codes_size(-1, 4) == -1 and L.icsa_mx_scales_size(4, 0) == -1
    assert L.icsa_mx_linear_workspace_size(4, 0, 4, _lib.BF16) == -1
    over = (1 << 31) - 1                         # past the limits, where rounding up would overflow
    assert L.icsa_mx_codes_size(4, over) == L.icsa_mx_scales_size(4, over) == L.icsa_mx_codes_size(1 << 62, 4) == -1
    assert L.icsa_mx_linear_workspace_size(4, 8, over, _lib.BF16) == L.icsa_mx_linear_workspace_size(4, over, 8, _lib.F32) == -1
    assert L.icsa_masked_attn_workspace_size(1, 9373, 9373, 12, 12, 128, 1, 1) == 0
    assert L.icsa_masked_attn_workspace_size(1, 1, 65536, 40, 8, 128, 1, 0) > 0
    assert L.icsa_masked_attn_workspace_size(1, 1, 65536, 40, 7, 128, 1, 0) == -1
    assert L.icsa_masked_attn_workspace_size(1, 1, 65536, 40, 8, 96, 1, 0) == -1


def _mx_linear_args(**kw):
    a = dict(x=PTR, xs=PTR, xd=_lib.MXFP4, x_ss=0, w=PTR, ws=PTR, b=0, bd=_lib.F32, act=0, M=4, N=8, K=256, out=PTR, os=PTR,
             od=_lib.BF16, o_ss=8, wsp=0, wsb=0, stream=0)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(M=-1), _lib.EINVAL), (dict(K=0), _lib.EINVAL), (dict(N=0), _lib.EINVAL), (dict(K=(1 << 22) + 1), _lib.EUNSUPPORTED),
    (dict(M=(1 << 30) + 1), _lib.EUNSUPPORTED), (dict(xd=7), _lib.EINVAL), (dict(od=7), _lib.EINVAL),
    (dict(b=PTR, bd=2), _lib.EINVAL), (dict(act=2), _lib.EINVAL), (dict(w=0), _lib.EINVAL), (dict(ws=0), _lib.EINVAL),
    (dict(w=PTR + 8), _lib.EINVAL), (dict(x=0), _lib.EINVAL), (dict(xs=0), _lib.EINVAL), (dict(out=0), _lib.EINVAL),
    (dict(out=PTR + 4), _lib.EINVAL), (dict(o_ss=7), _lib.EINVAL), (dict(od=_lib.MXFP4, os=0), _lib.EINVAL),
    (dict(xd=_lib.BF16, x_ss=256), _lib.EWORKSPACE), (dict(xd=_lib.F32, x_ss=256, wsp=PTR, wsb=16), _lib.EWORKSPACE),
])
def test_mx_linear_refuses(kw, code):
    L = _lib.lib()
    assert L.icsa_mx_linear(*_mx_linear_args(**kw)) == code
    assert L.icsa_last_error()


def test_mx_linear_without_rows_is_nothing():
    assert _lib.lib().icsa_mx_linear(*_mx_linear_args(M=0, x=0, out=0)) == _lib.OK


def test_mx_quantize_refuses():
    L = _lib.lib()
    assert L.icsa_mx_quantize(PTR, 2, 256, 4, 256, PTR, PTR, 0) == _lib.EINVAL
    assert L.icsa_mx_quantize(0, _lib.F32, 256, 4, 256, PTR, PTR, 0) == _lib.EINVAL
    assert L.icsa_mx_quantize(PTR, _lib.F32, 256, 4, 0, PTR, PTR, 0) == _lib.EINVAL
    assert L.icsa_mx_quantize(PTR, _lib.F32, 256, 4, 256, PTR + 4, PTR, 0) == _lib.EINVAL
    assert L.icsa_mx_quantize(0, _lib.F32, 256, 0, 256, 0, 0, 0) == _lib.OK
    assert L.icsa_mx_dequantize(PTR, 0, 4, 256, PTR, _lib.F32, 256, 0) == _lib.EINVAL
    assert L.icsa_mx_dequantize(PTR, PTR, 4, 256, PTR, _lib.F32, 255, 0) == _lib.EINVAL
    assert L.icsa_mx_dequantize(PTR, PTR, 4, 256, PTR, _lib.MXFP4, 256, 0) == _lib.EINVAL


def _masked_args(**kw):
    a = dict(q=PTR, q_sb=0, q_ss=128, q_sh=128, k=PTR, k_sb=0, k_ss=128, k_sh=128, v=PTR, v_sb=0, v_ss=128, v_sh=128,
             B=1, Sq=8, Sk=8, H=1, Hk=1, D=128, qst=0, kst=0, docs=1, causal=0, prefix=0, scale=0.1, cap=0.0, bias=0, radius=0,
             out=PTR, od=_lib.BF16, o_sb=0, o_ss=128, o_sh=128, ws=0, wsb=0, stream=0)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(B=0), _lib.EINVAL), (dict(Sq=-1), _lib.EINVAL), (dict(H=3, Hk=2), _lib.EINVAL), (dict(Hk=0), _lib.EINVAL),
    (dict(D=96), _lib.EUNSUPPORTED), (dict(Sq=1 << 30, H=2), _lib.EUNSUPPORTED), (dict(od=2), _lib.EINVAL),
    (dict(qst=PTR), _lib.EINVAL), (dict(docs=2), _lib.EINVAL), (dict(docs=0, qst=PTR, kst=PTR), _lib.EINVAL),
    (dict(prefix=PTR), _lib.EINVAL), (dict(scale=math.inf), _lib.EINVAL), (dict(scale=0.0), _lib.EINVAL),
    (dict(scale=-0.1), _lib.EINVAL), (dict(cap=-1.0), _lib.EINVAL),
    (dict(cap=math.nan), _lib.EINVAL), (dict(bias=PTR, radius=-1), _lib.EUNSUPPORTED),
    (dict(bias=PTR, radius=1 << 20), _lib.EUNSUPPORTED), (dict(q=0), _lib.EINVAL), (dict(k=0), _lib.EINVAL),
    (dict(out=0), _lib.EINVAL), (dict(q=PTR + 2), _lib.EINVAL), (dict(k_ss=130), _lib.EINVAL), (dict(k_ss=-128), _lib.EINVAL),
    (dict(Sk=65536), _lib.EWORKSPACE), (dict(cap=4097.0), _lib.EUNSUPPORTED), (dict(cap=1e-31), _lib.EUNSUPPORTED),
    (dict(cap=1e-20, scale=1e20), _lib.EUNSUPPORTED), (dict(scale=2e38), _lib.EUNSUPPORTED),
    (dict(k_ss=1 << 24), _lib.EUNSUPPORTED), (dict(v_ss=1 << 24), _lib.EUNSUPPORTED),
])
def test_masked_attn_refuses(kw, code):
    L = _lib.lib()
    assert L.icsa_masked_attn(*_masked_args(**kw)) == code
    assert L.icsa_last_error()


def test_masked_attn_without_queries_is_nothing():
    assert _lib.lib().icsa_masked_attn(*_masked_args(Sq=0, q=0, out=0)) == _lib.OK


def test_container():
    codes, scales = O.quantize(torch.randn(6, 300))
    t = MXFP4Tensor(codes, scales, (2, 3, 300))
    assert t.shape == (2, 3, 300) and t.device.type == "cpu"
    for bad in ((codes, scales, (2, 3, 600)), (codes, scales, (5, 300)), (codes.int(), scales, (6, 300)),
                (codes[:, ::2], scales, (6, 300)), (codes, scales.permute(1, 0, 2), (6, 300)), (codes, scales, (6, 0))):
        with pytest.raises(IcsaArgumentError):
            MXFP4Tensor(*bad)


def test_python_refusals():
    """Off the GPU every entry refuses (as an AssertionError and a ValueError); nothing is computed another way."""
    w = MXFP4Tensor(*O.quantize(torch.randn(8, 256)), (8, 256))
    x = torch.randn(2, 256)
    for call in (lambda: mx_quantize(x), lambda: w.dequantize(), lambda: mx_linear(x, w), lambda: MXLinear(torch.nn.Linear(256, 8)),
                 lambda: mx_linear(x, x), lambda: mx_linear(x, w, activation="relu"), lambda: mx_linear(x, w, out_dtype=torch.half),
                 lambda: mx_quantize(x.clone().requires_grad_())):
        with pytest.raises(IcsaArgumentError):
            call()
    q = torch.randn(1, 4, 2, 64).to(BF)
    with pytest.raises(IcsaArgumentError, match="GPU"):
        masked_attn_func(q, q, q)
    with pytest.raises(IcsaArgumentError, match="bfloat16"):
        masked_attn_func(q.float(), q, q)


# ---------------------------------------------------------------------------- the oracles
def test_quantizer_oracle_by_search():
    """Each code is a nearest entry of the table under the block's scale, the even one at a tie."""
    x = torch.cat([torch.randn(40, 64) * 3, torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9] * 8)[None]])
    codes, scales = O.quantize(x)
    v = O.values(codes, scales, 64)
    s = torch.exp2(scales.permute(1, 0, 2).reshape(41, -1).double() - 127)[:, :2].repeat_interleave(32, 1)
    table = torch.cat([O.E2M1, -O.E2M1])
    best = (x.double()[..., None] - table * s[..., None]).abs().amin(-1)
    assert torch.equal((x.double() - v).abs(), best)
    amax = x.view(41, 2, 32).abs().amax(-1)
    e = scales.permute(1, 0, 2).reshape(41, -1)[:, :2].long() - 127
    assert ((amax >= torch.exp2(e + 2.0)) & (amax < torch.exp2(e + 3.0))).all()
    tie = v[-1].abs() / s[-1]
    assert tie.tolist() == [0, 1, 1, 2, 2, 4, 4, 6] * 8


@pytest.mark.parametrize("causal", [False, True])
def test_attention_oracle_against_torch(causal):
    q, k, v = (torch.randn(2, 33, 4, 64, dtype=torch.float64) for _ in range(3))
    ref = F.scaled_dot_product_attention(*(t.transpose(1, 2) for t in (q, k, v)), is_causal=causal).transpose(1, 2)
    out, _ = A.attention(q, k, v, causal=causal)
    assert torch.allclose(out, ref, rtol=1e-12, atol=1e-12)


def test_attention_oracle_documents_one_by_one():
    """A packed call is its documents' calls side by side; distances count from each query's own key."""
    q, k, v = (torch.randn(1, n, 2, 64, dtype=torch.float64) for n in (50, 70, 70))
    qs, ks = torch.tensor([[0, 20, 45]]), torch.tensor([[0, 30, 65]])
    bias = torch.randn(2, 9)
    out, _ = A.attention(q, k, v, q_starts=qs, k_starts=ks, causal=True, prefix=torch.tensor([[4, 12]]), bias=bias, softcap=3.0)
    for a, b, c, d, pre in ((0, 20, 0, 30, 4), (20, 45, 30, 65, 12)):
        one, _ = A.attention(q[:, a:b], k[:, c:d], v[:, c:d], causal=True, prefix=torch.tensor([[pre]]), bias=bias, softcap=3.0)
        assert torch.allclose(out[:, a:b], one, rtol=1e-12, atol=1e-12)
    assert (out[:, 45:] == 0).all()


def test_entry_points_are_exported():
    assert {"icsa_mx_linear", "icsa_masked_attn"} <= set(_lib.EXPORTS)
    assert isinstance(ctypes.cast(_lib.lib().icsa_mx_quantize, ctypes.c_void_p).value, int)
