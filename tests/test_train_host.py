"""Argument checks of the training operators that need no GPU: the C entry points refuse before any device work, and the
Python functions refuse tensors that are not on a GPU."""
import ctypes

import pytest
import torch

from icsa_hip import (_lib, cross_attn_bwd_hip, cross_attn_fwd_hip, cross_attn_func, layer_norm_func, rms_norm_func, rotary_func)
from icsa_hip.hip_host import IcsaArgumentError

pytestmark = pytest.mark.cpu
BF = torch.bfloat16
PTR = 1 << 20                # a 16-byte aligned address that no check may follow
EIN, EUN, EWS = _lib.EINVAL, _lib.EUNSUPPORTED, _lib.EWORKSPACE


def _fwd(**kw):
    a = dict(q=PTR, q_sb=0, q_ss=128, q_sh=128, k=PTR, k_sb=0, k_ss=128, k_sh=128, v=PTR, v_sb=0, v_ss=128, v_sh=128,
             B=1, Sq=8, Sk=8, H=1, Hk=1, D=128, qst=0, kst=0, docs=1, scale=0.1, out=PTR, o_sb=0, o_ss=128, o_sh=128, lse=PTR, rest=PTR,
             ws=0, wsb=0, stream=0)
    a.update(kw)
    return _lib.lib().icsa_cross_attn_fwd(*a.values())


def _bwd(**kw):
    a = dict(do=PTR, do_sb=0, do_ss=128, do_sh=128, q=PTR, q_sb=0, q_ss=128, q_sh=128, k=PTR, k_sb=0, k_ss=128, k_sh=128,
             v=PTR, v_sb=0, v_ss=128, v_sh=128, out=PTR, o_sb=0, o_ss=128, o_sh=128, lse=PTR, rest=PTR,
             B=1, Sq=8, Sk=8, H=1, Hk=1, D=128, qst=0, kst=0, docs=1, scale=0.1, gd=_lib.BF16,
             dq=PTR, dq_sb=0, dq_ss=128, dq_sh=128, dk=PTR, dk_sb=0, dk_ss=128, dk_sh=128, dv=PTR, dv_sb=0, dv_ss=128, dv_sh=128,
             ws=PTR, wsb=1 << 30, stream=0)
    a.update(kw)
    return _lib.lib().icsa_cross_attn_bwd(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(B=0), EIN), (dict(H=3, Hk=2), EIN), (dict(D=96), EUN), (dict(docs=0), EIN), (dict(docs=2), EIN), (dict(qst=PTR), EIN),
    (dict(scale=0.0), EIN), (dict(scale=float("nan")), EIN), (dict(q=0), EIN), (dict(k=0), EIN), (dict(q=PTR + 2), EIN),
    (dict(k_ss=129), EIN), (dict(rest=PTR + 8), EIN), (dict(Sk=(1 << 30) + 1), EUN), (dict(Sq=(1 << 30) + 1), EUN),
])
def test_cross_attention_refuses(kw, code):
    assert _fwd(**kw) == code and _lib.lib().icsa_last_error()
    assert _bwd(**kw) == code and _lib.lib().icsa_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(gd=7), EIN), (dict(do=0), EIN), (dict(out=0), EIN), (dict(lse=0), EIN), (dict(dq=PTR + 8), EIN), (dict(dk_ss=4), EIN),
    (dict(ws=0), EWS), (dict(wsb=8), EWS), (dict(ws=PTR + 8), EWS), (dict(k_ss=-128), EIN), (dict(q_ss=-128), EIN),
    (dict(k_ss=1 << 28), EUN), (dict(q_ss=1 << 28), EUN), (dict(do_ss=1 << 28), EUN), (dict(H=8, q_sh=1 << 28), EUN),
    (dict(H=8, do_sh=-128), EIN), (dict(scale=1e-30), EIN),
])
def test_cross_attention_backward_refuses(kw, code):
    assert _bwd(**kw) == code and _lib.lib().icsa_last_error()


def test_cross_attention_workspaces():
    L = _lib.lib()
    for sizes in ((1, 1, 1, 1, 1, 64), (1, 65520, 512, 40, 40, 128), (2, 9373, 1009, 24, 8, 64), (1, 1, 65536, 40, 8, 128)):
        B, Sq, Sk, H, Hk, D = sizes
        assert L.icsa_cross_attn_bwd_workspace_size(*sizes, 1) >= 4 * B * Sq * H
    assert L.icsa_cross_attn_bwd_workspace_size(1, 4, 4, 3, 2, 64, 1) == -1
    assert L.icsa_cross_attn_workspace_size(1, 4, 4, 2, 2, 96, 1) == -1
    assert L.icsa_cross_attn_workspace_size(1, 9373, 512, 12, 12, 128, 1) == 0


def _norm(back, **kw):
    L = _lib.lib()
    if back:
        a = dict(dy=PTR, yd=_lib.F32, dy_ss=8, x=PTR, xd=_lib.BF16, x_ss=8, rows=4, groups=1, dim=8, gain=PTR, pd=_lib.F32, p_sg=8, plus=0,
                 rms=0, mean=PTR, rstd=PTR, dx=PTR, dx_ss=8, dgain=PTR, dshift=PTR, ws=PTR, wsb=1 << 20, stream=0)
    else:
        a = dict(x=PTR, xd=_lib.BF16, x_ss=8, rows=4, groups=1, dim=8, gain=PTR, shift=PTR, pd=_lib.F32, p_sg=8, plus=0, rms=0, eps=1e-6,
                 y=PTR, yd=_lib.F32, y_ss=8, mean=PTR, rstd=PTR, stream=0)
    a.update(kw)
    return (L.icsa_norm_bwd if back else L.icsa_norm_fwd)(*a.values())


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("kw,code", [
    (dict(xd=5), EIN), (dict(yd=5), EIN), (dict(pd=5), EIN), (dict(rows=-1), EIN), (dict(groups=0), EIN), (dict(dim=0), EIN),
    (dict(dim=8193), EUN), (dict(groups=65536), EUN), (dict(x=0), EIN), (dict(mean=0), EIN),
])
def test_norms_refuse(back, kw, code):
    assert _norm(back, **kw) == code and _lib.lib().icsa_last_error()


def test_norms_refuse_more():
    assert _norm(False, eps=-1.0) == _norm(False, eps=float("nan")) == _norm(False, y=0) == EIN
    assert _norm(True, dy=0) == _norm(True, rstd=0) == _norm(True, rows=0) == EIN
    assert _norm(True, rows=40, ws=0) == _norm(True, rows=40, wsb=4) == _norm(True, rows=40, ws=PTR + 4) == EWS
    assert _norm(False, rows=0, x=0, y=0) == _norm(True, rows=0, dgain=0, dshift=0) == _norm(True, dx=0, dgain=0, dshift=0) == _lib.OK
    L = _lib.lib()
    assert L.icsa_norm_bwd_workspace_size(9, 1, 5) >= 2 * 8 * 4 and L.icsa_norm_bwd_workspace_size(4, 0, 8) == -1
    assert L.icsa_norm_bwd_workspace_size(0, 1, 8) == L.icsa_norm_bwd_workspace_size(2, 4, 8192) == 0


def _rotary(sections=None, **kw):
    a = dict(x0=PTR, sb0=0, ss0=64, sh0=64, H0=2, y0=PTR, x1=PTR, sb1=0, ss1=64, sh1=64, H1=1, y1=PTR, dt=_lib.BF16, B=1, S=4, D=64, R=64,
             inter=1, back=0, pos=PTR, pos_sb=0, axes=1, sec=None, cos=PTR, sin=PTR, rows=16, stream=0)
    if sections is not None:
        a.update(axes=len(sections), sec=ctypes.cast((ctypes.c_int32 * len(sections))(*sections), ctypes.c_void_p))
    a.update(kw)
    return _lib.lib().icsa_rotary(*a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(dt=5), EIN), (dict(R=63), EIN), (dict(R=0), EIN), (dict(R=66), EIN), (dict(B=-1), EIN), (dict(axes=0), EIN), (dict(axes=5), EIN),
    (dict(axes=2), EIN), (dict(sections=(8, 8, 8)), EIN), (dict(sections=(40, -8)), EIN), (dict(rows=0), EIN), (dict(pos=0), EIN),
    (dict(cos=0), EIN), (dict(x0=0), EIN), (dict(y1=0), EIN), (dict(H0=1 << 21), EUN),
])
def test_rotary_refuses(kw, code):
    assert _rotary(**kw) == code and _lib.lib().icsa_last_error()


def test_rotary_without_work_is_nothing():
    assert _rotary(S=0, x0=0, x1=0) == _rotary(B=0) == _rotary(H0=0, H1=0) == _lib.OK


def test_tensors_on_the_cpu_are_refused():
    q, k = torch.zeros(1, 4, 2, 64, dtype=BF), torch.zeros(1, 5, 1, 64, dtype=BF)
    x, t = torch.zeros(3, 8), torch.zeros(4, 32)
    for call in (lambda: cross_attn_func(q, k, k), lambda: cross_attn_fwd_hip(q, k, k),
                 lambda: cross_attn_bwd_hip(q, q, k, k, q, torch.zeros(1, 1, 4, 2)), lambda: layer_norm_func(x), lambda: rms_norm_func(x),
                 lambda: rotary_func(q, None, t, t, torch.zeros(4, dtype=torch.int32)), lambda: cross_attn_func(q.float(), k, k)):
        with pytest.raises(IcsaArgumentError):
            call()
