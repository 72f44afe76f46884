"""The float64 oracles of the training operators against automatic differentiation of the plain formulas and against
differences, and the long-context tables against their definitions."""
import math

import pytest
import torch

from icsa_hip import rotary_table
from icsa_hip.hip_host import IcsaArgumentError
from oracle import cross_attn as A
from oracle import norm_rotary as N

pytestmark = pytest.mark.cpu


def _r(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape)), dtype=torch.float64)


def _plain_attention(q, k, v, q_starts, k_starts):
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1:3]
    see = torch.zeros(B, 1, Sq, Sk, dtype=torch.bool)
    for b, i0, i1, j0, j1 in A.documents(B, Sq, Sk, q_starts, k_starts):
        see[b, :, i0:i1, j0:j1] = True
    k, v = (t.repeat_interleave(H // Hk, 2).transpose(1, 2) for t in (k, v))
    s = (q.transpose(1, 2) @ k.transpose(2, 3)) / math.sqrt(D)
    p = torch.where(see, torch.exp(s - s.amax(-1, keepdim=True)), 0.0)
    total = p.sum(-1, keepdim=True)
    return (p / torch.where(total > 0, total, 1.0) @ v).transpose(1, 2)


@pytest.mark.parametrize("starts", [None, ([[0, 3, 3, 9], [2, 5, 9, 11]], [[0, 4, 6, 8], [1, 1, 7, 8]])])
def test_cross_attention_against_autograd_and_differences(starts):
    q, k, v, do = _r(2, 11, 4, 8), _r(2, 9, 2, 8), _r(2, 9, 2, 8, seed=1), _r(2, 11, 4, 8, seed=2)
    qs, ks = (None, None) if starts is None else (torch.tensor(x) for x in starts)
    val, tol = A.cross_attention(q, k, v, do, q_starts=qs, k_starts=ks)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = _plain_attention(*leaves, qs, ks)
    grads = torch.autograd.grad(out, leaves, do)
    assert torch.allclose(val["out"], out.detach(), atol=1e-13)
    for n, g in zip(("dq", "dk", "dv"), grads):
        assert torch.allclose(val[n], g, atol=1e-12) and (tol[n] >= 0).all()
    h = 1e-5                                                # central differences: h^2 / 6 of third derivatives, 1e-16 / h of rounding
    for i, n in enumerate(("dq", "dk", "dv")):
        for at in ((0, 2, 1, 3), (1, 7, 0, 5), (1, 4, 1, 0)):
            f = []
            for sign in (1, -1):
                x = [t.clone() for t in (q, k, v)]
                x[i][at] += sign * h
                f.append((A.cross_attention(*x, do, q_starts=qs, k_starts=ks)[0]["out"] * do).sum())
            assert abs((f[0] - f[1]) / (2 * h) - val[n][at]) < 1e-8


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("G", [1, 3])
def test_norm_against_autograd(rms, G):
    x, dy, a, b = _r(G, 5, 12), _r(G, 5, 12, seed=1), _r(G, 12), _r(G, 12, seed=3)
    val, tol = N.norm(x, dy, a, b, rms=rms, eps=1e-3)
    leaves = [t.clone().requires_grad_() for t in (x, a, b)]
    X, A_, B_ = leaves
    v = X if rms else X - X.mean(-1, keepdim=True)
    y = v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-3) * A_[:, None] + B_[:, None]
    grads = torch.autograd.grad(y, leaves, dy)
    for n, g in zip(("y", "dx", "da", "db"), (y.detach(), *grads)):
        assert torch.allclose(val[n], g, atol=1e-12) and (tol[n] >= 0).all()


@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_is_a_rotation_and_its_transpose(interleaved):
    x, dy = _r(2, 3, 2, 10), _r(2, 3, 2, 10, seed=1)
    ang = _r(7, 4)
    pos = torch.tensor([[[0, 6], [3, -1], [7, 2]], [[1, 1], [2, 5], [6, 0]]])
    y, _ = N.rotary(x, ang.cos(), ang.sin(), pos, (1, 3), interleaved)
    back, _ = N.rotary(dy, ang.cos(), ang.sin(), pos, (1, 3), interleaved, backward=True)
    assert torch.allclose((y * dy).sum(), (x * back).sum())                # <R x, dy> = <x, R^T dy>
    assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1)) and torch.equal(y[..., 8:], x[..., 8:])
    j = (0, 1) if interleaved else (0, 4)
    assert torch.equal(y[0, 2][:, list(j)], x[0, 2][:, list(j)])            # position 7 is outside the table
    z = torch.complex(x[0, 1, :, j[0]], x[0, 1, :, j[1]]) * torch.exp(1j * ang[3, 0])
    assert torch.allclose(y[0, 1, :, j[0]], z.real) and torch.allclose(y[0, 1, :, j[1]], z.imag)


def test_tables_for_long_contexts():
    cpu = dict(device="cpu")
    c, s = rotary_table(100, 16, **cpu)
    assert c.shape == (100, 8) and c.dtype == torch.float32
    ang = 37 * 10000.0 ** (-2 * 3 / 16)
    assert abs(c[37, 3].item() - math.cos(ang)) < 1e-7 and abs(s[37, 3].item() - math.sin(ang)) < 1e-7
    lin = rotary_table(400, 16, scaling="linear", factor=4.0, **cpu)
    assert torch.allclose(lin[0][::4], c) and torch.allclose(lin[1][::4], s)
    base = rotary_table(400, 16, scaling="base", factor=4.0, **cpu)
    assert torch.allclose(base[0][:, 0], rotary_table(400, 16, **cpu)[0][:, 0])           # the fastest pair stays
    assert torch.allclose(base[1][:, 7], lin[1][:, 7], atol=1e-6)                          # the slowest as with "linear"
    far = rotary_table(1 << 17, 4, **cpu)[0][131071, 0].item()                             # an angle of 131,071 needs float64
    assert abs(far - math.cos(131071.0)) < 1e-7
    mix = rotary_table(400, 64, scaling="blend", factor=4.0, trained=100, **cpu)
    gain = 0.1 * math.log(4) + 1
    turns = [100 * 10000.0 ** (-2 * j / 64) / (2 * math.pi) for j in range(32)]
    for j, t in enumerate(turns):
        keep = min(max((t - 1) / 31, 0), 1)
        inv = 10000.0 ** (-2 * j / 64) * (keep + (1 - keep) / 4)
        assert abs(mix[1][399, j].item() - gain * math.sin(399 * inv)) < 2e-7
    one = rotary_table(10, 2, scaling="linear", factor=2.0, **cpu)
    assert one[0].shape == (10, 1)
    for kw in (dict(positions=0, rotary_dim=4), dict(positions=4, rotary_dim=3), dict(positions=4, rotary_dim=4, scaling="other"),
               dict(positions=4, rotary_dim=4, factor=2.0), dict(positions=4, rotary_dim=4, scaling="linear", factor=0.5),
               dict(positions=4, rotary_dim=4, scaling="blend", factor=2.0), dict(positions=4, rotary_dim=2, scaling="base", factor=2.0),
               dict(positions=4, rotary_dim=4, theta=0.0)):
        with pytest.raises(IcsaArgumentError):
            rotary_table(**kw, **cpu)
