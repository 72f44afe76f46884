"""Layer norm, RMS norm and rotary positions with their gradients on the GPU against float64 (oracle.norm_rotary, whose bounds
count float32 arithmetic; a result's own rounding, half a step of its type, is added here)."""
import pytest
import torch

from icsa_hip import layer_norm_func, rms_norm_func, rotary_func, rotary_table
from icsa_hip._lib import IcsaError
from icsa_hip.hip_host import IcsaArgumentError
from oracle import norm_rotary as O

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def _near(name, x, ref, tol):
    x = x.double().cpu()
    t = tol + torch.finfo(BF if tol is None else _near.dtype).eps / 2 * (ref.abs() + tol)
    d = (x - ref).abs()
    assert (d <= t).all(), f"{name}: {(d / t.clamp(min=1e-300)).max().item():.2f} of the tolerance, {d.max().item():.3e}"


def _close(name, x, ref, tol):
    _near.dtype = x.dtype
    _near(name, x, ref.reshape(x.shape), tol.reshape(x.shape))


def _norm_inputs(G, rows, dim, xt, yt, pt, seed=0):
    g = torch.Generator().manual_seed(seed + dim)
    r = lambda *s: torch.randn(*s, generator=g)
    return ((r(G, rows, dim) * torch.exp(0.5 * r(dim)) + 0.5 * r(G, rows, 1)).to(xt), r(G, rows, dim).to(yt), (0.3 * r(G, dim)).to(pt),
            (0.3 * r(G, dim)).to(pt))


DIMS = [1, 2, 7, 8, 64, 100, 128, 129, 256, 257, 512, 1000, 1024, 1536, 2047, 2048, 4096, 5120, 6144, 8191, 8192]
TYPES = [(BF, BF, F32), (F32, BF, F32), (F32, F32, BF), (BF, F32, BF)]


@pytest.mark.parametrize("i,dim", enumerate(DIMS))
@pytest.mark.parametrize("form", ["affine", "weight", "modulate", "none", "rms", "rms_none"])
def test_norms(gpu, form, i, dim):
    xt, yt, pt = TYPES[i % 4]
    G, rows = (3, 5) if form == "modulate" else (1, (1, 17, 64)[i % 3])
    print(f"[norm] {form} dim={dim} {xt} {yt} {pt} rows={G}x{rows}", flush=True)
    x, dy, a, b = _norm_inputs(G, rows, dim, xt, yt, pt)
    rms = form.startswith("rms")
    gain = None if form.endswith("none") else 1 + a.double() if form == "modulate" else a
    shift = b if form in ("affine", "modulate") else None
    val, tol = O.norm(x, dy, gain, shift, rms=rms, eps=1e-5)
    X, A, B = (t.to(gpu).requires_grad_() for t in (x, a, b))
    if form == "modulate":
        y, leaves = layer_norm_func(X, scale=A, shift=B, eps=1e-5, out_dtype=yt), (X, A, B)
    elif form == "affine":
        w, c = (t.detach()[0].clone().requires_grad_() for t in (A, B))
        y, leaves = layer_norm_func(X, w, c, eps=1e-5, out_dtype=yt), (X, w, c)
    elif form.endswith("none"):
        y, leaves = (rms_norm_func if rms else layer_norm_func)(X, eps=1e-5, out_dtype=yt), (X,)
    else:
        w = A.detach()[0].clone().requires_grad_()
        y, leaves = (rms_norm_func if rms else layer_norm_func)(X, w, eps=1e-5, out_dtype=yt), (X, w)
    grads = torch.autograd.grad(y, leaves, dy.to(gpu))
    for n, got in zip(("y", "dx", "da", "db"), (y.detach(), *grads)):
        _close(n, got, val[n], tol[n])
    with torch.no_grad():
        fn = rms_norm_func if rms else layer_norm_func
        kw = dict(scale=leaves[1], shift=leaves[2]) if form == "modulate" else {}
        assert torch.equal(fn(X, *(() if kw else leaves[1:]), **kw, eps=1e-5, out_dtype=yt), y)


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("G,rows,dim,i", [(1, 8, 5120, 0), (1, 9, 5120, 1), (4, 2, 513, 2), (3, 3, 513, 3), (8, 1, 8192, 0), (9, 1, 8192, 1),
                                          (2, 4, 77, 2), (2, 4, 1, 1), (1, 1, 7, 0), (3, 30, 1536, 3), (2, 40, 100, 0), (5, 3, 2, 1), (300, 2, 512, 2), (40, 2, 2048, 3)])
def test_few_rows_and_many_groups(gpu, G, rows, dim, i, rms):
    """On either side of where columns instead of rows are dealt to workgroups, and of one workgroup a group; strided rows."""
    xt, yt, pt = TYPES[i]
    x, dy, a, b = _norm_inputs(G, rows, dim, xt, yt, pt, 5)
    if rms:
        x, dy, a = x.reshape(1, G * rows, dim), dy.reshape(1, G * rows, dim), a[:1]
        val, tol = O.norm(x, dy, a, None, rms=True)
    else:
        val, tol = O.norm(x, dy, 1 + a.double(), b)
    wide = torch.zeros(*x.shape[:-1], dim + 3, dtype=xt, device=gpu)
    wide[..., 3:] = x.to(gpu)
    X, A, B = wide[..., 3:].requires_grad_(), a.to(gpu).requires_grad_(), b.to(gpu).requires_grad_()
    if rms:
        w = A.detach()[0].clone().requires_grad_()
        y, leaves = rms_norm_func(X, w, out_dtype=yt), (X, w)
    else:
        y, leaves = layer_norm_func(X, scale=A, shift=B, out_dtype=yt), (X, A, B)
    d = dy.to(gpu)
    grads = torch.autograd.grad(y, leaves, d, retain_graph=True)
    for n, got in zip(("y", "dx", "da", "db"), (y.detach(), *grads)):
        _close(n, got, val[n], tol[n])
    for n in range(len(leaves)):                             # one at a time
        assert torch.equal(torch.autograd.grad(y, leaves[n], d, retain_graph=True)[0], grads[n])


@pytest.mark.parametrize("rows,dim", [(4000, 64), (2500, 640), (3121, 1536), (1, 8192), (700, 5120)])
def test_sums_over_many_rows(gpu, rows, dim):
    x, dy, a, b = _norm_inputs(1, rows, dim, BF, BF, F32)
    val, tol = O.norm(x, dy, a, b)
    leaves = [t.to(gpu).requires_grad_() for t in (x, a[0], b[0])]
    run = lambda: torch.autograd.grad(layer_norm_func(*leaves), leaves, dy.to(gpu))
    first, second = run(), run()
    for n, got, again in zip(("dx", "da", "db"), first, second):
        _close(n, got, val[n], tol[n])
        assert torch.equal(got, again)                       # fixed order


def test_norm_rows_with_a_large_mean(gpu):
    """A mean a thousand times the deviation: the variance is of the centred values."""
    x, dy, a, b = _norm_inputs(1, 9, 1536, F32, F32, F32)
    x = x + 1000
    val, tol = O.norm(x, dy, a, b)
    leaves = [t.to(gpu).requires_grad_() for t in (x, a[0], b[0])]
    y = layer_norm_func(*leaves)
    for n, got in zip(("y", "dx", "da", "db"), (y.detach(), *torch.autograd.grad(y, leaves, dy.to(gpu)))):
        _close(n, got, val[n], tol[n])


def test_norm_layouts(gpu):
    """Rows with a stride, transposed batches, slices off 16 bytes, one gradient for all, scale and shift as chunks of one tensor in
    the block's manner ([B, 1, dim]), and one row for every batch row."""
    B, S, dim = 3, 10, 96
    x, dy, a, b = (t.to(gpu) for t in _norm_inputs(B, S, dim, BF, BF, F32))
    w, c = a[0].clone().requires_grad_(), b[0].clone().requires_grad_()
    def run(X, DY):
        X = X.detach().requires_grad_()
        y = layer_norm_func(X, w, c)
        return (y.detach(), *torch.autograd.grad(y, (X, w, c), DY))
    want = run(x, dy)
    wide = torch.zeros(B, S, 2 * dim + 5, dtype=BF, device=gpu)
    wide[..., 3:dim + 3] = x
    wd = torch.zeros(B, S, 2 * dim + 5, dtype=BF, device=gpu)
    wd[..., 1:dim + 1] = dy
    for X, DY in ((wide[..., 3:dim + 3], wd[..., 1:dim + 1]), (x.transpose(0, 1).contiguous().transpose(0, 1), dy),
                  (x.transpose(1, 2).contiguous().transpose(1, 2), dy.transpose(1, 2).contiguous().transpose(1, 2))):
        for p, q in zip(want, run(X, DY)):
            assert torch.equal(p, q)
    one = torch.ones((), dtype=BF, device=gpu).expand_as(x)
    for p, q in zip(run(x, one), run(x, one.contiguous())):
        assert torch.equal(p, q)
    em = torch.randn(B, 6, dim, device=gpu).requires_grad_()
    parts = em.chunk(6, dim=1)
    X = x.detach().requires_grad_()
    gx, gem = torch.autograd.grad(layer_norm_func(X, scale=parts[1], shift=parts[0]), (X, em), dy)
    val, tol = O.norm(x.cpu(), dy.cpu(), 1 + em.detach()[:, 1].cpu().double(), em.detach()[:, 0].cpu())
    _close("dx", gx, val["dx"], tol["dx"])
    _close("scale", gem[:, 1], val["da"], tol["da"])
    _close("shift", gem[:, 0], val["db"], tol["db"])
    assert not gem[:, 2:].any()
    for shape in ((dim,), (1, dim), (1, 1, dim)):
        sc, sh = a[0].reshape(shape).clone().requires_grad_(), b[0].reshape(shape).clone().requires_grad_()
        y = layer_norm_func(x, scale=sc, shift=sh)
        got = torch.autograd.grad(y, (sc, sh), dy)
        val, tol = O.norm(x.reshape(1, -1, dim).cpu(), dy.reshape(1, -1, dim).cpu(), 1 + a[:1].cpu().double(), b[:1].cpu())
        _close("y", y.detach(), val["y"], tol["y"])
        _close("scale", got[0], val["da"], tol["da"])
        _close("shift", got[1], val["db"], tol["db"])


def test_norm_partial_needs_and_empty(gpu):
    x, dy, a, b = (t.to(gpu) for t in _norm_inputs(1, 20, 64, BF, BF, F32))
    w, c = a[0].clone().requires_grad_(), b[0].clone().requires_grad_()
    X = x.detach().requires_grad_()
    full = torch.autograd.grad(layer_norm_func(X, w, c), (X, w, c), dy)
    only_x, = torch.autograd.grad(layer_norm_func(X, w.detach(), c.detach()), X, dy)
    only_b, = torch.autograd.grad(layer_norm_func(x, w.detach(), c), c, dy)
    only_w, = torch.autograd.grad(layer_norm_func(x, w, c.detach()), w, dy)
    assert torch.equal(only_x, full[0]) and torch.equal(only_w, full[1]) and torch.equal(only_b, full[2])
    none = torch.zeros(1, 0, 64, dtype=BF, device=gpu).requires_grad_()
    y = layer_norm_func(none, w, c)
    gx, gw, gb = torch.autograd.grad(y, (none, w, c), torch.zeros_like(y))
    assert y.shape == gx.shape == (1, 0, 64) and not gw.any() and not gb.any()
    none = torch.zeros(0, 5, 64, device=gpu).requires_grad_()              # no batch rows, so no scales either
    s = torch.zeros(0, 64, device=gpu).requires_grad_()
    y = layer_norm_func(none, scale=s, shift=s.detach())
    gx, gs = torch.autograd.grad(y, (none, s), torch.zeros_like(y))
    assert y.shape == gx.shape == (0, 5, 64) and gs.shape == (0, 64)
    X = torch.full((2, 64), 3.0, device=gpu).requires_grad_()              # rows of one value: a variance of 0
    y = layer_norm_func(X, w, c)
    assert torch.equal(y[0], c.detach())
    assert torch.autograd.grad(y, X, torch.ones_like(y))[0].isfinite().all()


def test_a_row_that_is_not_finite_stays_alone(gpu):
    for dim in (96, 640, 5120):
        x, dy, a, b = (t.to(gpu) for t in _norm_inputs(1, 40, dim, F32, F32, F32))
        bad = x.clone()
        bad[0, 7, 3] = float("nan")
        X, Y = x.requires_grad_(), bad.requires_grad_()
        w = a[0].clone().requires_grad_()
        y0, y1 = layer_norm_func(X, w), layer_norm_func(Y, w)
        g0, g1 = torch.autograd.grad(y0, X, dy)[0], torch.autograd.grad(y1, Y, dy)[0]
        keep = [i for i in range(40) if i != 7]
        assert torch.equal(y0[0, keep], y1[0, keep]) and torch.equal(g0[0, keep], g1[0, keep])
        assert y1[0, 7].isnan().all() and g1[0, 7].isnan().all()


def test_norm_refusals(gpu):
    x = torch.zeros(2, 3, 16, device=gpu)
    w, s = torch.ones(16, device=gpu), torch.ones(2, 16, device=gpu)
    for call in (lambda: layer_norm_func(x.half()), lambda: layer_norm_func(x, w[:8]), lambda: layer_norm_func(x, None, w),
                 lambda: layer_norm_func(x, w, scale=s, shift=s), lambda: layer_norm_func(x, scale=s),
                 lambda: layer_norm_func(x, scale=s, shift=w), lambda: layer_norm_func(x, scale=s[:, :8], shift=s[:, :8]),
                 lambda: layer_norm_func(x, scale=s.repeat(2, 1), shift=s.repeat(2, 1)), lambda: layer_norm_func(x[0], scale=s, shift=s),
                 lambda: layer_norm_func(x, w, w.to(BF)), lambda: layer_norm_func(x, w.cpu()), lambda: layer_norm_func(x, eps=-1.0),
                 lambda: layer_norm_func(x, out_dtype=torch.float16), lambda: rms_norm_func(x, s),
                 lambda: rms_norm_func(torch.zeros(1, 8193, device=gpu)), lambda: rms_norm_func(torch.zeros(2, 0, device=gpu))):
        with pytest.raises(IcsaArgumentError):
            call()
    many = torch.zeros(70000, 1, 8, device=gpu, requires_grad=True)          # what the library refuses, a node raises
    with pytest.raises(IcsaError, match="icsa_norm_fwd"):
        layer_norm_func(many, scale=many.detach(), shift=many.detach())


# ------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------
def _turn_inputs(B, S, H, Hk, D, dt, seed=0):
    g = torch.Generator().manual_seed(seed + S)
    return [torch.randn(B, S, h, D, generator=g).to(dt) for h in (H, Hk, H, Hk)]


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("B,S,H,Hk,D,R,sections,dt", [
    (1, 1, 1, 1, 64, 64, None, BF), (2, 5, 3, 1, 128, 128, None, BF), (1, 70, 40, 8, 128, 64, None, BF), (2, 3, 5, 5, 80, 80, None, F32),
    (1, 9, 12, 12, 128, 128, (22, 21, 21), BF), (1, 9, 2, 1, 80, 80, (14, 13, 13), F32), (3, 4, 7, 2, 64, 48, (8, 8, 8), BF),
    (1, 6, 2, 2, 10, 6, None, BF), (1, 6, 2, 2, 7, 2, None, F32), (1, 4, 3, 1, 512, 512, None, BF), (1, 4, 3, 1, 520, 16, None, BF),
    (1, 11, 2, 2, 16, 16, (0, 3, 5, 0), F32), (1, 5, 9, 3, 24, 8, None, BF), (2, 2100, 2, 1, 64, 32, None, BF)])
def test_rotary(gpu, B, S, H, Hk, D, R, sections, dt, interleaved):
    print(f"[rotary] B={B} S={S} H={H}/{Hk} D={D} R={R} {sections} {dt} {interleaved}", flush=True)
    q, k, dq, dk = _turn_inputs(B, S, H, Hk, D, dt)
    A = 1 if sections is None else len(sections)
    P = 50
    pos = torch.randint(-2, P + 2, (B, S, A), generator=torch.Generator().manual_seed(S), dtype=torch.int32)   # some outside
    cos, sin = rotary_table(P, R, device="cpu")
    Q, K = (t.to(gpu).requires_grad_() for t in (q, k))
    args = (cos.to(gpu), sin.to(gpu), (pos[..., 0] if sections is None else pos).to(gpu))
    got = rotary_func(Q, K, *args, sections=sections, interleaved=interleaved)
    grads = torch.autograd.grad(got, (Q, K), (dq.to(gpu), dk.to(gpu)))
    for name, x, back, y in (("q", q, False, got[0]), ("k", k, False, got[1]), ("dq", dq, True, grads[0]), ("dk", dk, True, grads[1])):
        ref, tol = O.rotary(x, cos, sin, pos, sections or (R // 2,), interleaved, back)
        _close(name, y.detach(), ref, tol)
        assert torch.equal(y.detach().cpu()[..., R:], x[..., R:])
    with torch.no_grad():
        alone = rotary_func(Q, None, *args, sections=sections, interleaved=interleaved)
        assert torch.equal(alone, got[0]) and alone.data_ptr() != Q.data_ptr()


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("D,R,sections", [(64, 64, None), (128, 128, (22, 21, 21)), (128, 32, None), (80, 80, (14, 13, 13)), (10, 6, None)])
def test_what_is_not_turned_is_copied(gpu, D, R, sections, interleaved):
    """Pairs whose position is outside the table are the same bits in either direction, infinities and negative zeros too."""
    q, _, dq, _ = _turn_inputs(1, 6, 3, 1, D, BF)
    A = 1 if sections is None else len(sections)
    pos = torch.arange(6, dtype=torch.int32)[None, :, None].repeat(1, 1, A)
    pos[0, 2] = -1
    pos[0, 4, -1] = 50                                       # the last axis alone
    last = (sections or (R // 2,))[-1]
    still = torch.zeros(1, 6, 3, D, dtype=torch.bool)
    still[0, 2] = True
    j = torch.arange(R // 2 - last, R // 2)
    still[0, 4][:, torch.cat([2 * j, 2 * j + 1] if interleaved else [j, j + R // 2])] = True
    hard = torch.tensor([float("inf"), 1.0, -0.0, float("nan"), float("-inf"), 0.0, -0.0, 5.0], dtype=BF)
    for t in (q, dq):
        t[still] = hard.repeat(still.sum() // 8 + 1)[:still.sum()]
    cos, sin = rotary_table(50, R)
    Q = q.to(gpu).requires_grad_()
    y = rotary_func(Q, None, cos, sin, (pos[..., 0] if sections is None else pos).to(gpu), sections=sections, interleaved=interleaved)
    g, = torch.autograd.grad(y, Q, dq.to(gpu))
    bits = lambda t: t.detach().cpu().view(torch.int16)
    for a, b in ((y, q), (g, dq)):
        assert torch.equal(bits(a)[still], bits(b)[still]) and a.detach().cpu()[~still].isfinite().all()


def test_rotary_layouts_and_needs(gpu):
    """Heads first, slices off 16 bytes, shared positions, gradients of one output alone and of one value for all."""
    q, k, dq, dk = (t.to(gpu) for t in _turn_inputs(2, 9, 4, 2, 64, BF))
    cos, sin = rotary_table(100, 64)
    pos = torch.arange(9, dtype=torch.int32, device=gpu) * 11
    want = rotary_func(q, k, cos, sin, pos)
    each = rotary_func(q, k, cos, sin, pos.expand(2, 9))
    wide = torch.zeros(2, 9, 4, 70, dtype=BF, device=gpu)
    wide[..., 3:67] = q
    turned = k.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1)
    first = k.transpose(1, 2).contiguous().transpose(1, 2)
    for a, b in ((each, want), (rotary_func(wide[..., 3:67], turned, cos, sin, pos), want), (rotary_func(q, first, cos, sin, pos), want)):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    Q, K = q.clone().requires_grad_(), k.clone().requires_grad_()
    out = rotary_func(Q, K, cos, sin, pos)
    full = torch.autograd.grad(out, (Q, K), (dq, dk), retain_graph=True)
    assert torch.equal(torch.autograd.grad(out[0], Q, dq, retain_graph=True)[0], full[0])
    assert torch.equal(torch.autograd.grad(out[1], K, dk, retain_graph=True)[0], full[1])
    one = torch.ones((), dtype=BF, device=gpu).expand_as(out[0])
    assert torch.equal(torch.autograd.grad(out[0], Q, one)[0], rotary_func(one, None, cos, -sin, pos))
    K = k.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(rotary_func(q, K, cos, sin, pos)[1], K, dk)[0], full[1])
    empty = rotary_func(q[:, :0], k[:, :0], cos, sin, pos[:0])
    assert empty[0].shape == (2, 0, 4, 64)


def test_rotary_refusals(gpu):
    q, k, _, _ = (t.to(gpu) for t in _turn_inputs(2, 3, 2, 1, 64, BF))
    cos, sin = rotary_table(8, 64)
    pos = torch.zeros(2, 3, dtype=torch.int32, device=gpu)
    p3 = torch.zeros(2, 3, 3, dtype=torch.int32, device=gpu)
    for call in (lambda: rotary_func(q[0], None, cos, sin, pos), lambda: rotary_func(q.half(), None, cos, sin, pos),
                 lambda: rotary_func(q, k.float(), cos, sin, pos), lambda: rotary_func(q, k[:, :2], cos, sin, pos),
                 lambda: rotary_func(q, k, cos, sin[:4], pos), lambda: rotary_func(q, k, cos.to(BF), sin.to(BF), pos),
                 lambda: rotary_func(q[..., :32], k[..., :32], cos, sin, pos), lambda: rotary_func(q, k, cos, sin, pos.long()),
                 lambda: rotary_func(q, k, cos, sin, p3), lambda: rotary_func(q, k, cos, sin, pos, sections=(16, 16)),
                 lambda: rotary_func(q, k, cos, sin, p3, sections=(16, 8, 4)), lambda: rotary_func(q, k, cos, sin, pos[:, :2]),
                 lambda: rotary_func(q, k, cos, sin, pos.cpu()), lambda: rotary_func(q, k, cos.clone().requires_grad_(), sin, pos)):
        with pytest.raises(IcsaArgumentError):
            call()
