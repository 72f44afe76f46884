"""The training operators as they are used together: the cross attention's sublayer with its norms, the sparse attention behind
its q / k norm and rotation; on other streams, in captured graphs, under hooks that move what is saved."""
import pytest
import torch

from icsa_hip import (SparsePiecewiseAttn1stIntervalsFunction, cross_attn_bwd_hip, cross_attn_func, cross_attn_fwd_hip,
                      layer_norm_func, rms_norm_func, rotary_func, rotary_table, wan)
from icsa_hip._lib import IcsaError

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _leaf(t):
    return t.detach().clone().requires_grad_()


def _near(name, got, ref, roundings):
    """2-norm: a rounding to bf16 moves a tensor by 2^-8 of its norm at most, each passes through linear maps and norms whose
    relative condition is about one here (scores under 1), and roundings of the value and of the gradient meet in a product."""
    ref = ref.to(got.device)
    err = (got.double() - ref).norm() / ref.norm().clamp(min=1e-30)
    assert err <= roundings * 2.0 ** -8, f"{name}: {err:.4f}"


@pytest.mark.parametrize("lens", [None, [50, 7]])
def test_cross_attention_sublayer(gpu, lens):
    """x + o(attention(norm3(x))) of the block with text lengths, against the same formulas in float64.  Roundings to bf16 on a
    gradient's longest way: norm3, q, its norm, P, out, o's input and result, and back dout, dS, dq, dx of the norm, of q
    and of norm3: 16 with the weights' own."""
    torch.manual_seed(0)
    dim, H, B, S, T = 256, 2, 2, 70, 60
    att = wan.WanT2VCrossAttention(dim, H, trainable=True).to(gpu, BF)
    with torch.no_grad():
        for n in (att.norm_q, att.norm_k):
            n.weight.copy_(0.5 + 0.1 * torch.randn(dim))
    w, b = (0.2 * torch.randn(dim, device=gpu) + 1).requires_grad_(), (0.2 * torch.randn(dim, device=gpu)).requires_grad_()
    x = torch.randn(B, S, dim, device=gpu).requires_grad_()
    text = torch.randn(B, T, dim, device=gpu).to(BF).requires_grad_()
    dy = torch.randn(B, S, dim, device=gpu)
    y = x + att(layer_norm_func(x, w, b, out_dtype=BF), text, lens).float()
    params = [p for n, p in att.named_parameters() if "alpha" not in n]
    names = [n for n, _ in att.named_parameters() if "alpha" not in n]
    grads = torch.autograd.grad(y, [x, w, b, text, *params], dy)

    d = lambda t: t.detach().double().requires_grad_()
    X, W, Bi, C = d(x), d(w), d(b), d(text)
    P = {n: d(p) for n, p in zip(names, params)}
    lin = lambda v, n: v @ P[n + ".weight"].t() + P[n + ".bias"]
    rms = lambda v, g: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + att.eps) * g
    v = X - X.mean(-1, keepdim=True)
    h = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6) * W + Bi
    q, k = rms(lin(h, "q"), P["norm_q.weight"]), rms(lin(C, "k"), P["norm_k.weight"])
    q, k, vv = (t.unflatten(2, (H, dim // H)).transpose(1, 2).contiguous() for t in (q, k, lin(C, "v")))
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * (dim // H) ** -0.5
    if lens is not None:
        see = torch.arange(T, device=gpu)[None] < torch.tensor(lens, device=gpu)[:, None]
        s = s.masked_fill(~see[:, None, None], float("-inf"))
    o = torch.matmul(torch.softmax(s, -1), vv).transpose(1, 2).flatten(2)
    ref = X + lin(o, "o")
    want = torch.autograd.grad(ref, [X, W, Bi, C, *P.values()], dy.double())
    _near("y", y, ref.detach(), 8)
    for n, a, r in zip(["x", "norm3.weight", "norm3.bias", "text", *names], grads, want):
        if n == "k.bias":                               # shifts all scores of a row alike where k's norm is not there: small by itself
            continue
        _near(n, a, r, 16)
    if lens is not None:
        assert not grads[3][1, lens[1]:].any()          # padding tokens of the text


def test_cross_attention_default_is_as_before(gpu):
    """trainable off: the result has no gradient; both ways agree to the roundings of the norm's row (2, before and after its
    weight) and of the attention (P, out), behind one projection."""
    torch.manual_seed(1)
    att = wan.WanT2VCrossAttention(256, 2).to(gpu, BF)
    x, text = torch.randn(1, 40, 256, device=gpu).to(BF), torch.randn(1, 30, 256, device=gpu).to(BF)
    with torch.no_grad():
        a = att(x, text)
        att.trainable = True
        b = att(x, text)
    _near("out", b, a.double(), 6)
    assert b.requires_grad is False and att(x, text).requires_grad


def test_self_attention_q_k(gpu):
    """Projections -> RMS norm -> rotation -> sparse attention: q and k are the prologue's (to the rounding that it has
    elsewhere: 2 steps), and the gradients are those of the parts put together by hand, bit for bit."""
    torch.manual_seed(2)
    B, H, D, grid, src = 1, 2, 128, (2, 5, 6), (1, 5, 6)
    S, dim = 128, H * D                                     # 90 tokens on the grids, 38 of padding
    yq, yk = (torch.randn(B, S, dim, device=gpu).to(BF).requires_grad_() for _ in range(2))
    wq, wk = ((1 + 0.2 * torch.randn(dim, device=gpu)).requires_grad_() for _ in range(2))
    v = torch.randn(B, H, S, D, device=gpu).to(BF).requires_grad_()
    freqs = wan.wan_freqs(D)
    pos = wan.rope_positions([grid], [src], 1, B, S, gpu)
    q, k = wan.wan_qk_trainable(yq, yk, wq, wk, pos, freqs, H)
    q0, k0 = wan.wan_qk_prologue(yq, yk, wq, wk, [grid], [src], 1, freqs, H)[:2]
    _near("q", q.detach(), q0.double(), 2)
    _near("k", k.detach(), k0.double(), 2)
    out = SparsePiecewiseAttn1stIntervalsFunction.apply(q.transpose(1, 2), k.transpose(1, 2), v, 0.5, 64)
    do = torch.randn_like(out)
    grads = torch.autograd.grad(out, (yq, yk, wq, wk, v), do)

    nq, nk = (rms_norm_func(y, w, out_dtype=BF) for y, w in ((yq, wq), (yk, wk)))
    cos, sin = wan.rope_tables(freqs, gpu)
    tq, tk = (_leaf(t.view(B, S, H, D)) for t in (nq, nk))
    rq, rk = rotary_func(tq, tk, cos, sin, pos, sections=(22, 21, 21))
    assert torch.equal(rq, q) and torch.equal(rk, k)
    lq, lk, lv = (_leaf(t) for t in (rq.transpose(1, 2), rk.transpose(1, 2), v))
    dq, dk, dv = torch.autograd.grad(SparsePiecewiseAttn1stIntervalsFunction.apply(lq, lk, lv, 0.5, 64), (lq, lk, lv), do)
    dq, dk = torch.autograd.grad((rq, rk), (tq, tk), (dq.transpose(1, 2), dk.transpose(1, 2)))
    want = [*torch.autograd.grad(nq, (yq, wq), dq.flatten(2)), *torch.autograd.grad(nk, (yk, wk), dk.flatten(2))]
    for a, b in zip(grads, (want[0], want[2], want[1], want[3], dv)):
        assert torch.equal(a, b)


def _step(t):
    """One pass through all four, and its gradients."""
    x, w, sc, sh, k, v = t["leaves"]
    h = layer_norm_func(x, scale=sc, shift=sh)
    q = rms_norm_func(h, w).unflatten(2, (2, 64))
    q, kk = rotary_func(q, k, *t["table"], t["pos"], interleaved=False)
    y = cross_attn_func(q, kk, v, q_starts=t["qs"], k_starts=t["ks"])
    return (y, *torch.autograd.grad(y, t["leaves"], t["dy"]))


def _tensors(gpu, seed=0, S=100):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(gpu)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)
    leaves = [r(2, S, 128).to(BF), r(128), r(2, 1, 128), r(2, 1, 128), r(2, S, 1, 64).to(BF), r(2, S, 1, 64).to(BF)]
    return dict(leaves=[t.requires_grad_() for t in leaves], dy=r(2, S, 2, 64).to(BF), table=rotary_table(200, 64),
                pos=torch.arange(S, dtype=torch.int32, device=gpu), qs=i([[0, 40, S], [0, S, S]]), ks=i([[0, 70, S], [0, 33, 33]]))


def test_another_stream(gpu):
    t = _tensors(gpu)
    want = _step(t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(t)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_two_captured_graphs(gpu):
    """Forward and backward captured, twice with inputs of their own in one memory pool; replayed in turn with eager work and
    changed borders between, each replay against the eager result."""
    sets = [_tensors(gpu, s) for s in (1, 2)]
    for t in sets:
        _step(t)                                            # first launches set limits
    graphs, outs, pool = [], [], None
    side = torch.cuda.Stream()
    for t in sets:
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool, stream=side):
            outs.append(_step(t))
        pool = g.pool()
        graphs.append(g)
    for turn in range(4):
        for t, g, out in zip(sets, graphs, outs):
            with torch.no_grad():
                t["leaves"][0].copy_(torch.randn_like(t["leaves"][0]))
                t["ks"][0, 1] = 20 + 10 * turn
            g.replay()
            torch.cuda.synchronize()
            kept = [o.clone() for o in out]
            for a, b in zip(kept, _step(t)):
                assert torch.equal(a, b), turn


def test_a_capture_with_an_eager_graph_alive_is_refused(gpu):
    """Nodes of an eager graph that lives, a leaf's and another's; without it, from the capture's own stream, and without
    gradients the same calls are captured."""
    x = torch.randn(2, 9, 128, device=gpu, requires_grad=True)
    q = torch.randn(1, 9, 2, 64, device=gpu).to(BF).requires_grad_()
    table, pos = rotary_table(9, 64), torch.arange(9, dtype=torch.int32, device=gpu)
    calls = [lambda: layer_norm_func(x), lambda: rms_norm_func(x), lambda: cross_attn_func(q, q, q), lambda: rotary_func(q, None, *table, pos)]
    for call in calls:
        call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def captured(call, refused):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            if refused:
                with pytest.raises(IcsaError, match="eager graph"):
                    call()
            else:
                call()
            torch.zeros(1, device=gpu)                       # something to capture
        g.replay()
        torch.cuda.synchronize()

    held = [x * 2, q * 2]
    for call in calls:
        captured(call, True)
        with torch.no_grad():
            captured(call, False)
    h = held[0]
    captured(lambda: layer_norm_func(h), True)               # no leaf: its own node
    captured(lambda: layer_norm_func(h.detach().requires_grad_()), False)
    del held, h
    for call in calls:
        captured(call, False)
    with torch.cuda.stream(side):
        held = [x * 2, q * 2]
    for call in calls:
        captured(call, False)
    torch.cuda.current_stream().wait_stream(side)


def test_the_attentions_pair_in_a_graph(gpu):
    """Parts joined (few queries over many keys, few keys under many queries)."""
    for Sq, Sk in ((3, 2500), (2500, 3)):
        q, k, v, do = (torch.randn(1, n, 4, 64, device=gpu).to(BF) for n in (Sq, Sk, Sk, Sq))
        run = lambda: (lambda o, *s: (o, *cross_attn_bwd_hip(do, q, k, v, o, *s)))(*cross_attn_fwd_hip(q, k, v))
        run()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = run()
        for _ in range(3):
            q.copy_(torch.randn_like(q))
            g.replay()
            torch.cuda.synchronize()
            kept = [o.clone() for o in out]
            for a, b in zip(kept, run()):
                assert torch.equal(a, b)


def test_saved_tensors_moved_and_changed(gpu):
    """Hooks that keep what is saved in host memory (the addresses of the forward no longer hold it), and the refusal of what was
    changed in between."""
    t = _tensors(gpu, 3)
    want = _step(t)
    with torch.autograd.graph.save_on_cpu():
        x, w, sc, sh, k, v = t["leaves"]
        h = layer_norm_func(x, scale=sc, shift=sh)
        q = rms_norm_func(h, w).unflatten(2, (2, 64))
        q, kk = rotary_func(q, k, *t["table"], t["pos"], interleaved=False)
        y = cross_attn_func(q, kk, v, q_starts=t["qs"], k_starts=t["ks"])
    del h, q, kk
    fill = [torch.full((1 << 20,), float("nan"), device=gpu) for _ in range(4)]     # over what was freed
    got = (y, *torch.autograd.grad(y, t["leaves"], t["dy"]))
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    del fill
    v = t["leaves"][5].detach().clone().requires_grad_()
    u = v * 1
    y = cross_attn_func(u, v, v)
    with torch.no_grad():
        u.add_(1)
    with pytest.raises(RuntimeError):
        y.float().sum().backward()


class _Nothing(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x * 1

    @staticmethod
    def backward(ctx, g):
        return None


def test_the_graphs_rules(gpu):
    """A graph used twice, a result changed in place, no gradient for a result, views of it, forward-mode derivatives."""
    x = torch.randn(2, 9, 128, device=gpu, requires_grad=True)
    q = torch.randn(1, 9, 2, 64, device=gpu).to(BF).requires_grad_()
    table, pos = rotary_table(9, 64), torch.arange(9, dtype=torch.int32, device=gpu)
    calls = [(x, lambda t: layer_norm_func(t)), (x, lambda t: rms_norm_func(t)), (q, lambda t: cross_attn_func(t, t, t)),
             (q, lambda t: rotary_func(t, None, *table, pos))]
    for t, f in calls:
        y = f(t)
        dy = torch.randn_like(y)
        assert y.requires_grad and y.is_leaf is False and not f(t.detach()).requires_grad
        want, = torch.autograd.grad(y, t, dy, retain_graph=True)
        assert torch.equal(torch.autograd.grad(y, t, dy)[0], want)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, t, dy)
        got, = torch.autograd.grad(_Nothing.apply(f(t)), t, dy, allow_unused=True)
        assert got is None
        part, = torch.autograd.grad(f(t)[:, :4], t, dy[:, :4])
        assert torch.equal(part, torch.autograd.grad(f(t), t, torch.cat([dy[:, :4], torch.zeros_like(dy[:, 4:])], 1))[0])
        with torch.autograd.forward_ad.dual_level():
            with pytest.raises(NotImplementedError):
                f(torch.autograd.forward_ad.make_dual(t.detach(), dy.to(t.dtype)))
    y = cross_attn_func(q, q, q)                            # its backward reads the result
    with torch.no_grad():
        y.mul_(2)
    with pytest.raises(RuntimeError):
        y.float().sum().backward()
    u = x * 1
    y = layer_norm_func(u.view(18, 128))                    # saved by a view
    with torch.no_grad():
        u.add_(1)
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_backward_into_grads_and_accumulation(gpu):
    t = _tensors(gpu, 4)
    want = _step(t)[1:]
    for _ in range(2):
        x, w, sc, sh, k, v = t["leaves"]
        q, kk = rotary_func(rms_norm_func(layer_norm_func(x, scale=sc, shift=sh), w).unflatten(2, (2, 64)), k, *t["table"], t["pos"],
                            interleaved=False)
        cross_attn_func(q, kk, v, q_starts=t["qs"], k_starts=t["ks"]).backward(t["dy"])
    for leaf, g in zip(t["leaves"], want):
        assert torch.equal(leaf.grad, g + g)
