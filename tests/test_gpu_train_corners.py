"""Corners of the training operators: sizes at the ends of their ranges, layouts and transforms outside the usual ones, what the
host does during a call, and results that must not depend on how a launch is divided."""
import sys
import threading
import time

import pytest
import torch

from icsa_hip import (_lib, cross_attn_bwd_hip, cross_attn_func, cross_attn_fwd_hip, layer_norm_func, rms_norm_func, rotary_func,
                      rotary_table, wan)
from icsa_hip._lib import IcsaError
from icsa_hip.hip_host import IcsaArgumentError

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


# ------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("H", [1 << 20, (1 << 20) - 3])
def test_rotary_of_one_token_with_as_many_heads_as_there_may_be(gpu, H):
    """Every head is written: heads are alike, so each result is the first one's."""
    x = torch.randn(1, 1, 1, 512, device=gpu).to(BF)
    cos, sin = rotary_table(9, 512)
    pos = torch.full((1, 1), 7, dtype=torch.int32, device=gpu)
    want = rotary_func(x, None, cos, sin, pos)
    fill = torch.full((H, 512), float("nan"), dtype=BF, device=gpu)        # what the result's memory may hold
    del fill
    y = rotary_func(x.expand(1, 1, H, 512), None, cos, sin, pos)
    assert bool((y == want).all())


def test_rotary_tables_with_a_tangent_are_refused(gpu):
    """Forward mode, as with q and k."""
    q = torch.randn(1, 5, 2, 64, device=gpu)
    cos, sin = rotary_table(5, 64)
    pos = torch.arange(5, dtype=torch.int32, device=gpu)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual
        for c, s in ((dual(cos, -sin), sin), (cos, dual(sin, cos))):
            for grad in (False, True):
                with pytest.raises(NotImplementedError), torch.set_grad_enabled(grad):
                    rotary_func(q, None, c, s, pos)


# ------------------------------------------------------------------------------------------
# the producer in front of the sparse attention
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("grid,src,tag,rows", [((2, 5, 6), (1, 5, 6), 1, 5), ((9, 2, 3), (1, 2, 3), 0, 8), ((1, 2, 3), (1, 2, 9), 1, 8),
                                               ((1, -2, 3), (1, 2, 3), 0, 64), ((1, 2, 3), (1, 2, 3), 2, 64),
                                               ((2, 3), (2, 3), 1, 64)])
def test_grids_that_the_prologue_refuses(gpu, grid, src, tag, rows):
    """An axis longer than the table, a negative one, another TAG, two entries: neither way turns some tokens and not others."""
    B, S, H, D = 1, 128, 2, 64
    yq, yk = (torch.randn(B, S, H * D, device=gpu).to(BF) for _ in range(2))
    w = torch.ones(H * D, device=gpu)
    freqs = wan.wan_freqs(D, rows)
    for call in (lambda: wan.wan_qk_prologue(yq, yk, w, w, [grid], [src], tag, freqs, H),
                 lambda: wan.wan_qk_trainable(yq, yk, w, w, wan.rope_positions([grid], [src], tag, B, S, gpu), freqs, H)):
        with pytest.raises((IcsaError, IcsaArgumentError)):
            call()


# ------------------------------------------------------------------------------------------
# norms
# ------------------------------------------------------------------------------------------
def test_norm_means_alone(gpu):
    """Of the C entry point: mean and rstd are optional each."""
    x = torch.randn(7, 640, device=gpu) + 3
    y = torch.empty_like(x)
    both = [torch.full((7,), float("nan"), device=gpu) for _ in range(2)]
    alone = torch.full((7,), float("nan"), device=gpu)

    def run(mean, rstd):
        ptr = lambda t: 0 if t is None else t.data_ptr()
        return _lib.lib().icsa_norm_fwd(x.data_ptr(), _lib.F32, 640, 7, 1, 640, 0, 0, _lib.F32, 0, 0, 0, 1e-6, y.data_ptr(), _lib.F32, 640,
                                        ptr(mean), ptr(rstd), torch.cuda.current_stream().cuda_stream)
    assert run(*both) == run(alone, None) == _lib.OK
    torch.cuda.synchronize()
    assert both[0].isfinite().all() and torch.equal(alone, both[0])


# ------------------------------------------------------------------------------------------
# cross attention
# ------------------------------------------------------------------------------------------
def _far(t, step, dim):
    """t's values with `step` elements between neighbours of one dim."""
    strides = list(t.contiguous().stride())
    strides[dim] = step
    span = sum((n - 1) * s for n, s in zip(t.shape, strides)) + 1
    view = torch.empty(span, dtype=t.dtype, device=t.device).as_strided(t.shape, strides)
    return view.copy_(t)


@pytest.mark.parametrize("far", ["q rows", "k rows", "v rows", "dout rows", "q heads"])
def test_what_the_forward_takes_the_backward_takes(gpu, far):
    """64 rows, with the heads of a group, over more than 2 GiB (heads first in memory, of long sequences): gradients, and the
    same bits as from contiguous tensors."""
    torch.manual_seed(0)
    Sq, Sk, H, Hk = 70, 66, 6, 2
    x = dict(q=torch.randn(1, Sq, H, 64), k=torch.randn(1, Sk, Hk, 64), v=torch.randn(1, Sk, Hk, 64), dout=torch.randn(1, Sq, H, 64))
    x = {n: t.to(gpu, BF) for n, t in x.items()}
    run = lambda q, k, v, dout: (lambda o: (o.detach(), *torch.autograd.grad(o, (q, k, v), dout)))(cross_attn_func(q, k, v))
    leaf = lambda y: [y[n].detach().requires_grad_(n != "dout") for n in ("q", "k", "v", "dout")]
    want = run(*leaf(x))
    name, which = far.split()
    y = dict(x)
    y[name] = _far(x[name], (1 << 28) + (1 << 27) if which == "heads" else (1 << 24) - 64, 2 if which == "heads" else 1)
    for a, b in zip(want, run(*leaf(y))):
        assert torch.equal(a, b)
    out, lse, rest = cross_attn_fwd_hip(y["q"], y["k"], y["v"])
    for a, b in zip(want, (out, *cross_attn_bwd_hip(y["dout"], y["q"], y["k"], y["v"], out, lse, rest))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128])
def test_dq_does_not_depend_on_the_number_of_parts(gpu, D):
    """The same rows by themselves (their keys cut in parts) and beside many others (in one): each dq is divided by its row's total of P
    either way.  A row whose weight lies on few keys would be off by most of a bf16 rounding, 2^-9 or so, without; the order of the
    sums, of at most n float32 terms, moves an element by n 2^-24 of its terms' absolute sum, scale sum |dS k|, where |dS| <= p (|dP| + |D|)."""
    torch.manual_seed(1)
    Sq, Sk, many = 200, 2000, 400
    q, k, v, do = (torch.randn(1, n, 2, D, device=gpu).to(BF) for n in (Sq, Sk, Sk, Sq))
    q = (4 * q).to(BF)                                       # scores of deviation 4: few keys carry a row
    st = lambda n, B: torch.tensor([[0, n]] * B, dtype=torch.int32, device=gpu)

    def dq(B):
        y = [t.expand(B, -1, -1, -1) for t in (q, k, v, do)]
        out, lse, rest = cross_attn_fwd_hip(*y[:3], st(Sq, B), st(Sk, B))
        # its forward's own parts differ too: state of the rows by themselves for both
        return (out, lse, rest), lambda s: cross_attn_bwd_hip(y[3], *y[:3], *s, st(Sq, B), st(Sk, B), grad_dtype=torch.float32,
                                                              need=(True, False, False))[0]
    size = lambda B: _lib.lib().icsa_cross_attn_bwd_workspace_size(B, Sq, Sk, 2, 2, D, 1)
    assert size(1) > 4 * Sq * 2 * D * 2 and size(many) < 4 * many * Sq * 2 * D      # parts, none
    state, one = dq(1)
    _, all_of_them = dq(many)
    a = one(state)[0].double()
    b = all_of_them([t.expand(many, *t.shape[1:]).contiguous() for t in state])[-1].double()
    p = torch.softmax(D ** -0.5 * torch.einsum("qhd,khd->hqk", q[0].float(), k[0].float()), -1)
    dP = torch.einsum("qhd,khd->hqk", do[0].float(), v[0].float())
    dS = p * (dP.abs() + (p * dP).sum(-1, keepdim=True).abs())
    terms = D ** -0.5 * torch.einsum("hqk,khd->qhd", dS, k[0].float().abs())
    assert ((a - b).abs() <= 1.1 * (Sk + 64) * 2.0 ** -24 * terms.double()).all(), ((a - b).norm() / b.norm()).item()


# ------------------------------------------------------------------------------------------
# the host
# ------------------------------------------------------------------------------------------
def test_other_threads_run_during_a_call(gpu):
    """The operators leave the interpreter to others while they allocate and launch.  The other thread counts; the interpreter is not
    taken from this one by time (the switch interval), so that it counts only where a call lets go of it.  Results of 1 GiB of new
    memory each make the calls long enough."""
    x = torch.zeros(1 << 17, 4096, dtype=BF, device=gpu)
    q = torch.zeros(1, 1 << 16, 64, 128, dtype=BF, device=gpu)
    k = torch.zeros(1, 1, 64, 128, dtype=BF, device=gpu)
    table, pos = rotary_table(1, 128), torch.zeros(1 << 16, dtype=torch.int32, device=gpu)
    calls = [lambda: rms_norm_func(x), lambda: rotary_func(q, None, *table, pos), lambda: cross_attn_func(q, k, k)]
    for call in calls:
        call()
    torch.cuda.synchronize()
    counted, stop = [0], threading.Event()

    def count():
        while not stop.is_set():
            counted[0] += 1
            time.sleep(0)
    other = threading.Thread(target=count)
    interval = sys.getswitchinterval()
    other.start()
    try:
        sys.setswitchinterval(30.0)
        for call in calls:
            moved = False
            for _ in range(60):
                torch.cuda.empty_cache()
                before = counted[0]
                y = call()
                moved = moved or counted[0] > before
                del y
                if moved:
                    break
            assert moved
    finally:
        sys.setswitchinterval(interval)
        stop.set()
        other.join()


# ------------------------------------------------------------------------------------------
# transforms
# ------------------------------------------------------------------------------------------
def _calls(gpu):
    """(an input, the operator of it) for each."""
    torch.manual_seed(2)
    x, q = torch.randn(3, 2, 9, 128, device=gpu), torch.randn(3, 1, 9, 2, 64, device=gpu).to(BF)
    table, pos = rotary_table(9, 64), torch.arange(9, dtype=torch.int32, device=gpu)
    return [(x, lambda t: layer_norm_func(t)), (x, lambda t: rms_norm_func(t)), (q, lambda t: cross_attn_func(t, t, t)),
            (q, lambda t: rotary_func(t, None, *table, pos)), (q, lambda t: cross_attn_fwd_hip(t, t, t)[0])]


def test_transforms_are_refused(gpu):
    """vmap, torch.func, batched gradients, tracing (whose result would be memory that nothing fills) and tensors without memory."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    for x, f in _calls(gpu):
        for transformed in (lambda: torch.func.vmap(f)(x), lambda: torch.func.grad(lambda t: f(t).float().sum())(x[0]),
                            lambda: torch.func.functionalize(f)(x[0])):
            with pytest.raises((NotImplementedError, RuntimeError)):
                transformed()
        with pytest.raises(NotImplementedError, match="memory of their own"):
            torch.jit.trace(f, (x[0],))
        with FakeTensorMode(allow_non_fake_inputs=True) as mode:
            with pytest.raises((NotImplementedError, RuntimeError)):
                f(mode.from_tensor(x[0]))
    for x, f in _calls(gpu)[:4]:
        with pytest.raises(NotImplementedError, match="memory of their own"):
            torch.func.vmap(f)(x)
        leaf = x[0].requires_grad_()
        y = f(leaf)
        with pytest.raises(NotImplementedError, match="memory of their own"):
            torch.autograd.grad(y, leaf, torch.ones(2, *y.shape, dtype=y.dtype, device=gpu), is_grads_batched=True)
    x, w = torch.randn(4, 16, device=gpu), torch._efficientzerotensor(16, device=gpu)
    with pytest.raises(NotImplementedError, match="memory of their own"):
        layer_norm_func(x, w)                                # its address is null, as that of no weight


def test_views_with_a_sign(gpu):
    """What a conjugate's imaginary part is: values of the other sign than memory's."""
    x, w = torch.randn(6, 64, device=gpu), torch.randn(64, device=gpu)
    neg = torch._neg_view
    assert torch.equal(layer_norm_func(neg(x), neg(w)), layer_norm_func(-x, -w))
    assert torch.equal(rms_norm_func(neg(x)), rms_norm_func(-x))
    q = torch.randn(1, 6, 2, 64, device=gpu)
    cos, sin = rotary_table(6, 64)
    pos = torch.arange(6, dtype=torch.int32, device=gpu)
    want = rotary_func(-q, None, cos, -sin, pos)
    assert torch.equal(rotary_func(neg(q), None, cos, neg(sin), pos), want)
    assert torch.equal(rotary_func(-q, None, cos, torch.complex(cos, sin).conj().imag, pos), want)
    leaf = x.clone().requires_grad_()
    a, = torch.autograd.grad(layer_norm_func(leaf), leaf, neg(x))
    b, = torch.autograd.grad(layer_norm_func(leaf), leaf, -x)
    assert torch.equal(a, b)


def test_checkpointed(gpu):
    """Recomputed in the backward: the same gradients."""
    from torch.utils.checkpoint import checkpoint
    for x, f in _calls(gpu)[:4]:
        leaf = x[0].clone().requires_grad_()
        dy = torch.randn_like(f(x[0]))
        want, = torch.autograd.grad(f(leaf), leaf, dy)
        for reentrant in (False, True):
            leaf.grad = None
            checkpoint(f, leaf, use_reentrant=reentrant).backward(dy)
            assert torch.equal(leaf.grad, want)


# ------------------------------------------------------------------------------------------
# the cross attention's sublayer
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lens", [None, [50, 7]])
def test_the_key_bias_has_its_gradient(gpu, lens):
    """A bias of the keys shifts all scores of a row alike but for the norm behind it; over text tokens of different sizes its gradient is
    several times the tokens' terms.  These are of at most 16 roundings to bf16, 2^-8 of a tensor's 2-norm each (norm, q and k, their norms,
    P, out, o's input and result, and back), and a sum of n rows is off by sqrt(n) times their error's 2-norm at most.  The gradient
    is over twice that bound, so that a missing one, off by all of it, fails."""
    torch.manual_seed(0)
    dim, H, B, S, T = 256, 2, 2, 70, 60
    att = wan.WanT2VCrossAttention(dim, H, trainable=True).to(gpu, BF)
    with torch.no_grad():
        for n in (att.norm_q, att.norm_k):
            n.weight.copy_(0.5 + 0.1 * torch.randn(dim))
    x = torch.randn(B, S, dim, device=gpu).to(BF)
    text = (torch.randn(B, T, dim, device=gpu) * torch.exp(torch.randn(B, T, 1, device=gpu))).to(BF)
    dy = torch.randn(B, S, dim, device=gpu).to(BF)
    got, = torch.autograd.grad(att(x, text, lens), att.k.bias, dy)

    P = {n: p.detach().double() for n, p in att.named_parameters() if "alpha" not in n}
    lin = lambda v, n: v @ P[n + ".weight"].t() + P[n + ".bias"]
    rms = lambda v, g: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + att.eps) * g
    C = text.double()
    yk = lin(C, "k").requires_grad_()
    q, k = rms(lin(x.double(), "q"), P["norm_q.weight"]), rms(yk, P["norm_k.weight"])
    q, k, v = (t.unflatten(2, (H, dim // H)).transpose(1, 2).contiguous() for t in (q, k, lin(C, "v")))
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * (dim // H) ** -0.5
    if lens is not None:
        see = torch.arange(T, device=gpu)[None] < torch.tensor(lens, device=gpu)[:, None]
        s = s.masked_fill(~see[:, None, None], float("-inf"))
    y = lin(torch.matmul(torch.softmax(s, -1), v).transpose(1, 2).flatten(2), "o")
    terms, = torch.autograd.grad(y, yk, dy.double())
    want = terms.sum((0, 1))
    n = B * T if lens is None else sum(lens)                # padding has no terms
    bound = 16 * 2.0 ** -8 * n ** 0.5 * terms.norm()
    assert want.norm() > 2 * bound
    assert (got.double() - want).norm() <= bound, ((got.double() - want).norm() / bound).item()
