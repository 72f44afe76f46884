"""Cross attention and its gradients on the GPU against float64 (oracle.cross_attn, whose bounds count f32 scores and sums and
P and dS in bf16; a result's own rounding, 2^-8 of the value in bf16, 2^-22 with sums joined in float32, is added here)."""
import pytest
import torch

from icsa_hip import cross_attn_bwd_hip, cross_attn_func, cross_attn_fwd_hip, masked_attn_func
from icsa_hip.hip_host import IcsaArgumentError
from oracle import cross_attn as O

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
NAMES = ("out", "dq", "dk", "dv")


def _inputs(B, Sq, Sk, H, Hk, D, seed=0):
    g = torch.Generator().manual_seed(seed)
    return ((1.5 * torch.randn(B, Sq, H, D, generator=g)).to(BF), torch.randn(B, Sk, Hk, D, generator=g).to(BF),
            torch.randn(B, Sk, Hk, D, generator=g).to(BF), torch.randn(B, Sq, H, D, generator=g).to(BF))


def _i32(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32)


def _run(gpu, q, k, v, do, qs=None, ks=None, scale=None, grad_dtype=BF):
    q, k, v, do = (t.to(gpu) for t in (q, k, v, do))
    qs, ks = (None if t is None else t.to(gpu) for t in (qs, ks))
    out, lse, rest = cross_attn_fwd_hip(q, k, v, qs, ks, scale)
    return (out, *cross_attn_bwd_hip(do, q, k, v, out, lse, rest, qs, ks, scale, grad_dtype))


def _compare(got, val, tol, own=(2.0 ** -8,) * 4, where=None):
    for i, n in enumerate(NAMES):
        x, ref = got[i].double().cpu(), val[n]
        t = tol[n] + own[i] * (ref.abs() + tol[n])
        d = (x - ref).abs()
        ok = d <= t
        if where is not None:
            ok = ok | ~where[n]
        assert ok.all(), f"{n}: {(d / t.clamp(min=1e-30)).max().item():.2f} of the tolerance, {d.max().item():.3e}"


def _check(gpu, q, k, v, do, qs=None, ks=None, scale=None, grad_dtype=BF):
    keeps = qs is not None or k.shape[1] <= (1024 if q.shape[3] == 64 else 256) or q.shape[1] * (q.shape[2] // k.shape[2]) <= 128
    val, tol = O.cross_attention(q, k, v, do, q_starts=qs, k_starts=ks, scale=scale, rest=keeps)
    got = _run(gpu, q, k, v, do, qs, ks, scale, grad_dtype)
    assert all(x.dtype == (BF if i == 0 else grad_dtype) for i, x in enumerate(got))
    _compare(got, val, tol, (2.0 ** -8,) + ((2.0 ** -8 if grad_dtype == BF else 2.0 ** -22),) * 3)
    return got


SIZES = [(1, 1, 1, 1, 1), (1, 1, 65, 3, 3), (2, 31, 64, 2, 2), (1, 33, 63, 4, 2), (1, 128, 128, 2, 1), (1, 129, 257, 2, 2),
         (3, 7, 130, 10, 2), (1, 200, 77, 5, 5), (1, 1, 3000, 8, 2), (1, 3, 2001, 5, 1), (1, 2000, 1, 2, 2), (1, 1500, 3, 3, 1),
         (1, 300, 513, 6, 2), (1, 0, 10, 2, 1), (1, 10, 0, 2, 2), (1, 65, 500, 7, 1)]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Sq,Sk,H,Hk", SIZES)
def test_sizes(gpu, B, Sq, Sk, H, Hk, D):
    print(f"[cross] B={B} Sq={Sq} Sk={Sk} H={H}/{Hk} D={D}", flush=True)
    _check(gpu, *_inputs(B, Sq, Sk, H, Hk, D, Sq + Sk), grad_dtype=BF if Sq % 2 else torch.float32)


DOCS = [
    # query starts, key starts: ragged documents, empty ones, gaps in front and behind, past the lengths
    ([[0, 64, 128]], [[0, 64, 128]]),
    ([[0, 50, 50, 190]], [[0, 80, 90, 200]]),
    ([[0, 50, 100, 190]], [[0, 80, 80, 200]]),
    ([[7, 20, 150]], [[3, 90, 170]]),
    ([[0, 10, 20, 30, 40, 50, 200]], [[0, 5, 15, 40, 41, 130, 210]]),
    ([[0, 200], [0, 1], [0, 0], [100, 100]], [[0, 77], [0, 210], [0, 210], [3, 50]]),
    ([[0, 100, 250]], [[0, 100, 400]]),
    ([[-20, 90, 1 << 30]], [[-5, 100, 1 << 30]]),
    ([list(range(0, 201, 2))], [list(range(0, 101))]),        # 100 documents of 2 queries and a key
]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 3])
@pytest.mark.parametrize("qs,ks", DOCS)
def test_documents(gpu, qs, ks, G, D):
    print(f"[cross] documents {qs} {ks} G={G} D={D}"[:100], flush=True)
    _check(gpu, *_inputs(len(qs), 200, 210, 2 * G, 2, D, G), _i32(qs), _i32(ks))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 2])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_what_is_outside_every_document_reaches_nothing(gpu, bad, G, D):
    """Rows and keys in front, behind and in documents without a partner: whatever they hold the others' results are the
    same bits, and their own are zeros."""
    qs, ks = _i32([[5, 60, 80, 150]]), _i32([[3, 70, 70, 140]])     # document 1 has queries and no keys
    x = _inputs(1, 170, 160, 2 * G, 2, D)
    clean = _run(gpu, *x, qs, ks)
    out_q = [i for i in range(170) if i < 5 or 60 <= i < 80 or i >= 150]
    out_k = [j for j in range(160) if j < 3 or j >= 140]
    q, k, v, do = (t.clone() for t in x)
    q[:, out_q], do[:, out_q], k[:, out_k], v[:, out_k] = bad, bad, bad, bad
    dirty = _run(gpu, q, k, v, do, qs, ks)
    for n, a, b in zip(NAMES, clean, dirty):
        assert torch.equal(a, b), n
    assert not dirty[0][:, out_q].any() and not dirty[1][:, out_q].any()
    assert not dirty[2][:, out_k].any() and not dirty[3][:, out_k].any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_is_not_finite_stays_in_its_document(gpu, bad, which, D):
    """A NaN or an infinity in one document, beside others in the same tiles: their gradients are the same bits.  In its own, every
    gradient whose formula is NaN everywhere is: all of a query's row that holds it (q: dq; do: dq), or of all queries (k, v)."""
    qs, ks = _i32([[0, 40, 90, 150]]), _i32([[0, 50, 110, 160]])
    x = dict(zip(("q", "k", "v", "do"), _inputs(1, 150, 160, 2, 2, D)))
    clean = _run(gpu, *x.values(), qs, ks)
    y = {n: t.clone() for n, t in x.items()}
    y[which][0, 60, 1, 3] = bad                              # document 1, head 1
    dirty = _run(gpu, *y.values(), qs, ks)
    for n, a, b in zip(NAMES, clean, dirty):
        lo, hi = (40, 90) if n in ("out", "dq") else (50, 110)
        assert torch.equal(a[:, :, 0], b[:, :, 0]), n
        assert torch.equal(a[:, :lo], b[:, :lo]) and torch.equal(a[:, hi:], b[:, hi:]), n
    dq, dk, dv = (t[0, :, 1] for t in dirty[1:])
    if which in ("q", "do"):
        assert dq[60].isnan().all() and dk[50:110].isnan().all()
        assert not (dv[50:110, 3] if which == "do" else dv[50:110]).isfinite().any()
    if which == "v":
        assert dq[40:90].isnan().all() and dk[50:110].isnan().all()
        assert dv[50:110].isfinite().all()
    if which == "k":                                         # an infinite key has weight 0 where its score is -inf
        seen = dirty[0][0, 40:90, 1].isnan().all(-1)
        assert seen.any() and dq[40:90][seen].isnan().all()


def test_a_document_of_whole_tiles_that_is_not_finite(gpu):
    """The same where no tile is seen in part."""
    q, k, v, do = _inputs(1, 256, 256, 1, 1, 128)
    do[0, 100, 0, 7] = float("nan")
    out, dq, dk, dv = _run(gpu, q, k, v, do)
    assert out.isfinite().all() and dq[0, 100].isnan().all() and dk.isnan().all() and dv[..., 7].isnan().all()
    assert dq[0, :100].isfinite().all() and dq[0, 101:].isfinite().all()


@pytest.mark.parametrize("D", [64, 128])
def test_scales_and_large_scores(gpu, D):
    q, k, v, do = _inputs(1, 100, 90, 2, 1, D)
    _check(gpu, q, k, v, do, scale=0.5)
    _check(gpu, (q * 8).to(BF), (k * 4).to(BF), v, do)        # one key carries a row
    _check(gpu, q, k, v, do, scale=1e-4)


def test_order_strides_and_alignment(gpu):
    """Layouts other than the contiguous one give the same bits: heads first, slices of a wider tensor, rows off 16 bytes, batch rows
    shared by stride 0, gradients of one value for all."""
    x = _inputs(2, 70, 90, 4, 2, 64)
    want = _run(gpu, *x)
    dev = [t.to(gpu) for t in x]

    def run(q, k, v, do):
        out, lse, rest = cross_attn_fwd_hip(q, k, v)
        return (out, *cross_attn_bwd_hip(do, q, k, v, out, lse, rest))
    heads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in dev]
    wide = [torch.full((*t.shape[:3], 100), float("nan"), dtype=BF, device=gpu) for t in dev]
    odd = []
    for w, t in zip(wide, dev):
        w[..., 3:67] = t
        odd.append(w[..., 3:67])
    for y in (heads, odd):
        for a, b in zip(want, run(*y)):
            assert torch.equal(a, b)
    q, k, v, do = dev
    same = run(q, k[:1].expand_as(k), v[:1].expand_as(v), do)
    for a, b in zip(same, run(q, k[:1].expand_as(k).contiguous(), v[:1].expand_as(v).contiguous(), do)):
        assert torch.equal(a, b)
    one = torch.ones((), dtype=BF, device=gpu).expand_as(q)
    for a, b in zip(run(q, k, v, one), run(q, k, v, one.contiguous())):
        assert torch.equal(a, b)


@pytest.mark.parametrize("far", ["q", "k"])
def test_rows_far_apart(gpu, far):
    """A tensor of over 4 GiB of which 600 rows are used: offsets past 32 bits."""
    q, k, v, do = _inputs(1, 600 if far == "q" else 70, 600 if far == "k" else 70, 1, 1, 64)
    want = _run(gpu, q, k, v, do)
    dev = dict(q=q.to(gpu), k=k.to(gpu))
    step = 1 << 22
    buf = torch.empty(599 * step + 64, dtype=BF, device=gpu)
    view = buf.as_strided((1, 600, 1, 64), (0, step, 64, 1))
    view.copy_(dev[far])
    dev[far] = view
    out, lse, rest = cross_attn_fwd_hip(dev["q"], dev["k"], v.to(gpu))
    got = (out, *cross_attn_bwd_hip(do.to(gpu), dev["q"], dev["k"], v.to(gpu), out, lse, rest))
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_same_bits_and_parts(gpu):
    """Few rows beside a long other side are split in parts; the results are the oracle's and the same bits each time."""
    for sizes in ((1, 5, 4000, 4, 2, 128), (1, 4000, 5, 4, 2, 128), (1, 700, 900, 1, 1, 64)):
        x = _inputs(*sizes)
        a, b = _check(gpu, *x), _run(gpu, *x)
        assert all(torch.equal(s, t) for s, t in zip(a, b))
        for need in ((True, False, False), (False, True, False), (False, False, True)):
            q, k, v, do = (t.to(gpu) for t in x)
            out, lse, rest = cross_attn_fwd_hip(q, k, v)
            got = cross_attn_bwd_hip(do, q, k, v, out, lse, rest, need=need)
            for want, g, n in zip(a[1:], got, need):
                assert (g is None) != n and (g is None or torch.equal(g, want))


@pytest.mark.parametrize("D", [64, 128])
def test_few_keys_and_what_the_rounding_left(gpu, D):
    """Rows of 3 to 8 keys: with the byte beside each result dq and dk are nearer to the exact ones, in the 2-norm, than from the rounded
    result alone; the byte is the difference to the exact result, to a 256th of a last place where the forward's own error is small against it
    (one key: out is v itself and nothing is left)."""
    for Sk in (3, 8):
        x = _inputs(1, 400, Sk, 2, 2, D, Sk)
        val, _ = O.cross_attention(*x)
        q, k, v, do = (t.to(gpu) for t in x)
        out, lse, rest = cross_attn_fwd_hip(q, k, v)
        err = lambda r: [((g.double().cpu() - val[n]).norm() / val[n].norm()).item()
                         for n, g in zip(("dq", "dk"), cross_attn_bwd_hip(do, q, k, v, out, lse, r)[:2])]
        for a, b in zip(err(rest), err(None)):
            assert a < b
    q, k, v, do = (t.to(gpu) for t in _inputs(1, 40, 1, 2, 2, D))
    out, lse, rest = cross_attn_fwd_hip(q, k, v)
    assert torch.equal(out, v.expand_as(out)) and (rest == 128).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,H,Hk", [(1, 3, 3), (64, 2, 2), (21, 6, 2)])
def test_few_queries_keep_the_weights(gpu, Sq, H, Hk, D):
    """Up to 128 rows of a key head take P and dS as two bf16.  What is left of their rounding is in the forward's totals and results:
    over 600 keys with scores of deviation 1.5, sqrt(sum p^2) is about sqrt(e^2.25 / 600) = 0.13, so of a half step of
    2^-8 (2^-8 / sqrt 3 of a deviation) 0.13 or 3e-4 reaches a row's total and as much its D; one bf16 would leave 1.7e-3 (2-norms)."""
    x = _inputs(1, Sq, 600, H, Hk, D, Sq)
    got = _check(gpu, *x, grad_dtype=torch.float32)
    val, _ = O.cross_attention(*x)
    for n, a in zip(NAMES[1:], got[1:]):
        assert (a.double().cpu() - val[n]).norm() < 2.0 ** -10 * val[n].norm(), n


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,H,Hk,Sk", [(128, 2, 2, 600), (128, 2, 2, 100), (42, 6, 2, 300), (700, 2, 2, 8), (700, 4, 2, 3)])
def test_a_block_of_queries_keeps_the_weights(gpu, Sq, H, Hk, Sk, D):
    """And up to 8 keys.  What the forward's rounded weights leave, row by row.  bf16 rounds a weight m 2^e by 2^-8 / (m sqrt 3) of it (deviation), over
    log-uniform m u = 2^-8 sqrt((1 - 1/4) / (2 ln 2) / 3) = 0.00166.  Its total is off by u |p| of itself, which scales the row's P (not
    in dq, which divides by its own total), and D by u |p (dP - D)|.  Rows are independent: 1.5 deviations of their sum, and
    2^-14 for the rest.  One bf16 would add u |dS| to every row."""
    x = _inputs(1, Sq, Sk, H, Hk, D, 11)
    got = _check(gpu, *x, grad_dtype=torch.float32)
    val, _ = O.cross_attention(*x)
    u, G = 2.0 ** -8 * (0.75 / (2 * 0.6931) / 3) ** 0.5, H // Hk
    q, k, v, do = (t.double()[0].transpose(0, 1) for t in x)
    k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    p = torch.softmax(D ** -0.5 * q @ k.transpose(1, 2), -1)
    dP = do @ v.transpose(1, 2)
    c = dP - (p * dP).sum(-1, keepdim=True)
    norm = lambda t: t.norm(dim=-1, keepdim=True)
    eps, delta = u * norm(p), u * norm(p * c)
    dev = dict(dq=D ** -0.5 * norm(p @ k) * delta, dk=D ** -0.5 * norm(q) * ((eps * norm(p * c)) ** 2 + (delta * norm(p)) ** 2).sqrt(),
               dv=norm(do) * eps * norm(p))
    for n, a in zip(NAMES[1:], got[1:]):
        assert (a.double().cpu() - val[n]).norm() < 1.5 * dev[n].norm() + 2.0 ** -14 * val[n].norm(), n


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G", [1, 3])
@pytest.mark.parametrize("qs,ks", [([[0, 5, 5, 19]], [[0, 80, 90, 200]]), ([[2, 7, 15]], [[3, 90, 170]]), ([[0, 21], [0, 1], [0, 0]], [[0, 77], [0, 210], [0, 210]])])
def test_documents_of_few_queries(gpu, qs, ks, G, D):
    _check(gpu, *_inputs(len(qs), 21, 210, 2 * G, 2, D, G), _i32(qs), _i32(ks))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_few_queries_and_what_is_not_finite(gpu, bad, D):
    """As with many: outside the documents it reaches nothing, inside one it stays there."""
    qs, ks = _i32([[2, 20, 40]]), _i32([[3, 70, 140]])
    x = _inputs(1, 44, 150, 2, 2, D)
    clean = _run(gpu, *x, qs, ks)
    q, k, v, do = (t.clone() for t in x)
    for t, lo, hi in ((q, 2, 40), (k, 3, 140), (v, 3, 140), (do, 2, 40)):
        t[:, :lo], t[:, hi:] = bad, bad
    assert all(torch.equal(a, b) for a, b in zip(clean, _run(gpu, q, k, v, do, qs, ks)))
    do[0, 30, 1, 5] = bad                                    # document 1, head 1
    dirty = _run(gpu, q, k, v, do, qs, ks)
    for n, a, b in zip(NAMES, clean, dirty):
        assert torch.equal(a[:, :, 0], b[:, :, 0]), n
        end = 20 if n in ("out", "dq") else 70
        assert torch.equal(a[:, :end], b[:, :end]), n
    assert dirty[1][0, 30, 1].isnan().all() and dirty[2][0, 70:140, 1].isnan().all() and not dirty[3][0, 70:140, 1, 5].isfinite().any()


def test_where_the_rounding_is_kept(gpu):
    """By keys, documents, or where the queries are few; the node keeps the same: a hook sees it or not."""
    def kept(Sq, Sk, H, Hk, docs=0, D=128):
        q, k, v, _ = (t.to(gpu) for t in _inputs(1, Sq, Sk, H, Hk, D))
        st = [None, None] if not docs else [torch.linspace(0, n, docs + 1).int()[None].to(gpu) for n in (Sq, Sk)]
        pair = cross_attn_fwd_hip(q, k, v, *st)[2] is not None
        seen = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t.dtype) or t, lambda t: t):
            cross_attn_func(q.requires_grad_(True), k, v, q_starts=st[0], k_starts=st[1])
        assert (torch.uint8 in seen) == pair
        return pair
    assert [kept(*x) for x in ((129, 256, 2, 2), (129, 257, 2, 2), (128, 257, 2, 2), (65, 257, 4, 2), (100, 512, 2, 1, 1), (100, 513, 2, 1, 2),
                                   (129, 1024, 2, 2, 0, 64), (129, 1025, 2, 2, 0, 64))] == \
        [True, False, True, False, True, True, True, False]


def test_autograd(gpu):
    """Shared key heads, a key tensor broadcast over the batch (its gradient is the sum), a query that needs none, and the
    forward's value, which is masked_attn_func's."""
    q, k, v, do = (t.to(gpu) for t in _inputs(3, 60, 80, 4, 2, 64))
    qs = torch.tensor([[0, 60]] * 3, dtype=torch.int32, device=gpu)
    ks = torch.tensor([[0, 80], [0, 33], [0, 0]], dtype=torch.int32, device=gpu)
    k1 = k[:1].clone().requires_grad_()
    vv = v.clone().requires_grad_()
    out = cross_attn_func(q, k1.expand(3, -1, -1, -1), vv, q_starts=qs, k_starts=ks)
    with torch.no_grad():
        assert torch.equal(out, masked_attn_func(q, k1.expand(3, -1, -1, -1), v, q_starts=qs, k_starts=ks))
        plain = cross_attn_func(q, k1.expand(3, -1, -1, -1), vv, q_starts=qs, k_starts=ks)
    assert torch.equal(plain, out) and plain.grad_fn is None
    dk, dv = torch.autograd.grad(out, (k1, vv), do)
    o, lse, rest = cross_attn_fwd_hip(q, k1.expand(3, -1, -1, -1), v, qs, ks)
    _, wk, wv = cross_attn_bwd_hip(do, q, k1.expand(3, -1, -1, -1), v, o, lse, rest, qs, ks)
    assert torch.equal(dv, wv) and torch.equal(dk, wk.sum(0, keepdim=True))
    with pytest.raises(RuntimeError):
        x = q.clone().requires_grad_()
        g, = torch.autograd.grad(cross_attn_func(x, k, v), x, do, create_graph=True)
        g.sum().backward()


def test_refusals(gpu):
    q, k, v, do = (t.to(gpu) for t in _inputs(2, 6, 8, 4, 2, 64))
    s = torch.zeros(2, 2, dtype=torch.int32, device=gpu)
    out, lse, rest = cross_attn_fwd_hip(q, k, v)
    for call in (lambda: cross_attn_func(q.float(), k, v), lambda: cross_attn_func(q, k, v[:, :4]), lambda: cross_attn_func(q[:1], k, v),
                 lambda: cross_attn_func(q[..., :32], k[..., :32], v[..., :32]), lambda: cross_attn_func(q[:, :, :3], k, v),
                 lambda: cross_attn_func(q, k, v, q_starts=s), lambda: cross_attn_func(q, k, v, q_starts=s, k_starts=s[:1]),
                 lambda: cross_attn_func(q, k, v, q_starts=s.long(), k_starts=s.long()),
                 lambda: cross_attn_func(q, k, v, q_starts=s.cpu(), k_starts=s.cpu()), lambda: cross_attn_func(q, k, v, softmax_scale=-1.0),
                 lambda: cross_attn_func(q, k, v, softmax_scale=1e-30),
                 lambda: cross_attn_func(q, k.cpu(), v.cpu()), lambda: cross_attn_bwd_hip(do[:, :3], q, k, v, out, lse, rest),
                 lambda: cross_attn_bwd_hip(do.float(), q, k, v, out, lse, rest), lambda: cross_attn_bwd_hip(do, q, k, v, out, lse[:, :1], rest),
                 lambda: cross_attn_bwd_hip(do, q, k, v, out, lse, rest[:, :3]), lambda: cross_attn_bwd_hip(do, q, k, v, out, lse, rest.char()),
                 lambda: cross_attn_bwd_hip(do, q, k, v, out, lse.cpu(), rest), lambda: cross_attn_bwd_hip(do, q, k, v, out, lse, rest.cpu()),
                 lambda: cross_attn_bwd_hip(do, q, k, v, out, lse, rest, grad_dtype=torch.float16)):
        with pytest.raises(IcsaArgumentError):
            call()
