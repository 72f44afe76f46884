"""Attention under masks on the GPU against float64 (oracle.masked_attn, whose bound counts f32
scores and P rounded to bf16; the output's rounding, eps / 2 of the value, is added here)."""
import math

import pytest
import torch

from icsa_hip import flash_attn_func, masked_attn_func
from oracle import masked_attn as O

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _inputs(B, Sq, Sk, H, Hk, D, seed=0, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    return ((spread * torch.randn(B, Sq, H, D, generator=g)).to(BF), torch.randn(B, Sk, Hk, D, generator=g).to(BF),
            torch.randn(B, Sk, Hk, D, generator=g).to(BF))


def _i32(x):
    return torch.tensor(x, dtype=torch.int32)


def _check(gpu, q, k, v, out_dtype=BF, **kw):
    scale = kw.pop("softmax_scale", None)
    ref, bound = O.attention(q, k, v, scale=scale, **kw)
    dev = {n: x.to(gpu) if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    out = masked_attn_func(q.to(gpu), k.to(gpu), v.to(gpu), softmax_scale=scale, out_dtype=out_dtype, **dev)
    assert out.shape == q.shape and out.dtype == out_dtype
    got = out.double().cpu()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fine), "not finite in other places than it should be"
    tol = bound + (2.0 ** -8 if out_dtype == BF else 2.0 ** -22) * ref.abs()
    d = torch.where(fine, (got - ref).abs(), 0.0)
    tol = torch.where(fine, tol, 1.0)
    assert (d <= tol).all(), f"{(d / tol).max().item():.2f} of the tolerance, {d.max().item():.3e}"
    return got


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,Sq,Sk,H,Hk", [(1, 1, 1, 1, 1), (1, 1, 65, 3, 3), (2, 31, 64, 2, 2), (1, 33, 63, 4, 2), (1, 128, 128, 2, 1),
                                          (1, 129, 257, 2, 2), (3, 7, 130, 10, 2), (1, 200, 77, 5, 5), (1, 1, 5000, 8, 2),
                                          (1, 3, 3001, 5, 1), (1, 0, 10, 1, 1), (1, 10, 0, 2, 2)])
def test_no_mask(gpu, B, Sq, Sk, H, Hk, D):
    print(f"[masked] plain B={B} Sq={Sq} Sk={Sk} H={H}/{Hk} D={D}", flush=True)
    _check(gpu, *_inputs(B, Sq, Sk, H, Hk, D, Sq + Sk), out_dtype=BF if Sq % 2 else torch.float32)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,Sk,prefix", [(1, 1, None), (64, 64, None), (65, 65, None), (130, 200, None), (200, 130, None),
                                          (1, 700, None), (3, 700, None), (300, 300, 100), (300, 300, 299), (300, 300, 1000),
                                          (300, 200, 64), (257, 257, -5), (100, 40, 0)])
def test_causal_and_prefix(gpu, Sq, Sk, prefix, D):
    print(f"[masked] causal Sq={Sq} Sk={Sk} prefix={prefix} D={D}", flush=True)
    kw = {} if prefix is None else dict(prefix=_i32([[prefix], [prefix // 2]]))
    _check(gpu, *_inputs(2, Sq, Sk, 4, 2, D, Sq), causal=True, **kw)


DOCS = [
    # query starts, key starts: aligned and ragged documents, empty ones, gaps in front and behind
    ([[0, 64, 128]], [[0, 64, 128]]),
    ([[0, 50, 50, 190]], [[0, 80, 90, 200]]),
    ([[0, 50, 100, 190]], [[0, 80, 80, 200]]),
    ([[7, 20, 150]], [[3, 90, 170]]),
    ([[0, 10, 20, 30, 40, 50, 200]], [[0, 5, 15, 40, 41, 130, 210]]),
    ([[0, 200], [0, 1], [0, 0], [100, 100]], [[0, 77], [0, 210], [0, 210], [3, 50]]),
    ([[0, 100, 250]], [[0, 100, 400]]),                      # past both lengths: clamped
]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mask", ["none", "causal", "prefix"])
@pytest.mark.parametrize("case", range(len(DOCS)))
def test_documents(gpu, case, mask, D):
    qs, ks = map(_i32, DOCS[case])
    print(f"[masked] documents {case} {mask} D={D}", flush=True)
    B = qs.shape[0]
    kw = dict(q_starts=qs, k_starts=ks, causal=mask != "none")
    if mask == "prefix":
        kw["prefix"] = _i32([[11 * n + 5 for n in range(qs.shape[1] - 1)]] * B)
    if case == 6:
        # the oracle takes the clamped borders: the last document ends at the last query and key
        ref, bound = O.attention(*_inputs(B, 200, 210, 2, 1, D, case),
                                 **{**kw, "q_starts": qs.clamp(max=200), "k_starts": ks.clamp(max=210)})
        out = masked_attn_func(*(t.to(gpu) for t in _inputs(B, 200, 210, 2, 1, D, case)),
                               **{n: x.to(gpu) if isinstance(x, torch.Tensor) else x for n, x in kw.items()})
        assert ((out.double().cpu() - ref).abs() <= bound + 2.0 ** -8 * ref.abs()).all()
        return
    _check(gpu, *_inputs(B, 200, 210, 2, 1, D, case), **kw)


@pytest.mark.parametrize("n", [62, 63, 64, 65, 150])
def test_many_documents(gpu, n):
    """Around the number of documents whose borders fit a wave's lanes, one query to several each, some empty."""
    print(f"[masked] {n} documents", flush=True)
    g = torch.Generator().manual_seed(n)
    qs = torch.sort(torch.randint(0, 201, (2, n + 1), generator=g), 1).values.to(torch.int32)
    ks = torch.sort(torch.randint(0, 301, (2, n + 1), generator=g), 1).values.to(torch.int32)
    kw = dict(q_starts=qs, k_starts=ks)
    _check(gpu, *_inputs(2, 200, 300, 2, 1, 64, n), **kw)
    _check(gpu, *_inputs(2, 200, 300, 2, 1, 64, n), causal=True, prefix=torch.full((2, n), 2, dtype=torch.int32), **kw)


def test_starts_that_decrease_stay_inside(gpu):
    """Borders in no order: no promise on the values, but nothing outside the tensors is read and what is written is finite."""
    q, k, v = _inputs(1, 300, 300, 2, 2, 64, 1)
    g = torch.Generator().manual_seed(2)
    for n in (5, 80):
        st = torch.randint(-1000, 1000, (2, 1, n + 1), generator=g, dtype=torch.int32)
        out = masked_attn_func(q.to(gpu), k.to(gpu), v.to(gpu), q_starts=st[0].to(gpu), k_starts=st[1].to(gpu), causal=True)
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("softcap", [0.0, 4.0])
def test_softmax_scale(gpu, softcap):
    q, k, v = _inputs(1, 90, 130, 2, 2, 128, 12)
    for scale in (1e-4, 0.3):
        _check(gpu, q, k, v, softmax_scale=scale, softcap=softcap)
    with pytest.raises(ValueError):
        masked_attn_func(q.to(gpu), k.to(gpu), v.to(gpu), softmax_scale=-1.0)


def test_bias_not_a_number(gpu):
    """A NaN of the table reaches the rows that see a key at its distance."""
    q, k, v = _inputs(1, 40, 40, 2, 2, 64, 13)
    bias = torch.zeros(2, 9)
    bias[1, 6] = math.nan                                    # two keys ahead, head 1
    out = masked_attn_func(q.to(gpu), k.to(gpu), v.to(gpu), bias=bias.to(gpu)).cpu()
    assert torch.isfinite(out[:, :, 0]).all()
    assert torch.isnan(out[0, :38, 1]).all() and torch.isfinite(out[0, 38:, 1]).all()


def test_last_round_in_parts(gpu):
    """Alike items that leave the last round of workgroups short: its items' keys in parts.  Against the dense kernel, both
    within (2^-8 of P + 2^-8 of the output + the scores' few 2^-20) max |v|."""
    for H, S, D in ((9, 8300, 128), (12, 6200, 128)):
        q, k, v = (torch.randn(1, S, H, D, device=gpu).to(BF) for _ in range(3))
        out, ref = masked_attn_func(q, k, v), flash_attn_func(q, k, v)
        top = v.abs().max().item()
        assert (out.float() - ref.float()).abs().max().item() <= 2.0 ** -6 * 1.05 * top
        assert torch.equal(out, masked_attn_func(q, k, v))


@pytest.mark.parametrize("D,R,cap,H,Hk", [(64, 0, 0.0, 3, 3), (64, 16, 0.0, 4, 2), (128, 128, 0.0, 2, 2), (128, 5, 30.0, 2, 1),
                                          (64, 300, 10.0, 2, 2), (128, 0, 5.0, 4, 4), (64, 128, 0.0, 8, 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_cap_and_bias(gpu, D, R, cap, H, Hk, causal):
    print(f"[masked] cap={cap} R={R} D={D} causal={causal}", flush=True)
    bias = torch.randn(H, 2 * R + 1, generator=torch.Generator().manual_seed(R)) if R or not cap else None
    _check(gpu, *_inputs(2, 150, 420, H, Hk, D, R, 4.0), causal=causal, softcap=cap, bias=bias)


def test_bias_extremes(gpu):
    """-inf hides a distance; the type's lowest value hides it where another key is seen and is a plain
    shift where every key has it; a row all of whose keys are hidden gets zeros."""
    q, k, v = _inputs(1, 70, 70, 2, 2, 64, 3)
    for value in (-math.inf, torch.finfo(torch.float32).min):
        bias = torch.zeros(2, 9)
        bias[0, :4], bias[1, 5:] = value, value
        print(f"[masked] bias {value}", flush=True)
        _check(gpu, q, k, v, bias=bias)
    out = masked_attn_func(q.to(gpu), k.to(gpu), v.to(gpu), bias=torch.full((2, 9), -math.inf, device=gpu))
    assert (out == 0).all()
    # equal shifts: f32 keeps none of the score beside the lowest value, so the weights are equal
    out = masked_attn_func(q.to(gpu), k.to(gpu), v.to(gpu),
                           bias=torch.full((2, 9), torch.finfo(torch.float32).min, device=gpu))
    mean = v.double().mean(1, keepdim=True)
    assert ((out.double().cpu() - mean).abs() <= 2.0 ** -7 * v.double().abs().mean(1, keepdim=True) + 2.0 ** -8 * mean.abs()).all()


@pytest.mark.parametrize("spread", [0.0, 40.0, 300.0])
def test_large_scores(gpu, spread):
    """Uniform rows, and rows whose maximum rises by hundreds between tiles (the reference maximum is
    raised in the middle)."""
    q, k, v = _inputs(1, 100, 600, 2, 2, 128, 8, spread)
    k[:, 300:] *= 4
    _check(gpu, q, k, v)
    _check(gpu, q, k, v, causal=True)


@pytest.mark.parametrize("D", [64, 128])
def test_not_finite_in_masked_places(gpu, D):
    """NaN and infinities in keys and values of another document, behind the last one, ahead of a
    causal row, and in the queries of other rows reach only the rows that see them."""
    q, k, v = _inputs(1, 150, 230, 2, 1, D, 4)
    qs, ks = _i32([[0, 40, 100]]), _i32([[0, 70, 200]])
    k[0, 75], v[0, 80, 0, 3], v[0, 90, 0, 5], v[0, 100] = math.nan, math.nan, -math.inf, math.inf
    k[0, 210:], v[0, 205:] = math.nan, math.inf
    q[0, 120:] = math.nan                                    # behind the last document
    print(f"[masked] not finite D={D}", flush=True)
    dev = dict(q_starts=qs.to(gpu), k_starts=ks.to(gpu))
    out = masked_attn_func(q.to(gpu), k.to(gpu), v.to(gpu), **dev).cpu()
    clean = [t.clone() for t in (q, k, v)]
    for t in clean:
        t[~torch.isfinite(t)] = 0
    ref, bound = O.attention(*clean, q_starts=qs, k_starts=ks)
    d = (out.double() - ref).abs()
    assert (d[:, :40] <= (bound + 2.0 ** -8 * ref.abs())[:, :40]).all()      # the first document is clean
    assert torch.isnan(out[:, 40:100]).all()                                 # the second has a NaN key
    assert (out[:, 100:] == 0).all()
    # values alone: a NaN or an infinity in some dims, causal, so that earlier rows do not see it
    q, k, v = _inputs(1, 200, 200, 2, 2, D, 5)
    v[0, 77, 0, 3], v[0, 130, 1, 7], v[0, 131, 1, 8] = math.nan, math.inf, -math.inf
    _check(gpu, q, k, v, causal=True)
    _check(gpu, q, k, v, causal=True, prefix=_i32([[78]]))


@pytest.mark.parametrize("causal", [False, True])
def test_keys_split_over_workgroups(gpu, causal):
    """Few rows and many keys: the parts joined; rows whose document ends before the later parts begin."""
    for Sq, H, Hk, D in ((1, 40, 8, 128), (4, 6, 2, 64), (130, 2, 2, 128)):
        print(f"[masked] split Sq={Sq} H={H}/{Hk} D={D}", flush=True)
        q, k, v = _inputs(1, Sq, 4133, H, Hk, D, Sq)
        _check(gpu, q, k, v, causal=causal)
        if Sq > 1:
            _check(gpu, q, k, v, causal=causal, q_starts=_i32([[0, 1, 2, Sq]]), k_starts=_i32([[0, 40, 2000, 4000]]))


def test_strides(gpu):
    """Views: heads in front, a fused qkv tensor, rows a multiple of 16 bytes apart, an odd base."""
    g = torch.Generator().manual_seed(9)
    qkv = torch.randn(2, 90, 3, 4, 64, generator=g).to(BF)
    for q, k, v in ((qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2]), (qkv[:, 5:70, 0], qkv[:, 1:, 1, :2], qkv[:, 1:, 2, :2])):
        ref, bound = O.attention(q, k, v, causal=True)
        dq = qkv.to(gpu)
        dq, dk, dv = ((dq[:, :, 0], dq[:, :, 1], dq[:, :, 2]) if q.shape[1] == 90 else
                      (dq[:, 5:70, 0], dq[:, 1:, 1, :2], dq[:, 1:, 2, :2]))
        out = masked_attn_func(dq, dk, dv, causal=True)
        assert ((out.double().cpu() - ref).abs() <= bound + 2.0 ** -8 * ref.abs()).all()
        hd = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (dq, dk, dv)]
        assert torch.equal(masked_attn_func(*hd, causal=True), out)
        odd = [torch.empty(t.numel() + 1, dtype=BF, device=gpu)[1:].view(t.shape).copy_(t) for t in (dq, dk, dv)]
        assert torch.equal(masked_attn_func(*odd, causal=True), out)


def test_same_as_dense_attention(gpu):
    """Without masks it computes what flash_attn_func does (both within the bound of float64)."""
    q, k, v = _inputs(1, 300, 500, 2, 2, 128, 10)
    ref, bound = O.attention(q, k, v)
    for fn in (flash_attn_func, masked_attn_func):
        out = fn(q.to(gpu), k.to(gpu), v.to(gpu)).double().cpu()
        assert ((out - ref).abs() <= bound + 2.0 ** -8 * ref.abs()).all()


@pytest.mark.parametrize("cap", [1e-3, 4096.0])
def test_smallest_and_largest_caps(gpu, cap):
    """The bound counts a few roundings of numbers of the cap's size."""
    q, k, v = _inputs(1, 70, 200, 2, 1, 64, 21, 3.0)
    _check(gpu, q, k, v, causal=True, softcap=cap)
    _check(gpu, q, k, v, softcap=cap, bias=torch.randn(2, 9))


@pytest.mark.parametrize("D", [64, 128])
def test_rows_far_apart(gpu, D):
    """Rows 512 KB apart, 4.7 GB a tensor: what lies behind 32-bit offsets equals the same rows side by side."""
    big = torch.zeros(1, 9001, 1 << 18, dtype=BF, device=gpu)
    views = [big[:, :, 1000 * i:1000 * i + 2 * D].unflatten(2, (2, D)) for i in range(3)]
    for x in views:
        x.normal_()
    q, k, v = views
    near = [x.contiguous() for x in views]
    for kw in (dict(causal=True), dict(softcap=20.0)):
        assert torch.equal(masked_attn_func(q, k, v, **kw), masked_attn_func(*near, **kw))
    assert torch.equal(masked_attn_func(q[:, -1:], k, v), masked_attn_func(near[0][:, -1:], *near[1:]))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,Sk,kw", [(300, 300, {}), (40, 5000, {}), (200, 330, dict(softcap=5.0)),
                                      (150, 400, dict(q_starts=[[0, 70, 150]], k_starts=[[0, 33, 400]]))])
def test_infinities_of_values_keep_their_sign(gpu, Sq, Sk, kw, D):
    """Infinite and NaN values near the causal border (in tiles that some rows see in part, several of them a
    tile, whole items and parts): the queries that see one get it, of its sign, NaN for both signs; all others
    what they get without."""
    print(f"[masked] inf {Sq}x{Sk} {kw} D={D}", flush=True)
    q, k, v = _inputs(1, Sq, Sk, 2, 1, D, 31)
    bad = {Sk - 100: (3, math.inf), Sk - 61: (D - 1, -math.inf), Sk - 60: (3, -math.inf), Sk - 2: (17, math.nan), Sk - 40: (40, math.inf)}
    vb = v.clone()
    for key, (d, x) in bad.items():
        vb[0, key, 0, d] = x
    kw = {n: _i32(x) if isinstance(x, list) else x for n, x in kw.items()}
    dev = {n: x.to(gpu) if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    got = masked_attn_func(q.to(gpu), k.to(gpu), vb.to(gpu), causal=True, **dev).double().cpu()
    clean = v.clone()
    for key, (d, _) in bad.items():
        clean[0, key, 0, d] = 0
    plain = masked_attn_func(q.to(gpu), k.to(gpu), clean.to(gpu), causal=True, **dev).double().cpu()
    see, _ = O.visible(1, Sq, Sk, kw.get("q_starts"), kw.get("k_starts"), True)
    want = plain.clone()
    for key, (d, x) in bad.items():
        want[0, see[0, :, key], :, d] += x
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got, nan=0.0, posinf=1e30, neginf=-1e30), torch.nan_to_num(want, nan=0.0, posinf=1e30, neginf=-1e30))
