"""What a training step of the block needs around its sparse attention, as callers have it done: cross
attention to text of another length, layer norm and RMS norm with their parameters' gradients, and
rotary positions, each forward and backward.

Sizes follow the repository's own configurations: dim 5120 (40 heads of 128), 512 text tokens, 1,560
tokens per latent frame, 65,520 tokens for 21 frames of target and source, dim 1536 (12 heads), and odd
lengths around them.

`own` false: the plain form, elementary torch operations in 32 bits.  `own` true: the calls that a
user makes of icsa_hip.
"""
import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.getcwd(), "lightning-unified-video-editor-via-in-context-sparse-attention_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

DEV = "cuda"
BF = torch.bfloat16
EPS = 1e-6
GRID = (30, 52)            # rows and columns of a latent frame after the patch embedding: 1,560 tokens


# ------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------
def listed():
    return [
        # cross attention, forward and backward: a thumbnail's 64 tokens over a short prompt (latency)
        dict(name="attn_thumbnail", kind="attn", B=1, H=12, Hk=12, D=128, Sq=64, Sk=77, docs=0),
        # image editing: target and source of one frame, the prompt padded to 512 tokens
        dict(name="attn_image", kind="attn", B=1, H=40, Hk=40, D=128, Sq=3120, Sk=512, docs=0),
        # a batch of two odd-length clips, heads of 64 that share key heads, prompts of different lengths
        dict(name="attn_grouped", kind="attn", B=2, H=24, Hk=8, D=64, Sq=9373, Sk=1009, docs=1),
        # four packed clips, each with its own prompt
        dict(name="attn_packed", kind="attn", B=1, H=40, Hk=40, D=128, Sq=32760, Sk=1400, docs=4),
        # the full 21 frames of target and source over the padded prompt: the block's own cross attention
        dict(name="attn_21frames", kind="attn", B=1, H=40, Hk=40, D=128, Sq=65520, Sk=512, docs=0),
        # layer norm of the modulation's few rows (latency)
        dict(name="ln_few_rows", kind="norm", rms=False, mode="affine", B=1, S=6, dim=5120, x="f32", y="f32"),
        # norm1 / norm2 of two 9-frame clips: scale and shift of each clip's time embedding
        dict(name="ln_modulate_9frames", kind="norm", rms=False, mode="modulate", B=2, S=14040, dim=5120, x="bf16", y="bf16"),
        # norm3 of the f32 residual stream at the full length
        dict(name="ln_affine_21frames", kind="norm", rms=False, mode="affine", B=1, S=65520, dim=5120, x="f32", y="bf16"),
        # q norm of an odd-length clip, dim 1536
        dict(name="rms_odd", kind="norm", rms=True, mode="affine", B=1, S=9373, dim=1536, x="bf16", y="bf16"),
        # q norm of two 9-frame clips
        dict(name="rms_9frames", kind="norm", rms=True, mode="affine", B=2, S=14040, dim=5120, x="bf16", y="bf16"),
        # new tokens of eight requests far into a long context, half layout, half of the head (a serving step)
        dict(name="rotary_tokens", kind="rotary", B=8, S=1, H=40, Hk=8, D=128, R=64, layout="half", axes=1, x="bf16",
             rows=131072, grad=False),
        # q and k of the full 21 frames: frame, row and column positions
        dict(name="rotary_21frames", kind="rotary", B=1, S=65520, H=40, Hk=40, D=128, R=128, layout="interleaved", axes=3,
             x="bf16", rows=1024, grad=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "norm", "norm", "rotary", "rotary"])
    if kind == "attn":
        D = rng.choice([64, 128, 128])
        Hk = rng.choice([1, 2, 3, 5, 8, 12, 40])
        H = Hk * (rng.choice([1, 1, 1, 2, 3, 5]) if Hk <= 12 else 1)
        B = rng.choice([1, 1, 2, 3])
        Sk = rng.choice([77, 226, 512, _log(rng, 1, 4096)])
        Sq = rng.choice([1, _log(rng, 1, 65520), _log(rng, 64, 65520), 1560 * rng.randint(1, 42)])
        Sq = max(1, min(Sq, 1300000000 // (B * H * Sk)))
        docs = rng.choice([0, 0, 1, 2, 5]) if Sq >= 64 and Sk >= 64 else rng.choice([0, 0, 1])
        return dict(kind=kind, B=B, H=H, Hk=Hk, D=D, Sq=Sq, Sk=Sk, docs=docs)
    if kind == "norm":
        dim = rng.choice([5120, 1536, 128, _log(rng, 16, 8192), 8 * _log(rng, 8, 1024)])
        rows = min(_log(rng, 1, 131040), 300000000 // dim)
        B = rng.choice([1, 2, 3])
        rms = rng.choice([False, False, True])
        return dict(kind=kind, rms=rms, mode="affine" if rms else rng.choice(["affine", "modulate"]), B=B,
                    S=max(1, rows // B), dim=dim, x=rng.choice(["bf16", "bf16", "f32"]), y=rng.choice(["bf16", "bf16", "f32"]))
    D = rng.choice([64, 128, 128, 80])
    Hk = rng.choice([1, 2, 5, 8, 12])
    H = rng.choice([40, Hk, 5 * Hk])
    axes = rng.choice([1, 1, 3])
    R = D if axes == 3 else rng.choice([D, D, D // 2, D - 16, D // 4])
    B = rng.choice([1, 2, 5])
    S = rng.choice([1, _log(rng, 1, 65520), _log(rng, 64, 65520)])
    S = max(1, min(S, 400000000 // (B * (H + Hk) * D)))
    return dict(kind=kind, B=B, S=S, H=H, Hk=Hk, D=D, R=R, layout=rng.choice(["interleaved", "half"]), axes=axes,
                x=rng.choice(["bf16", "bf16", "f32"]), rows=1024 if axes == 3 else rng.choice([4096, 32768, 131072]),
                grad=S > 1)


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + 31)
    return g


def _n(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _dt(name):
    return torch.float32 if name == "f32" else BF


def _leaf(t):
    return t.requires_grad_(True)


def _borders(case):
    """Document borders of each batch row, queries and keys, [B][docs + 1] each.  One document: all queries over
    the row's real text tokens.  Several: clips of different lengths, each over its own prompt; the last ones
    end before the padded sequences do."""
    rng = random.Random(case["Sq"] * 7907 + case["Sk"] * 37 + case["docs"])
    qs, ks = [], []
    for _ in range(case["B"]):
        n, Sq, Sk = case["docs"], case["Sq"], case["Sk"]
        if n == 1:
            qs.append([0, Sq])
            ks.append([0, max(1, int(Sk * rng.uniform(0.1, 1.0)))])
            continue
        cut = sorted(rng.uniform(0, 0.95) for _ in range(n - 1)) + [rng.uniform(0.95, 1.0)]
        qs.append([0] + [int(c * Sq) for c in cut])
        kcut = sorted((i + 1) / n * rng.uniform(0.9, 1.0) for i in range(n))
        ks.append([0] + [int(c * Sk) for c in kcut])
    return qs, ks


def _sections(case):
    """Pairs of each axis: frames, rows, columns as the model cuts a head's."""
    if case["axes"] == 1:
        return (case["R"] // 2,)
    third = case["D"] // 6
    return (case["D"] // 2 - 2 * third, third, third)


def _table(case):
    """cos and sin, f32 [rows, R / 2], from angles in 64 bits.  One axis with many rows: positions scaled for a context
    eight times the trained one (all frequencies but the fastest are lowered, by a larger base)."""
    cols = []
    for pairs in _sections(case):
        r = 2 * pairs
        base = 10000.0
        if case["axes"] == 1 and case["rows"] > 8192 and r > 2:
            base *= 8.0 ** (r / (r - 2))
        inv = base ** (-torch.arange(0, r, 2, dtype=torch.float64, device=DEV) / r)
        cols.append(torch.outer(torch.arange(case["rows"], dtype=torch.float64, device=DEV), inv))
    ang = torch.cat(cols, 1)
    return torch.cos(ang).float(), torch.sin(ang).float()


def _positions(case):
    """int32 [B, S] (one axis) or [B, S, 3]."""
    B, S = case["B"], case["S"]
    rng = random.Random(S * 7907 + B)
    i = torch.arange(S, device=DEV)
    if case["axes"] == 1:                                      # each row somewhere into its context
        starts = [rng.randint(0, max(0, case["rows"] - S)) for _ in range(B)]
        return torch.stack([(i + s).clamp(max=case["rows"] - 1) for s in starts]).int()
    per = GRID[0] * GRID[1]
    half = -(-S // 2)                                          # target, then source, each from position 0 on
    j = i % half
    pos = torch.stack([j // per, j // GRID[1] % GRID[0], j % GRID[1]], -1)
    return pos.int().expand(B, S, 3).contiguous()


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    st = {"case": case}
    if kind == "attn":
        B, H, Hk, D, Sq, Sk = (case[n] for n in ("B", "H", "Hk", "D", "Sq", "Sk"))
        st["q"] = _leaf((1.5 * _n(g, B, Sq, H, D)).to(BF))
        st["k"] = _leaf(_n(g, B, Sk, Hk, D).to(BF))
        st["v"] = _leaf(_n(g, B, Sk, Hk, D).to(BF))
        st["do"] = _n(g, B, Sq, H, D).to(BF)
        if case["docs"]:
            qs, ks = _borders(case)
            st["q_starts"] = torch.tensor(qs, dtype=torch.int32, device=DEV)
            st["k_starts"] = torch.tensor(ks, dtype=torch.int32, device=DEV)
    elif kind == "norm":
        B, S, dim = case["B"], case["S"], case["dim"]
        # rows with a mean of their own, some channels several times larger
        st["x"] = _leaf(((_n(g, B, S, dim) + 0.5 * _n(g, B, S, 1)) * torch.exp(0.5 * _n(g, dim))).to(_dt(case["x"])))
        if case["mode"] == "affine":
            st["w"] = _leaf(1.0 + 0.2 * _n(g, dim))
            if not case["rms"]:
                st["b"] = _leaf(0.1 * _n(g, dim))
        else:
            st["scale"] = _leaf(0.3 * _n(g, B, 1, dim))
            st["shift"] = _leaf(0.3 * _n(g, B, 1, dim))
        st["dy"] = _n(g, B, S, dim).to(_dt(case["y"]))
    else:
        B, S, H, Hk, D = (case[n] for n in ("B", "S", "H", "Hk", "D"))
        st["q"], st["k"] = (_leaf(_n(g, B, S, h, D).to(_dt(case["x"]))) for h in (H, Hk))
        if case["grad"]:
            st["dq"], st["dk"] = (_n(g, B, S, h, D).to(_dt(case["x"])) for h in (H, Hk))
        st["cos"], st["sin"] = _table(case)
        st["pos"] = _positions(case)
    return st


# ------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------
def _visible(case, st):
    """[B, 1, Sq, Sk] truth values."""
    dev = st["q"].device
    i, j = torch.arange(case["Sq"], device=dev), torch.arange(case["Sk"], device=dev)
    qs, ks = st["q_starts"].long(), st["k_starts"].long()
    n = qs.shape[1] - 1
    qd = (i[None, :, None] >= qs[:, None, :]).sum(-1) - 1          # n behind the last document
    kd = (j[None, :, None] >= ks[:, None, :]).sum(-1) - 1
    return ((qd[:, :, None] == kd[:, None, :]) & (qd < n)[:, :, None])[:, None]


def _attention(case, st):
    """out, dq, dk, dv."""
    G, scale = case["H"] // case["Hk"], case["D"] ** -0.5
    q, do = (st[n].float().transpose(1, 2).contiguous() for n in ("q", "do"))
    k, v = (st[n].float().transpose(1, 2).repeat_interleave(G, 1).contiguous() for n in ("k", "v"))
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    if case["docs"]:
        s = s.masked_fill(~_visible(case, st), -math.inf)
        m = s.amax(-1, keepdim=True)
        s = s - torch.where(torch.isfinite(m), m, torch.zeros_like(m))
    else:
        s = s - s.amax(-1, keepdim=True)
    p = torch.exp(s)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p, v)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    dk, dv = (t.unflatten(1, (case["Hk"], G)).sum(2) for t in (dk, dv))
    return tuple(t.transpose(1, 2).to(BF) for t in (o, dq, dk, dv))


def _norm(case, st):
    """y, dx and the parameters' gradients."""
    x, dy = st["x"].float(), st["dy"].float()
    mean = 0.0 if case["rms"] else x.mean(-1, keepdim=True)
    xc = x - mean
    r = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xh = xc * r
    a = st["w"] if case["mode"] == "affine" else 1.0 + st["scale"]
    y = xh * a
    u = dy * a
    du = u - xh * (u * xh).mean(-1, keepdim=True)
    if not case["rms"]:
        du = du - u.mean(-1, keepdim=True)
    over = (0, 1) if case["mode"] == "affine" else (1,)
    keep = case["mode"] != "affine"
    res = [y, (du * r).to(st["x"].dtype), (dy * xh).sum(over, keepdim=keep)]
    if not case["rms"]:
        res[0] = y + (st["b"] if case["mode"] == "affine" else st["shift"])
        res.append(dy.sum(over, keepdim=keep))
    res[0] = res[0].to(st["dy"].dtype)
    return tuple(res)


def _rotate(case, st, x, back):
    """x [B, S, H, D] turned by the positions' angles, or back (the transposed matrix)."""
    parts, at = [], 0
    pos = st["pos"].long().unsqueeze(-1) if case["axes"] == 1 else st["pos"].long()
    for a, pairs in enumerate(_sections(case)):
        parts.append([t[:, at:at + pairs][pos[..., a]] for t in (st["cos"], st["sin"])])
        at += pairs
    c, s = (torch.cat(t, -1).unsqueeze(2) for t in zip(*parts))
    if back:
        s = -s
    R, y = case["R"], x.float()
    if case["layout"] == "interleaved":
        x0, x1 = y[..., 0:R:2], y[..., 1:R:2]
        turned = torch.stack([x0 * c - x1 * s, x0 * s + x1 * c], -1).flatten(-2)
    else:
        x0, x1 = y[..., :R // 2], y[..., R // 2:R]
        turned = torch.cat([x0 * c - x1 * s, x0 * s + x1 * c], -1)
    return torch.cat([turned, y[..., R:]], -1).to(x.dtype)


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        return _run_own(case, kind, st)
    with torch.no_grad():
        if kind == "attn":
            return _attention(case, st)
        if kind == "norm":
            return _norm(case, st)
        res = [_rotate(case, st, st[n], False) for n in ("q", "k")]
        if case["grad"]:
            res += [_rotate(case, st, st[n], True) for n in ("dq", "dk")]
        return tuple(res)


def _run_own(case, kind, st):
    from icsa_hip import cross_attn_func, layer_norm_func, rms_norm_func, rotary_func
    if kind == "rotary" and not case["grad"]:
        with torch.no_grad():
            return rotary_func(st["q"], st["k"], st["cos"], st["sin"], st["pos"], interleaved=case["layout"] == "interleaved",
                               sections=_sections(case) if case["axes"] > 1 else None)
    with torch.enable_grad():
        if kind == "attn":
            leaves = (st["q"], st["k"], st["v"])
            out = cross_attn_func(*leaves, q_starts=st.get("q_starts"), k_starts=st.get("k_starts"))
            return (out.detach(), *torch.autograd.grad(out, leaves, st["do"]))
        if kind == "norm":
            x, dt = st["x"], _dt(case["y"])
            if case["rms"]:
                leaves = (x, st["w"])
                y = rms_norm_func(*leaves, eps=EPS, out_dtype=dt)
            elif case["mode"] == "affine":
                leaves = (x, st["w"], st["b"])
                y = layer_norm_func(*leaves, eps=EPS, out_dtype=dt)
            else:
                leaves = (x, st["scale"], st["shift"])
                y = layer_norm_func(x, scale=leaves[1], shift=leaves[2], eps=EPS, out_dtype=dt)
            return (y.detach(), *torch.autograd.grad(y, leaves, st["dy"]))
        leaves = (st["q"], st["k"])
        q, k = rotary_func(*leaves, st["cos"], st["sin"], st["pos"], interleaved=case["layout"] == "interleaved",
                           sections=_sections(case) if case["axes"] > 1 else None)
        return (q.detach(), k.detach(), *torch.autograd.grad((q, k), leaves, (st["dq"], st["dk"])))


# ------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    size = {"f32": 4, "bf16": 2}
    if kind == "attn":
        B, H, Hk, D, Sq, Sk = (case[n] for n in ("B", "H", "Hk", "D", "Sq", "Sk"))
        pairs = B * Sq * Sk
        if case["docs"]:
            pairs = sum((q[n + 1] - q[n]) * (k[n + 1] - k[n]) for q, k in zip(*_borders(case)) for n in range(case["docs"]))
        # q, do in, out, dq out; k, v in, dk, dv out; two products forward, five backward (S again, dP, dq, dk, dv)
        return {"bytes": 2 * B * D * 4 * (Sq * H + Sk * Hk), "flops": 14 * D * H * pairs}
    if kind == "norm":
        n, params = case["B"] * case["S"] * case["dim"], (1 if case["mode"] == "affine" else case["B"]) * case["dim"]
        return {"bytes": n * (2 * size[case["x"]] + 2 * size[case["y"]]) + (8 if case["rms"] else 16) * params, "flops": 0}
    n = case["B"] * case["S"] * (case["H"] + case["Hk"]) * case["D"]
    table = min(case["B"] * case["S"], case["rows"]) * case["R"] // 2 * 8
    return {"bytes": n * size[case["x"]] * (4 if case["grad"] else 2) + table + 4 * case["B"] * case["S"] * case["axes"],
            "flops": 0}


# ------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------
def _exact_attn(case, st):
    B, H, Hk, D, Sq, Sk = (case[n] for n in ("B", "H", "Hk", "D", "Sq", "Sk"))
    q, k, v, do = (st[n].detach().double() for n in ("q", "k", "v", "do"))
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    qs, ks = _borders(case) if case["docs"] else ([[0, Sq]] * B, [[0, Sk]] * B)
    for b in range(B):
        for i0, i1, j0, j1 in zip(qs[b][:-1], qs[b][1:], ks[b][:-1], ks[b][1:]):
            if i1 <= i0 or j1 <= j0:
                continue
            for h in range(H):
                e = h // (H // Hk)
                Q, K, V, dO = q[b, i0:i1, h], k[b, j0:j1, e], v[b, j0:j1, e], do[b, i0:i1, h]
                P = torch.softmax(Q @ K.T / math.sqrt(D), 1)
                out[b, i0:i1, h] = P @ V
                dv[b, j0:j1, e] += P.T @ dO
                dP = dO @ V.T
                dS = P * (dP - (P * dP).sum(1, keepdim=True)) / math.sqrt(D)
                dq[b, i0:i1, h] = dS @ K
                dk[b, j0:j1, e] += dS.T @ Q
    return out, dq, dk, dv


def _exact_norm(case, st):
    x, dy = st["x"].detach().double(), st["dy"].double()
    n = case["dim"]
    affine = case["mode"] == "affine"
    gain = st["w"].detach().double() if affine else 1 + st["scale"].detach().double()
    if not case["rms"]:
        x = x - x.sum(-1, keepdim=True) / n
    r = torch.rsqrt(x.square().sum(-1, keepdim=True) / n + EPS)
    x *= r                                                      # normalised rows
    red = (lambda t: t.sum((0, 1))) if affine else (lambda t: t.sum(1, keepdim=True))
    y = x * gain
    dgain = red(x * dy)
    u = dy * gain
    dx = u - x * ((u * x).sum(-1, keepdim=True) / n)
    if case["rms"]:
        return y, dx * r, dgain
    dx -= u.sum(-1, keepdim=True) / n
    return y + (st["b"] if affine else st["shift"]).detach().double(), dx * r, dgain, red(dy)


def _exact_rotary(case, st):
    """The pairs as complex numbers times cos + i sin."""
    pos = st["pos"].long()
    table = torch.complex(st["cos"].double(), st["sin"].double())
    if case["axes"] == 1:
        f = table[pos]
    else:
        axis = torch.repeat_interleave(torch.arange(3, device=DEV), torch.tensor(_sections(case), device=DEV))
        f = table[pos[..., axis], torch.arange(case["R"] // 2, device=DEV)]
    f = f[:, :, None]
    R, inter = case["R"], case["layout"] == "interleaved"

    def turn(t, w):
        y = t.detach().double().clone()
        x = y[..., :R].unflatten(-1, (R // 2, 2) if inter else (2, R // 2))
        d = -1 if inter else -2
        z = torch.complex(x.select(d, 0), x.select(d, 1)) * w
        y[..., :R] = torch.stack([z.real, z.imag], d).flatten(-2)
        return y
    res = [turn(st["q"], f), turn(st["k"], f)]
    if case["grad"]:
        res += [turn(st["dq"], f.conj()), turn(st["dk"], f.conj())]
    return tuple(res)


def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        return {"attn": _exact_attn, "norm": _exact_norm, "rotary": _exact_rotary}[case["kind"]](case, st)
