"""The block's linear layers in microscaled 4-bit floating point (quantisation, product) and its
attention under masks, as callers have them done.

Sizes follow the repository's own configurations: dim 5120 (40 heads of 128), FFN 13,824, text
width 4,096 with 512 tokens, 1,560 tokens per latent frame, 65,520 tokens for 21 frames of target
and source, and odd lengths around them.

`own` false: the plain form, elementary torch operations in 32 bits.  `own` true: the calls that a
user makes of icsa_hip.
"""
import math
import os
import random
import sys

import torch
import torch.nn.functional as F

own = False

_PKG = os.path.join(os.getcwd(), "lightning-unified-video-editor-via-in-context-sparse-attention_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

DEV = "cuda"
BF = torch.bfloat16
GRP = 256                  # a row's length is padded to whole groups of 256 (8 blocks of 32)


# ------------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------------
def listed():
    return [
        # quantisation and back: the one modulation row of a denoising step (latency)
        dict(name="quant_time_row", kind="quant", M=1, K=5120, x="f32"),
        # odd rows and a length that ends inside a block (a checkpoint's odd layer)
        dict(name="quant_odd", kind="quant", M=3121, K=4100, x="f32"),
        # the activations of a 9-frame clip before the q / k / v projections
        dict(name="quant_9frames", kind="quant", M=14040, K=5120, x="bf16"),
        # the time projection: one row against 6 x 5120 outputs, f32 in and out (a single token's form)
        dict(name="linear_time_projection", kind="linear", M=1, N=30720, K=5120, x="f32", y="f32", act=None),
        # the text embedding's first layer: one prompt of 512 tokens
        dict(name="linear_text", kind="linear", M=512, N=5120, K=4096, x="bf16", y="bf16", act="gelu_tanh"),
        # a projection of the image-editing use: 2 x 1,560 tokens
        dict(name="linear_image", kind="linear", M=3120, N=5120, K=5120, x="bf16", y="bf16", act=None),
        # the FFN's first layer at the full 21-frame length: the largest product of the block
        dict(name="linear_ffn_21frames", kind="linear", M=65520, N=13824, K=5120, x="bf16", y="bf16", act="gelu_tanh"),
        # both layers of the FFN for a 9-frame clip, the hidden row in 4 bits between them
        dict(name="ffn_9frames", kind="ffn", M=14040, N=13824, K=5120),
        # one query token with grouped heads over a long context
        dict(name="attn_single_token", kind="attn", B=1, H=40, Hk=8, D=128, Sq=1, Sk=65536, docs=1, mask="none",
             cap=0.0, R=0),
        # a batch of text encodings of different lengths: heads of 64, a learned bias by distance
        dict(name="attn_text_encoder", kind="attn", B=4, H=64, Hk=64, D=64, Sq=512, Sk=512, docs=2, mask="none",
             cap=0.0, R=128),
        # an odd-length clip, the source frames as a prefix that every token sees, scores capped
        dict(name="attn_prefix_6frames", kind="attn", B=1, H=12, Hk=12, D=128, Sq=9373, Sk=9373, docs=1,
             mask="prefix", cap=30.0, R=0),
        # cross attention of four packed clips, each with its own prompt
        dict(name="attn_packed_text", kind="attn", B=1, H=40, Hk=40, D=128, Sq=32760, Sk=1400, docs=4, mask="none",
             cap=0.0, R=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quant", "linear", "linear", "linear", "ffn", "attn", "attn", "attn"])
    if kind == "quant":
        K = rng.choice([_log(rng, 1, 13824), 32 * _log(rng, 1, 432), 5120])
        return dict(kind=kind, M=_log(rng, 1, min(65520, 200000000 // K)), K=K, x=rng.choice(["bf16", "bf16", "f32"]))
    if kind == "linear":
        M = rng.choice([_log(rng, 1, 64), _log(rng, 1, 30000), 1560 * rng.randint(1, 9)])
        N = rng.choice([_log(rng, 16, 13824), 5120, 13824])
        K = rng.choice([_log(rng, 32, 13824), 5120, 4096])
        return dict(kind=kind, M=M, N=N, K=K, x=rng.choice(["bf16", "bf16", "f32"]),
                    y=rng.choice(["bf16", "bf16", "f32"]) if M <= 64 else "bf16", act=rng.choice([None, "gelu_tanh"]))
    if kind == "ffn":
        K = 128 * rng.choice([2, 5, 12, 13, 40])
        return dict(kind=kind, M=_log(rng, 1, 12000), N=_log(rng, 512, 13824) // 8 * 8, K=K)
    D = rng.choice([64, 128, 128])
    Hk = rng.choice([1, 2, 3, 5, 8, 12, 40])
    G = rng.choice([1, 1, 1, 2, 4, 5]) if Hk <= 12 else 1
    B = rng.choice([1, 1, 2, 3])
    form = rng.choice(["self", "self", "text", "few"])
    if form == "self":
        Sq = Sk = min(_log(rng, 64, 16384), int(math.sqrt(1.2e9 / (B * Hk * G))))
        mask = rng.choice(["none", "causal", "prefix"])
    elif form == "text":
        Sk = rng.choice([77, 226, 512, _log(rng, 32, 2048)])
        Sq = min(_log(rng, 64, 32768), int(1.2e9 / (B * Hk * G * Sk)))
        mask = "none"
    else:
        Sq = rng.randint(1, 4)
        Sk = min(_log(rng, 64, 131072), int(1.2e9 / (B * Hk * G * Sq)))
        mask = rng.choice(["none", "causal"])
    docs = rng.choice([1, 1, 2, 5]) if form != "few" else 1
    return dict(kind=kind, B=B, H=Hk * G, Hk=Hk, D=D, Sq=Sq, Sk=Sk, docs=docs, mask=mask,
                cap=rng.choice([0.0, 0.0, 20.0, 50.0]), R=rng.choice([0, 0, 16, 128]))


# ------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1000003 * int(seed) + 29)
    return g


def _n(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _dt(name):
    return torch.float32 if name == "f32" else BF


def _activations(g, M, K, dtype):
    """Rows after a modulated LayerNorm: unit variance, some channels several times larger."""
    return (_n(g, M, K) * torch.exp(0.7 * _n(g, K))).to(dtype)


def _weight(g, N, K):
    """A weight as a program keeps it: packed codes and block scales."""
    return _pack(*_quantise(_n(g, N, K) / math.sqrt(K)))


def _documents(case):
    """Document borders of each batch row, [B][docs + 1] for queries and for keys, and each
    document's prefix: the last documents end before the padded sequence does."""
    rng = random.Random(case["Sq"] * 7919 + case["Sk"] * 31 + case["docs"])
    B, n, Sq, Sk = case["B"], case["docs"], case["Sq"], case["Sk"]
    qs, ks, pre = [], [], []
    for _ in range(B):
        if n == 1:
            q, k = [0, Sq], [0, Sk]
        else:
            cut = sorted(rng.uniform(0, 1) for _ in range(n - 1)) + [rng.uniform(0.9, 1.0)]
            q = [0] + [int(c * Sq) for c in cut]
            kcut = cut if Sq == Sk else [(i + 1) / n * rng.uniform(0.9, 1.0) for i in range(n)]
            k = [0] + [int(c * Sk) for c in sorted(kcut)]
        qs.append(q)
        ks.append(k)
        pre.append([int((k[i + 1] - k[i]) * rng.uniform(0.2, 0.6)) for i in range(n)])
    return qs, ks, pre


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    st = {"case": case}
    if kind in ("quant", "linear", "ffn"):
        M, K = case["M"], case["K"]
        st["x"] = _activations(g, M, K, _dt(case.get("x", "bf16")))
    if kind in ("linear", "ffn"):
        N = case["N"]
        st["w"] = _weight(g, N, K)
        st["b"] = 0.1 * _n(g, N)
    if kind == "ffn":
        st["w2"] = _weight(g, K, N)
        st["b2"] = 0.1 * _n(g, K)
    if kind == "attn":
        B, H, Hk, D, Sq, Sk = (case[n] for n in ("B", "H", "Hk", "D", "Sq", "Sk"))
        st["q"] = (1.5 * _n(g, B, Sq, H, D)).to(BF)
        st["k"] = _n(g, B, Sk, Hk, D).to(BF)
        st["v"] = _n(g, B, Sk, Hk, D).to(BF)
        qs, ks, pre = _documents(case)
        if case["docs"] > 1:
            st["q_starts"] = torch.tensor(qs, dtype=torch.int32, device=DEV)
            st["k_starts"] = torch.tensor(ks, dtype=torch.int32, device=DEV)
        if case["mask"] == "prefix":
            st["prefix"] = torch.tensor(pre, dtype=torch.int32, device=DEV)
        if case["R"]:
            st["bias"] = _n(g, H, 2 * case["R"] + 1)
    return st


# ------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------
def _quantise(x):
    """e2m1 values [M, Kb, 32] (f32) and block exponents [M, Kb] of x [M, K]."""
    M, K = x.shape
    Kp = -(-K // GRP) * GRP
    b = F.pad(x.float(), (0, Kp - K)).view(M, Kp // 32, 32)
    amax = b.abs().amax(-1)
    e = (torch.frexp(amax).exponent - 3).clamp(-127, 127)
    e = torch.where(amax > 0, e, torch.full_like(e, -127))
    y = torch.ldexp(b, -e.unsqueeze(-1))
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = torch.clamp(torch.round(a / step) * step, max=6.0)
    return torch.where(y < 0, -q, q), e


def _pack(q, e):
    """Packed codes [M, Kp/2] and scale bytes [Kp/256, M, 8] of values and exponents."""
    a = q.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code | ((q < 0).to(torch.uint8) << 3)).view(q.shape[0], -1)
    sc = (e + 127).to(torch.uint8).view(q.shape[0], -1, 8).permute(1, 0, 2).contiguous()
    return code[:, 0::2] | (code[:, 1::2] << 4), sc


def _values(codes, scales):
    """f32 [M, Kp] of packed codes and scale bytes."""
    M = codes.shape[0]
    lut = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], -1).view(M, -1, 32)
    e = scales.permute(1, 0, 2).reshape(M, -1, 1).int() - 127
    return torch.ldexp(lut[c.long()], e).view(M, -1)


def _dequantised(x):
    q, e = _quantise(x)
    return torch.ldexp(q, e.unsqueeze(-1)).view(x.shape[0], -1)


def _gelu(t):
    return 0.5 * t * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t * t * t)))


def _linear(x, w, b, act):
    """f32 product of 4-bit x and w."""
    y = _dequantised(x) @ _values(*w).t() + b
    return _gelu(y) if act else y


def _visible(case, st, dev):
    """[B, Sq, Sk] truth values and the keys' distance from each query's aligned position."""
    B, Sq, Sk = case["B"], case["Sq"], case["Sk"]
    i, j = torch.arange(Sq, device=dev), torch.arange(Sk, device=dev)
    qs = st.get("q_starts", torch.tensor([[0, Sq]] * B, device=dev)).long()
    ks = st.get("k_starts", torch.tensor([[0, Sk]] * B, device=dev)).long()
    n = qs.shape[1] - 1
    qd = (i[None, :, None] >= qs[:, None, :]).sum(-1) - 1          # [B, Sq], n behind the last one
    kd = (j[None, :, None] >= ks[:, None, :]).sum(-1) - 1
    d = qd.clamp(max=n - 1)
    at = torch.gather(ks[:, 1:], 1, d) - torch.gather(qs[:, 1:], 1, d) + i      # aligned at the end
    dist = j[None, None, :] - at[:, :, None]
    see = (qd[:, :, None] == kd[:, None, :]) & (qd < n)[:, :, None]
    if case["mask"] != "none":
        ok = dist <= 0
        if case["mask"] == "prefix":
            end = torch.gather(ks[:, :-1] + st["prefix"], 1, d)
            ok = ok | (j[None, None, :] < end[:, :, None])
        see = see & ok
    return see, dist


def _attention(case, st):
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    G = case["H"] // case["Hk"]
    q = q.transpose(1, 2).contiguous()
    k = k.transpose(1, 2).repeat_interleave(G, 1)
    v = v.transpose(1, 2).repeat_interleave(G, 1)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(case["D"])
    if case["cap"]:
        s = case["cap"] * torch.tanh(s / case["cap"])
    see, dist = _visible(case, st, q.device)
    if case["R"]:
        at = dist.clamp(-case["R"], case["R"]) + case["R"]
        s = s + st["bias"][:, at].transpose(0, 1)
    s = s.masked_fill(~see[:, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))
    return o.transpose(1, 2).to(BF)


# ------------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------------
def run(st):
    case = st["case"]
    kind = case["kind"]
    if own:
        return _run_own(case, kind, st)
    with torch.no_grad():
        if kind == "quant":
            return _dequantised(st["x"])[:, :case["K"]].to(BF)
        if kind == "linear":
            return _linear(st["x"], st["w"], st["b"], case["act"]).to(_dt(case["y"]))
        if kind == "ffn":
            h = _linear(st["x"], st["w"], st["b"], "gelu_tanh")
            return _linear(h, st["w2"], st["b2"], None).to(BF)
        return _attention(case, st)


def _run_own(case, kind, st):
    from icsa_hip import MXFP4Tensor, masked_attn_func, mx_linear, mx_quantize
    if kind == "quant":
        return mx_quantize(st["x"]).dequantize(BF)
    if kind == "linear":
        w = MXFP4Tensor(*st["w"], (case["N"], case["K"]))
        return mx_linear(st["x"], w, st["b"], activation=case["act"], out_dtype=_dt(case["y"]))
    if kind == "ffn":
        w = MXFP4Tensor(*st["w"], (case["N"], case["K"]))
        w2 = MXFP4Tensor(*st["w2"], (case["K"], case["N"]))
        h = mx_linear(st["x"], w, st["b"], activation="gelu_tanh", out_dtype="mxfp4")
        return mx_linear(h, w2, st["b2"])
    return masked_attn_func(st["q"], st["k"], st["v"], q_starts=st.get("q_starts"), k_starts=st.get("k_starts"),
                            causal=case["mask"] != "none", prefix=st.get("prefix"), softcap=case["cap"],
                            bias=st.get("bias"))


# ------------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------------
def _mx_bytes(M, K):
    Kp = -(-K // GRP) * GRP
    return M * Kp * 17 / 32


def work(case):
    kind = case["kind"]
    size = {"f32": 4, "bf16": 2}
    if kind == "attn":
        B, H, Hk, D, Sq, Sk = (case[n] for n in ("B", "H", "Hk", "D", "Sq", "Sk"))
        qs, ks, pre = _documents(case)
        pairs = 0
        for b in range(B):
            for n in range(case["docs"]):
                lq, lk = qs[b][n + 1] - qs[b][n], ks[b][n + 1] - ks[b][n]
                if case["mask"] == "none":
                    pairs += lq * lk
                    continue
                least = pre[b][n] if case["mask"] == "prefix" else 0
                pairs += sum(min(lk, max(least, i + lk - lq + 1, 0)) for i in range(lq))
        return {"bytes": 2 * B * D * (2 * Sq * H + 2 * Sk * Hk), "flops": 4 * D * H * pairs}
    M, K = case["M"], case["K"]
    if kind == "quant":                              # to 4 bits, and back to bf16
        return {"bytes": M * K * (size[case["x"]] + 2) + 2 * _mx_bytes(M, K), "flops": 0}
    N = case["N"]
    if kind == "linear":
        return {"bytes": M * K * size[case["x"]] + _mx_bytes(N, K) + 4 * N + M * N * size[case["y"]],
                "flops": 2 * M * N * K}
    return {"bytes": 4 * M * K + _mx_bytes(N, K) + _mx_bytes(K, N) + 4 * (N + K), "flops": 4 * M * N * K}


# ------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------
def _exact_rounded(x):
    """f64 [M, K] of x's 4-bit values: nearest entry of the e2m1 table, ties to the even code."""
    M, K = x.shape
    b = F.pad(x.double(), (0, -K % 32)).view(M, -1, 32)
    amax = b.abs().amax(-1, keepdim=True)
    tiny = torch.full_like(amax, 2.0 ** -200)
    e = torch.floor(torch.log2(torch.maximum(amax, tiny)))
    e = torch.where(torch.exp2(e) > amax, e - 1, torch.where(torch.exp2(e + 1) <= amax, e + 1, e))
    s = torch.exp2((e - 2).clamp(-127, 127))
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
    mids = (table[1:] + table[:-1]) / 2
    a = (b / s).abs()
    low, high = torch.bucketize(a, mids), torch.bucketize(a, mids, right=True)   # differ at a tie alone
    code = torch.where(low == high, low, torch.where(low % 2 == 0, low, high))
    return (torch.sign(b) * table[code] * s).view(M, -1)[:, :K]


def _exact_weight(codes, scales, K):
    N = codes.shape[0]
    c = torch.stack([codes % 16, codes // 16], -1).view(N, -1).long()
    mag = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=codes.device)[c % 8]
    s = torch.exp2(scales.transpose(0, 1).reshape(N, -1).double() - 127)
    return (torch.where(c >= 8, -mag, mag) * s.repeat_interleave(32, 1))[:, :K]


def _exact_linear(x, w, b, act):
    y = _exact_rounded(x) @ _exact_weight(*w, x.shape[1]).t() + b.double()
    return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))) if act else y


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "quant":
        return _exact_rounded(st["x"])
    if kind == "linear":
        return _exact_linear(st["x"], st["w"], st["b"], case["act"])
    if kind == "ffn":
        h = _exact_linear(st["x"], st["w"], st["b"], True)
        return _exact_linear(h, st["w2"], st["b2"], None)
    B, H, Hk, D, Sq, Sk = (case[n] for n in ("B", "H", "Hk", "D", "Sq", "Sk"))
    qs, ks, pre = _documents(case)
    out = torch.zeros(B, Sq, H, D, dtype=torch.float64, device=DEV)
    for b in range(B):
        for n in range(case["docs"]):
            q0, q1, k0, k1 = qs[b][n], qs[b][n + 1], ks[b][n], ks[b][n + 1]
            if q1 == q0 or k1 == k0:
                continue
            d = torch.arange(k1 - k0, device=DEV)[None, :] - (torch.arange(q1 - q0, device=DEV)[:, None] + (k1 - k0) - (q1 - q0))
            hide = torch.zeros_like(d, dtype=torch.bool)
            if case["mask"] != "none":
                hide = d > 0
                if case["mask"] == "prefix":
                    hide[:, :pre[b][n]] = False
            empty = hide.all(1)
            for h in range(H):
                hk = h // (H // Hk)
                s = st["q"][b, q0:q1, h].double() @ st["k"][b, k0:k1, hk].double().t().contiguous() * D ** -0.5
                if case["cap"]:
                    s = torch.tanh(s / case["cap"]) * case["cap"]
                if case["R"]:
                    s += st["bias"][h].double()[d.clamp(-case["R"], case["R"]) + case["R"]]
                p = torch.softmax(s.masked_fill(hide, -math.inf), -1)
                o = p @ st["v"][b, k0:k1, hk].double()
                out[b, q0:q1, h] = torch.where(empty[:, None], torch.zeros_like(o), o)
    return out
