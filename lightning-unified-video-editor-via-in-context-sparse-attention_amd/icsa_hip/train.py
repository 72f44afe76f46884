"""What a training step of the block needs around its sparse attention, with gradients, on MI355X.

* :func:`cross_attn_func`: attention to an encoder's states of another length (documents, shared key heads).
* :func:`layer_norm_func`, :func:`rms_norm_func`: with the gradients of a weight and bias, or of a scale and
  shift per batch row.
* :func:`rotary_func`, :func:`rotary_table`: rotary positions, interleaved or in halves, of part of a
  head, over one to four axes, for contexts longer than the trained one.

Each is an autograd node over a pair of library calls (csrc/autograd.cpp); without an enabled grad mode, or inputs
that require gradients, the forward alone runs and keeps nothing.  Gradients are sums in a fixed order: the same
inputs give the same bits.  There is no second derivative and none of forward mode; inputs are tensors with memory of their
own (vmap, ``torch.func``, batched gradients and tracing are refused).  :func:`cross_attn_fwd_hip` and
:func:`cross_attn_bwd_hip` are the attention's pair by itself, for callers with their own graph.
"""
from __future__ import annotations

import math

import torch

from . import _lib
from .hip_host import IcsaArgumentError, _require, _rows16, on_device, ptr, stream_ptr

_BF = torch.bfloat16
_FLOATS = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}
NORM_MAX_DIM = 8192
_WALK = 0x3fffffff           # elements within 32-bit byte offsets


_native = None


def _nodes():
    """The autograd nodes' module, bound to the library that the package has loaded (raises OSError when not built)."""
    global _native
    if _native is None:
        _lib.lib()
        try:
            from . import _autograd
        except ImportError as e:
            raise OSError("icsa_hip/_autograd.so not found; build it with `python -m icsa_hip.build`") from e
        _autograd.bind(_lib.lib_path(), _lib.IcsaError)
        _native = _autograd
    return _native


# ------------------------------------------------------------------------------------------
# cross attention
# ------------------------------------------------------------------------------------------
def _check_attn(q, k, v, q_starts, k_starts, softmax_scale):
    """Sizes, documents, scale; the borders contiguous."""
    if q.dtype != _BF or k.dtype != _BF or v.dtype != _BF:
        raise IcsaArgumentError("q, k, v must be bfloat16")
    dev = q.device
    if not q.is_cuda or k.device != dev or v.device != dev:
        raise IcsaArgumentError("q, k, v must be on the same GPU")
    if q.ndim != 4 or k.ndim != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise IcsaArgumentError("q [B, Sq, H, D], k/v [B, Sk, Hk, D] expected")
    B, Sq, H, D = q.shape
    Sk, Hk = k.shape[1:3]
    if D not in (64, 128):
        raise IcsaArgumentError("D must be 64 or 128")
    if B < 1 or Hk < 1 or H < 1 or H % Hk:
        raise IcsaArgumentError("H must be a multiple of Hk")
    docs = 1
    if q_starts is not None or k_starts is not None:
        if q_starts is None or k_starts is None or q_starts.ndim != 2 or q_starts.shape[0] != B or \
                q_starts.shape[1] < 2 or q_starts.shape != k_starts.shape:
            raise IcsaArgumentError("q_starts and k_starts must be given together, [B, N + 1]")
        for t in (q_starts, k_starts):
            if t.dtype != torch.int32 or t.device != dev:
                raise IcsaArgumentError("q_starts and k_starts must be int32 on the GPU of q")
        docs = q_starts.shape[1] - 1
        q_starts, k_starts = q_starts.contiguous(), k_starts.contiguous()
    scale = D ** -0.5 if softmax_scale is None else float(softmax_scale)
    if not scale >= 2.0 ** -96:
        raise IcsaArgumentError("softmax_scale must be positive, 2 ** -96 or more")
    return (B, Sq, Sk, H, Hk, D), docs, scale, q_starts, k_starts


def _require_plain(*ts):
    """As the autograd nodes do of their inputs."""
    if torch._C._get_tracing_state() is not None or not all(t is None or torch._C._has_storage(t) for t in ts):
        raise NotImplementedError("icsa_hip's training operators take tensors with memory of their own: not under vmap, torch.func or tracing")


def _near16(t, group=1):
    """:func:`_rows16`, and 64 rows with the heads of a group within 2 GiB, as the backward reads them."""
    t, a = _rows16(t)
    _, n1, n2, n3 = t.shape
    ss, sh = a[2] if n1 > 1 else 0, a[3] if n2 > 1 else 0
    if ss > _WALK // 65 or (group > 1 and sh > (_WALK - 65 * ss) // group):
        t = t.contiguous()
        a = (t.data_ptr(), n1 * n2 * n3, n2 * n3, n3)
    return t, a


@torch.no_grad()
def cross_attn_fwd_hip(q, k, v, q_starts=None, k_starts=None, softmax_scale=None):
    """``(out, lse, rest)`` of :func:`cross_attn_func`'s forward: out bfloat16 like q; lse float32 [B, Hk, Sq, H / Hk], log2 of each
    row's sum of ``2 ** (score * log2 e)``, +inf for a row that sees nothing; rest uint8 like out, what its rounding
    left, or None where that does not show in a gradient (without documents: over 256 keys, with heads of 64 over 1,024, and over 128 queries)."""
    _require_plain(q, k, v, q_starts, k_starts)
    sizes, docs, scale, q_starts, k_starts = _check_attn(q, k, v, q_starts, k_starts, softmax_scale)
    B, Sq, Sk, H, Hk, D = sizes
    dev = q.device
    q, qa = _near16(q, H // Hk)
    k, ka = _near16(k)
    v, va = _near16(v)
    out = torch.empty(B, Sq, H, D, dtype=_BF, device=dev)
    lse = torch.empty(B, Hk, Sq, H // Hk, dtype=torch.float32, device=dev)
    L = _lib.lib()
    rest = torch.empty(B, Sq, H, D, dtype=torch.uint8, device=dev) if L.icsa_cross_attn_wants_rest(Sq, Sk, H, Hk, D, q_starts is not None) else None
    wsp, ws_bytes = 0, L.icsa_cross_attn_workspace_size(*sizes, docs)
    if ws_bytes:
        if ws_bytes < 0:
            raise _lib.IcsaError("icsa_cross_attn_workspace_size", int(ws_bytes))
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        wsp = ws.data_ptr()
    with on_device(dev):
        rc = L.icsa_cross_attn_fwd(*qa, *ka, *va, *sizes, ptr(q_starts), ptr(k_starts), docs, scale, out.data_ptr(), Sq * H * D, H * D, D,
                                   lse.data_ptr(), ptr(rest), wsp, ws_bytes, stream_ptr(dev))
    _lib.check("icsa_cross_attn_fwd", rc)
    return out, lse, rest


@torch.no_grad()
def cross_attn_bwd_hip(dout, q, k, v, out, lse, rest=None, q_starts=None, k_starts=None, softmax_scale=None, grad_dtype=_BF,
                       need=(True, True, True)):
    """Gradients ``(dq, dk, dv)`` (bfloat16 or float32 by ``grad_dtype``; None where ``need`` is false) from the forward's
    inputs and results.  Without ``rest`` rowsum(dout * out) comes from the rounded out alone, whose error shows in dq and
    dk where rows see few keys."""
    _require_plain(dout, q, k, v, out, lse, rest, q_starts, k_starts)
    sizes, docs, scale, q_starts, k_starts = _check_attn(q, k, v, q_starts, k_starts, softmax_scale)
    B, Sq, Sk, H, Hk, D = sizes
    dev = q.device
    if dout.dtype != _BF or out.dtype != _BF or dout.shape != q.shape or out.shape != q.shape:
        raise IcsaArgumentError("dout and out must be bfloat16 like q")
    if lse.dtype != torch.float32 or lse.shape != (B, Hk, Sq, H // Hk) or not lse.is_contiguous():
        raise IcsaArgumentError(f"lse must be float32 [{B}, {Hk}, {Sq}, {H // Hk}], contiguous")
    if rest is not None and (rest.dtype != torch.uint8 or rest.shape != q.shape or not rest.is_contiguous()):
        raise IcsaArgumentError("rest must be uint8 like q, contiguous")
    if any(t is not None and t.device != dev for t in (dout, out, lse, rest)):
        raise IcsaArgumentError("dout, out, lse and rest must be on the GPU of q")
    if grad_dtype not in _FLOATS:
        raise IcsaArgumentError("grad_dtype must be bfloat16 or float32")
    dout, da = _near16(dout, H // Hk)
    q, qa = _near16(q, H // Hk)
    k, ka = _near16(k)
    v, va = _near16(v)
    out, oa = _rows16(out)
    L = _lib.lib()
    ws_bytes = L.icsa_cross_attn_bwd_workspace_size(*sizes, docs)
    if ws_bytes < 0:
        raise _lib.IcsaError("icsa_cross_attn_bwd_workspace_size", int(ws_bytes))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    dq = torch.empty(B, Sq, H, D, dtype=grad_dtype, device=dev) if need[0] else None
    dk = torch.empty(B, Sk, Hk, D, dtype=grad_dtype, device=dev) if need[1] else None
    dv = torch.empty(B, Sk, Hk, D, dtype=grad_dtype, device=dev) if need[2] else None
    qs, ks = (Sq * H * D, H * D, D), (Sk * Hk * D, Hk * D, D)
    with on_device(dev):
        rc = L.icsa_cross_attn_bwd(*da, *qa, *ka, *va, *oa, lse.data_ptr(), ptr(rest), *sizes, ptr(q_starts), ptr(k_starts), docs, scale,
                                   _FLOATS[grad_dtype], ptr(dq), *qs, ptr(dk), *ks, ptr(dv), *ks, ws.data_ptr(), ws_bytes,
                                   stream_ptr(dev))
    _lib.check("icsa_cross_attn_bwd", rc)
    return dq, dk, dv


def cross_attn_func(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, q_starts: torch.Tensor = None,
                    k_starts: torch.Tensor = None, softmax_scale: float = None) -> torch.Tensor:
    """Attention of q [B, Sq, H, D] over an encoder's k / v [B, Sk, Hk, D], bfloat16, D 64 or 128, H a multiple of Hk (the
    H / Hk heads of a group share a key head), with gradients.  Returns bfloat16 [B, Sq, H, D].

    ``q_starts``, ``k_starts``: int32 [B, N + 1] on the GPU, not decreasing, as in ``masked_attn_func``: document n of
    batch row b has queries ``q_starts[b, n] .. q_starts[b, n + 1] - 1`` and keys likewise, and sees its own keys alone
    (a batch row whose text has ``n`` real tokens is one document, ``[0, Sq]`` and ``[0, n]``).  Values past the lengths
    are clamped on the GPU.  ``softmax_scale``: 2 ** -96 or more, default ``D ** -0.5``.
    With gradients, a tensor of which 64 rows (of q: with the heads of a group) do not lie within 2 GiB is copied.

    A query that sees nothing gets zeros; it, keys outside every document and padding take no part in any gradient and
    get zeros, whatever they and their ``dout`` hold.  A NaN or an infinity inside a document makes gradients of that
    document NaN, and reaches no other."""
    _, docs, scale, q_starts, k_starts = _check_attn(q, k, v, q_starts, k_starts, softmax_scale)
    return _nodes().cross_attn(q, k, v, q_starts, k_starts, docs, scale)


# ------------------------------------------------------------------------------------------
# layer norm, RMS norm
# ------------------------------------------------------------------------------------------
def _check_norm(x, out_dtype, eps, *params):
    if not x.is_cuda or x.dim() < 1 or x.dtype not in _FLOATS:
        raise IcsaArgumentError("x must be bfloat16 or float32 [..., dim] on the GPU")
    dim = x.shape[-1]
    if not 1 <= dim <= NORM_MAX_DIM:
        raise IcsaArgumentError(f"dim must be 1 to {NORM_MAX_DIM}")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in _FLOATS:
        raise IcsaArgumentError("out_dtype must be bfloat16 or float32")
    if not 0 <= eps < math.inf:
        raise IcsaArgumentError("eps must be finite and not negative")
    given = [t for t in params if t is not None]
    for t in given:
        if t.device != x.device or t.dtype not in _FLOATS or t.dtype != given[0].dtype:
            raise IcsaArgumentError("the parameters must be bfloat16 or float32, alike, on the GPU of x")
    return dim, float(eps), out_dtype


def layer_norm_func(x: torch.Tensor, weight: torch.Tensor = None, bias: torch.Tensor = None, *, scale: torch.Tensor = None,
                    shift: torch.Tensor = None, eps: float = 1e-6, out_dtype: torch.dtype = None) -> torch.Tensor:
    """Layer norm of x [..., dim] (bfloat16 or float32, dim up to 8,192), with gradients: ``(x - mean) * rstd * a + b``.

    ``a = weight``, ``b = bias``, [dim] each (a bias only beside a weight); or ``a = 1 + scale``, ``b = shift``, given
    together and alike in shape: one row for all ([dim] or [1, .., dim]), or for an x of three or more dims one of each
    batch row, [B, dim] or [B, 1, .., dim] with x's first dim B; or neither.  Parameters are bfloat16 or float32, their
    gradients of their type and shape.  All arithmetic is float32, rounded once, to ``out_dtype`` (default x's type)."""
    dim, eps, out_dtype = _check_norm(x, out_dtype, eps, weight, bias, scale, shift)
    if weight is not None or bias is not None:
        if scale is not None or shift is not None:
            raise IcsaArgumentError("weight and bias, or scale and shift, not both")
        if weight is None or weight.shape != (dim,) or (bias is not None and bias.shape != (dim,)):
            raise IcsaArgumentError(f"weight and bias must be [{dim}], a bias beside a weight")
        return _nodes().norm(x, weight, bias, False, False, eps, out_dtype)
    if scale is None and shift is None:
        return _nodes().norm(x, None, None, False, False, eps, out_dtype)
    if scale is None or shift is None or scale.shape != shift.shape:
        raise IcsaArgumentError("scale and shift come together, alike in shape")
    n = scale.dim()
    one = 1 <= n <= x.dim() and scale.shape[-1] == dim and scale.numel() == dim
    each = x.dim() >= 3 and n in (2, x.dim()) and scale.shape[0] == x.shape[0] and scale.shape[-1] == dim and \
        scale.numel() == x.shape[0] * dim
    if not (one or each):
        raise IcsaArgumentError(f"scale and shift must be [{dim}], [1, .., {dim}], or [B, {dim}] or [B, 1, .., {dim}] for x [B, .., {dim}]")
    return _nodes().norm(x, scale, shift, True, False, eps, out_dtype)


def rms_norm_func(x: torch.Tensor, weight: torch.Tensor = None, *, eps: float = 1e-6, out_dtype: torch.dtype = None) -> torch.Tensor:
    """RMS norm of x [..., dim] (bfloat16 or float32, dim up to 8,192), with gradients:
    ``x * rsqrt(mean(x^2) + eps) * weight``, weight [dim] bfloat16 or float32, or None.  All arithmetic is float32,
    rounded once, to ``out_dtype`` (default x's type)."""
    dim, eps, out_dtype = _check_norm(x, out_dtype, eps, weight)
    _require(weight is None or weight.shape == (dim,), f"weight must be [{dim}]")
    return _nodes().norm(x, weight, None, False, True, eps, out_dtype)


# ------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------
def rotary_table(positions: int, rotary_dim: int, theta: float = 10000.0, *, scaling: str = None, factor: float = 1.0,
                 trained: int = None, fast: float = 32.0, slow: float = 1.0, device="cuda"):
    """``(cos, sin)`` float32 [positions, rotary_dim / 2] for :func:`rotary_func`, from angles
    ``pos * theta^(-2 j / rotary_dim)`` in float64.  For contexts ``factor`` times the trained one, ``scaling``:

    * ``"linear"``: positions divided by ``factor``;
    * ``"base"``: theta times ``factor^(r / (r - 2))``, r = rotary_dim (4 or more): the slowest pair as with "linear", the
      fastest unchanged;
    * ``"blend"``: by each pair's turns over the ``trained`` length: those with more than ``fast`` unchanged, those with fewer
      than ``slow`` divided by ``factor``, linear between; both tables times ``0.1 ln(factor) + 1``.
    """
    _require(positions > 0 and rotary_dim > 0 and rotary_dim % 2 == 0, "positions must be positive, rotary_dim positive and even")
    _require(scaling in (None, "linear", "base", "blend"), "scaling must be None, 'linear', 'base' or 'blend'")
    _require(0 < theta < math.inf and 1 <= factor < math.inf, "theta must be positive, factor at least 1")
    _require(scaling is not None or factor == 1, "a factor needs a scaling")
    gain = 1.0
    if scaling == "base":
        _require(rotary_dim >= 4, "'base' needs two pairs")
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    inv = theta ** -(torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    if scaling == "linear":
        inv = inv / factor
    if scaling == "blend":
        _require(trained is not None and trained > 0 and fast > slow >= 0, "'blend' needs the trained length, and fast > slow")
        keep = ((trained * inv / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        inv = inv * keep + inv / factor * (1 - keep)
        gain = 0.1 * math.log(factor) + 1.0
    ang = torch.outer(torch.arange(positions, dtype=torch.float64, device=device), inv)
    return (torch.cos(ang) * gain).float(), (torch.sin(ang) * gain).float()


def rotary_func(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *,
                sections=None, interleaved: bool = True):
    """q [B, S, H, D] and k [B, S, Hk, D] (or None), bfloat16 or float32, turned by their tokens' angles in one launch, with
    gradients; returns new tensors ``(q, k)``, or q's alone without k.

    cos, sin: float32 [P, R / 2] (:func:`rotary_table`): the first R dims of a head are turned, the rest stays.  Pair j is
    dims ``2 j, 2 j + 1`` (``interleaved``) or ``j, j + R / 2``.  positions: int32 [B, S] or [S] on the GPU, rows of the
    tables; with ``sections`` (the pairs of each of up to 4 axes, R / 2 in all: frames, rows, columns) [B, S, A] or [S, A],
    each run of pairs turned by its axis' position.  A position outside the table (-1, say) leaves its pairs as they are.
    The tables have no gradient."""
    if not q.is_cuda or q.dim() != 4 or q.dtype not in _FLOATS:
        raise IcsaArgumentError("q must be bfloat16 or float32 [B, S, H, D] on the GPU")
    dev = q.device
    B, S, _, D = q.shape
    if k is not None and (k.dim() != 4 or k.dtype != q.dtype or k.device != dev or k.shape[:2] != q.shape[:2] or k.shape[3] != D):
        raise IcsaArgumentError("k must be [B, S, Hk, D] of q's type, on its GPU")
    f32 = torch.float32
    if cos.dtype != f32 or sin.dtype != f32 or cos.dim() != 2 or cos.shape != sin.shape or cos.device != dev or \
            sin.device != dev or cos.shape[0] < 1:
        raise IcsaArgumentError("cos and sin must be float32 [P, R / 2] on the GPU of q")
    if not 1 <= cos.shape[1] <= D // 2:
        raise IcsaArgumentError(f"the tables' R / 2 columns must be 1 to {D // 2}")
    if (cos.requires_grad or sin.requires_grad) and torch.is_grad_enabled():
        raise IcsaArgumentError("the tables have no gradient")
    want = (S,)
    if sections is not None:
        sections = tuple(int(n) for n in sections)
        if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) != cos.shape[1]:
            raise IcsaArgumentError(f"sections must be 1 to 4 counts of pairs, {cos.shape[1]} in all")
        want = (S, len(sections))
    if positions.dtype != torch.int32 or positions.device != dev or positions.shape not in (want, (B, *want)):
        raise IcsaArgumentError(f"positions must be int32 {[*want]} or {[B, *want]} on the GPU of q")
    out = _nodes().rotary(q, k, cos, sin, positions, sections or (), bool(interleaved))
    return out[0] if k is None else tuple(out)


__all__ = ["cross_attn_func", "cross_attn_fwd_hip", "cross_attn_bwd_hip", "layer_norm_func", "rms_norm_func", "rotary_func",
           "rotary_table"]
