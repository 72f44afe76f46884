"""Linear layers in microscaled 4-bit floating point (OCP MXFP4) on MI355X.

* :class:`MXFP4Tensor`: rows of e2m1 codes with a power of two for every 32 values.
* :func:`mx_quantize` / :meth:`MXFP4Tensor.dequantize`: to that form and back.
* :func:`mx_linear`: ``act(x w^T + bias)`` on the block-scaled matrix instructions.
* :class:`MXLinear`, :func:`quantize_linears`: the same for the layers of a model.

These are inference operators, like the dense attention and the block they serve: under an
enabled grad mode an input that requires a gradient is refused.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib
from .hip_host import _require, dtype_code, on_device, ptr, stream_ptr

MX_GROUP = 256        # k values of one padded group (8 blocks of 32)

_ACTIVATIONS = {None: 0, "gelu_tanh": 1}


def _padded(k: int) -> int:
    return (k + MX_GROUP - 1) // MX_GROUP * MX_GROUP


def _no_grad_inputs(*tensors) -> None:
    if torch.is_grad_enabled():
        _require(not any(t is not None and t.requires_grad for t in tensors),
                 "the 4-bit operators have no backward: call them under torch.no_grad()")


class MXFP4Tensor:
    """A tensor ``[..., K]`` in 4 bits.

    Rows (the leading dims flattened) are padded with zeros to ``Kp``, K rounded up to 256.
    ``codes`` uint8 ``[rows, Kp / 2]``: e2m1 (sign, 2 exponent bits, 1 mantissa bit), the even k in
    the low nibble.  ``scales`` uint8 ``[Kp / 256, rows, 8]``: the 8 blocks of 32 of each group of
    256; a block's values are its codes' times ``2^(scale - 127)``, 255 stands for NaN."""

    __slots__ = ("codes", "scales", "shape")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape):
        shape = torch.Size(shape)
        _require(len(shape) >= 1 and shape[-1] > 0, "shape must end in a positive length")
        rows, Kp = shape[:-1].numel(), _padded(shape[-1])
        _require(codes.dtype == torch.uint8 and scales.dtype == torch.uint8, "codes and scales must be uint8")
        _require(tuple(codes.shape) == (rows, Kp // 2), f"codes must be [{rows}, {Kp // 2}]")
        _require(tuple(scales.shape) == (Kp // MX_GROUP, rows, 8), f"scales must be [{Kp // MX_GROUP}, {rows}, 8]")
        _require(codes.device == scales.device, "codes and scales must be on one device")
        _require(codes.is_contiguous() and scales.is_contiguous(), "codes and scales must be contiguous")
        self.codes, self.scales, self.shape = codes, scales, shape

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def __repr__(self) -> str:
        return f"MXFP4Tensor(shape={tuple(self.shape)}, device={self.device})"

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values as bf16 (which holds each of them exactly) or float32, a new tensor."""
        _require(self.codes.is_cuda, "codes must be on the GPU")
        _require(dtype in (torch.bfloat16, torch.float32), "dtype must be bfloat16 or float32")
        K = self.shape[-1]
        out = torch.empty(self.shape, dtype=dtype, device=self.device)
        with on_device(self.device):
            rc = _lib.lib().icsa_mx_dequantize(ptr(self.codes), ptr(self.scales), self.codes.shape[0], K,
                                               ptr(out), dtype_code(out), K, stream_ptr(self.device))
        _lib.check("icsa_mx_dequantize", rc)
        return out


def _empty(shape, device) -> MXFP4Tensor:
    shape = torch.Size(shape)
    rows, Kp = shape[:-1].numel(), _padded(shape[-1])
    return MXFP4Tensor(torch.empty(rows, Kp // 2, dtype=torch.uint8, device=device),
                       torch.empty(Kp // MX_GROUP, rows, 8, dtype=torch.uint8, device=device), shape)


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [..., K] as [rows, K] with a unit stride in each row (a view where there is one)."""
    x = x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()
    return x.reshape(-1, x.shape[-1])


def mx_quantize(x: torch.Tensor) -> MXFP4Tensor:
    """x [..., K] (bf16 or float32, rows at any stride) in 4 bits.  A block's scale is
    ``2^(floor(log2 max|x|) - 2)``, codes are rounded to the nearest (ties to even), what is over 6
    scales becomes 6, and a block with a NaN or an infinity reads as NaN."""
    _no_grad_inputs(x)
    _require(x.is_cuda, "x must be on the GPU")
    _require(x.dim() >= 1 and x.shape[-1] > 0, "x must be [..., K] with K > 0")
    code = dtype_code(x)
    t = _empty(x.shape, x.device)
    r = _rows(x)
    with on_device(x.device):
        rc = _lib.lib().icsa_mx_quantize(ptr(r), code, r.stride(0), r.shape[0], r.shape[1],
                                         ptr(t.codes), ptr(t.scales), stream_ptr(x.device))
    _lib.check("icsa_mx_quantize", rc)
    return t


def mx_linear(x, weight: MXFP4Tensor, bias: torch.Tensor = None, activation: str = None, out_dtype=torch.bfloat16):
    """``act(x weight^T + bias)``: x [..., K] as an :class:`MXFP4Tensor`, or bf16 / float32 that the
    call quantises; weight [N, K]; bias bf16 or float32 [N]; activation None or ``"gelu_tanh"``.
    Sums are float32 and the result is rounded once, to ``out_dtype``: ``torch.bfloat16``,
    ``torch.float32``, or ``"mxfp4"`` for an :class:`MXFP4Tensor` [..., N] that the next product takes."""
    mx_in = isinstance(x, MXFP4Tensor)
    _require(isinstance(weight, MXFP4Tensor) and len(weight.shape) == 2, "weight must be an MXFP4Tensor [N, K]")
    _require(activation in _ACTIVATIONS, "activation must be None or 'gelu_tanh'")
    _require(out_dtype in (torch.bfloat16, torch.float32, "mxfp4"), "out_dtype must be bfloat16, float32 or 'mxfp4'")
    _no_grad_inputs(None if mx_in else x, bias)
    N, K = weight.shape
    dev = weight.device
    _require(dev.type == "cuda" and x.device == dev, "x and weight must be on the same GPU")
    _require(len(x.shape) >= 1 and x.shape[-1] == K, f"x must be [..., {K}]")
    b_code = _lib.F32
    if bias is not None:
        _require(tuple(bias.shape) == (N,) and bias.device == dev, f"bias must be [{N}] on the weight's GPU")
        b_code = dtype_code(bias)
        bias = bias.contiguous()
    L = _lib.lib()
    if mx_in:
        M, xp, xs, x_code, x_ss = x.codes.shape[0], ptr(x.codes), ptr(x.scales), _lib.MXFP4, 0
        ws, ws_bytes = None, 0
    else:
        r = _rows(x)
        M, xp, xs, x_code, x_ss = r.shape[0], ptr(r), 0, dtype_code(r), r.stride(0)
        ws_bytes = L.icsa_mx_linear_workspace_size(M, N, K, x_code)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    shape = (*x.shape[:-1], N)
    if out_dtype == "mxfp4":
        out = _empty(shape, dev)
        op, osc, o_code = ptr(out.codes), ptr(out.scales), _lib.MXFP4
    else:
        out = torch.empty(shape, dtype=out_dtype, device=dev)
        op, osc, o_code = ptr(out), 0, dtype_code(out)
    with on_device(dev):
        rc = L.icsa_mx_linear(xp, xs, x_code, x_ss, ptr(weight.codes), ptr(weight.scales), ptr(bias), b_code,
                              _ACTIVATIONS[activation], M, N, K, op, osc, o_code, N, ptr(ws), ws_bytes, stream_ptr(dev))
    _lib.check("icsa_mx_linear", rc)
    return out


class MXLinear(nn.Module):
    """``nn.Linear`` with its weight in 4 bits, for inference: quantised once from ``linear``'s weight,
    the bias as it was.  ``forward`` takes bf16, float32 or an :class:`MXFP4Tensor` and returns
    ``out_dtype``, by default x's own type (bfloat16 for an x in 4 bits)."""

    def __init__(self, linear: nn.Linear):
        super().__init__()
        self.in_features, self.out_features = linear.in_features, linear.out_features
        w = mx_quantize(linear.weight.detach())
        self.register_buffer("codes", w.codes)
        self.register_buffer("scales", w.scales)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().clone())

    @property
    def weight(self) -> MXFP4Tensor:
        return MXFP4Tensor(self.codes, self.scales, (self.out_features, self.in_features))

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"

    def forward(self, x, activation: str = None, out_dtype=None):
        if out_dtype is None:
            out_dtype = torch.bfloat16 if isinstance(x, MXFP4Tensor) else x.dtype
        return mx_linear(x, self.weight, self.bias, activation, out_dtype)


__all__ = ["MXFP4Tensor", "mx_quantize", "mx_linear", "MXLinear"]
