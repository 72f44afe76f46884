"""Linear layers in microscaled 4-bit floating point (OCP MXFP4) on MI355X.

* :class:`MXFP4Tensor`: rows of e2m1 codes with a power of two for every 32 values.
* :func:`mx_quantize` / :meth:`MXFP4Tensor.dequantize`: to that form and back.
* :func:`mx_linear`: ``act(x w^T + bias)`` on the block-scaled matrix instructions.
* :class:`MXLinear`: the same as a module (``wan.quantize_linears`` puts it into a block).

These are inference operators, like the dense attention and the block they serve: under an
enabled grad mode an input that requires a gradient is refused.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from . import _lib
from .hip_host import IcsaArgumentError, dtype_code, on_device, stream_ptr

MX_GROUP = 256        # k values of one padded group (8 blocks of 32)

_ACTIVATIONS = {None: 0, "gelu_tanh": 1}
_OUT_CODES = {torch.bfloat16: _lib.BF16, torch.float32: _lib.F32}


def _padded(k: int) -> int:
    return (k + MX_GROUP - 1) // MX_GROUP * MX_GROUP


def _no_grad_inputs(*tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise IcsaArgumentError("the 4-bit operators have no backward: call them under torch.no_grad()")


class MXFP4Tensor:
    """A tensor ``[..., K]`` in 4 bits.

    Rows (the leading dims flattened) are padded with zeros to ``Kp``, K rounded up to 256.
    ``codes`` uint8 ``[rows, Kp / 2]``: e2m1 (sign, 2 exponent bits, 1 mantissa bit), the even k in
    the low nibble.  ``scales`` uint8 ``[Kp / 256, rows, 8]``: the 8 blocks of 32 of each group of
    256; a block's values are its codes' times ``2^(scale - 127)``, 255 stands for NaN.  Both
    16-byte aligned."""

    __slots__ = ("_codes", "_scales", "_buf", "shape", "rows", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, shape):
        shape = torch.Size(shape)
        if not shape or shape[-1] <= 0:
            raise IcsaArgumentError("shape must end in a positive length")
        rows, Kp = math.prod(shape[:-1]), _padded(shape[-1])
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise IcsaArgumentError("codes and scales must be uint8")
        if codes.shape != (rows, Kp // 2) or scales.shape != (Kp // MX_GROUP, rows, 8):
            raise IcsaArgumentError(f"codes must be [{rows}, {Kp // 2}] and scales [{Kp // MX_GROUP}, {rows}, 8]")
        if codes.device != scales.device or not codes.is_contiguous() or not scales.is_contiguous():
            raise IcsaArgumentError("codes and scales must be contiguous, on one device")
        self._codes, self._scales, self._buf = codes, scales, None
        self.shape, self.rows, self.device = shape, rows, codes.device

    @classmethod
    def _empty(cls, shape: torch.Size, rows: int, device) -> "MXFP4Tensor":
        """Codes and scales side by side in one new buffer; the views of it are made when asked for."""
        t = cls.__new__(cls)
        n = rows * (_padded(shape[-1]) // 2)                      # bytes of codes, a multiple of 128; a 16th of them is scales
        t._buf = torch.empty(n + n // 16, dtype=torch.uint8, device=device)
        t._codes = t._scales = None
        t.shape, t.rows, t.device = shape, rows, device
        return t

    def _ptrs(self):
        """Addresses of the codes and the scales."""
        if self._buf is None:
            return self._codes.data_ptr(), self._scales.data_ptr()
        p = self._buf.data_ptr()
        return p, p + self._buf.shape[0] // 17 * 16

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            Kp = _padded(self.shape[-1])
            self._codes = self._buf[:self.rows * (Kp // 2)].view(self.rows, Kp // 2)
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            Kp = _padded(self.shape[-1])
            self._scales = self._buf[self.rows * (Kp // 2):].view(Kp // MX_GROUP, self.rows, 8)
        return self._scales

    def __repr__(self) -> str:
        return f"MXFP4Tensor(shape={tuple(self.shape)}, device={self.device})"

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values as bf16 or float32, a new tensor: exactly, but for those from 2^128 on (scale bytes 253 and 254, which
        :func:`mx_quantize` does not write), which become infinities."""
        dev, K = self.device, self.shape[-1]
        if dev.type != "cuda":
            raise IcsaArgumentError("codes must be on the GPU")
        if dtype not in _OUT_CODES:
            raise IcsaArgumentError("dtype must be bfloat16 or float32")
        out = torch.empty(*self.shape, dtype=dtype, device=dev)
        with on_device(dev):
            rc = _lib.lib().icsa_mx_dequantize(*self._ptrs(), self.rows, K, out.data_ptr(), _OUT_CODES[dtype], K, stream_ptr(dev))
        _lib.check("icsa_mx_dequantize", rc)
        return out


def _rows(x: torch.Tensor) -> torch.Tensor:
    """x [..., K] as [rows, K] with a unit stride in each row (a view where there is one)."""
    if x.stride(-1) != 1 and x.shape[-1] != 1:
        x = x.contiguous()
    return x if x.dim() == 2 else x.reshape(-1, x.shape[-1])


def mx_quantize(x: torch.Tensor) -> MXFP4Tensor:
    """x [..., K] (bf16 or float32, rows at any stride) in 4 bits.  A block's scale is
    ``2^(floor(log2 max|x|) - 2)``, codes are rounded to the nearest (ties to even), what is over 6
    scales becomes 6, and a block with a NaN or an infinity reads as NaN."""
    _no_grad_inputs(x)
    shape, dev = x.shape, x.device
    if not x.is_cuda or len(shape) < 1 or shape[-1] < 1:
        raise IcsaArgumentError("x must be [..., K] with K > 0, on the GPU")
    code, K = dtype_code(x), shape[-1]
    rows = x.numel() // K
    t = MXFP4Tensor._empty(shape, rows, dev)
    r = _rows(x)
    with on_device(dev):
        rc = _lib.lib().icsa_mx_quantize(r.data_ptr(), code, r.stride(0), rows, K, *t._ptrs(), stream_ptr(dev))
    _lib.check("icsa_mx_quantize", rc)
    return t


def mx_linear(x, weight: MXFP4Tensor, bias: torch.Tensor = None, activation: str = None, out_dtype=torch.bfloat16):
    """``act(x weight^T + bias)``: x [..., K] as an :class:`MXFP4Tensor`, or bf16 / float32 that the
    call quantises; weight [N, K]; bias bf16 or float32 [N]; activation None or ``"gelu_tanh"``.
    Sums are float32 and the result is rounded once, to ``out_dtype``: ``torch.bfloat16``,
    ``torch.float32``, or ``"mxfp4"`` for an :class:`MXFP4Tensor` [..., N] that the next product takes."""
    mx_in = isinstance(x, MXFP4Tensor)
    if not isinstance(weight, MXFP4Tensor) or len(weight.shape) != 2:
        raise IcsaArgumentError("weight must be an MXFP4Tensor [N, K]")
    if activation not in _ACTIVATIONS:
        raise IcsaArgumentError("activation must be None or 'gelu_tanh'")
    if out_dtype != "mxfp4" and out_dtype not in _OUT_CODES:
        raise IcsaArgumentError("out_dtype must be bfloat16, float32 or 'mxfp4'")
    _no_grad_inputs(None if mx_in else x, bias)
    N, K = weight.shape
    dev = weight.device
    if dev.type != "cuda" or x.device != dev:
        raise IcsaArgumentError("x and weight must be on the same GPU")
    if len(x.shape) < 1 or x.shape[-1] != K:
        raise IcsaArgumentError(f"x must be [..., {K}]")
    bp, b_code = 0, _lib.F32
    if bias is not None:
        if bias.shape != (N,) or bias.device != dev:
            raise IcsaArgumentError(f"bias must be [{N}] on the weight's GPU")
        b_code = dtype_code(bias)
        bias = bias.contiguous()
        bp = bias.data_ptr()
    L = _lib.lib()
    if mx_in:
        M, (xp, xs), x_code, x_ss, wsp, ws_bytes = x.rows, x._ptrs(), _lib.MXFP4, 0, 0, 0
    else:
        r = _rows(x)
        M, xp, xs, x_code, x_ss = r.shape[0], r.data_ptr(), 0, dtype_code(r), r.stride(0)
        ws_bytes = L.icsa_mx_linear_workspace_size(M, N, K, x_code)
        wsp = 0
        if ws_bytes > 0:
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
            wsp = ws.data_ptr()
    shape = (*x.shape[:-1], N)
    if out_dtype == "mxfp4":
        out = MXFP4Tensor._empty(torch.Size(shape), M, dev)
        (op, osc), o_code = out._ptrs(), _lib.MXFP4
    else:
        out = torch.empty(*shape, dtype=out_dtype, device=dev)
        op, osc, o_code = out.data_ptr(), 0, _OUT_CODES[out_dtype]
    with on_device(dev):
        rc = L.icsa_mx_linear(xp, xs, x_code, x_ss, *weight._ptrs(), bp, b_code, _ACTIVATIONS[activation],
                              M, N, K, op, osc, o_code, N, wsp, ws_bytes, stream_ptr(dev))
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
        self.register_buffer("codes", w.codes.clone())            # tensors of their own: a state dict saves each
        self.register_buffer("scales", w.scales.clone())
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
