"""Root-mean-square norm with the residual's addition, and rows in 8 bits.

``rms_norm`` makes what the layer reads: its output is the layer's
``hidden_states``, or, in 8 bits with one scale a row, the rows that
``int8_matmul`` and ``FusedMoEForward.forward_few_int8`` take.
``quantize_rows`` makes such rows of weights and of activations. The reference
has neither: its layer begins behind the norm.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from . import _kernels as K

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_EIGHT_BITS = (torch.int8, torch.float8_e4m3fn)
MAX_HIDDEN = 32768  # columns of a row (csrc/norm.hip)


def _check_float(name: str, t: torch.Tensor):
    if t.dtype not in _FLOATS:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")


def _check_device(name: str, t: torch.Tensor):
    if not t.is_cuda:
        raise ValueError(f"{name} must be a HIP device tensor")


def _check_columns(name: str, columns: int):
    if not 1 <= columns <= MAX_HIDDEN:
        raise ValueError(f"{name} must have 1 to {MAX_HIDDEN} columns, got {columns}")


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, _, h, rstd = K.rms_norm(x, weight, residual, eps, x.dtype, keep_rstd=True)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x if residual is None else h, weight, rstd)
        ctx.x_dtype, ctx.has_residual = x.dtype, residual is not None
        return y if residual is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        # grad mode is on here only under create_graph, whose second backward must raise
        return _rms_norm_grads_once(ctx, dy, dh) if torch.is_grad_enabled() else _rms_norm_grads(ctx, dy, dh)


def _rms_norm_grads(ctx, dy, dh):
    h, weight, rstd = ctx.saved_tensors
    if dy is None and dh is None:
        return None, None, None, None
    if dy is None:
        dy = torch.zeros(h.shape, dtype=ctx.x_dtype, device=h.device)
    dx, dres, dw = K.rms_norm_bwd(dy, dh, h, weight, rstd, ctx.x_dtype, ctx.has_residual and ctx.needs_input_grad[2],
                                  weight is not None and ctx.needs_input_grad[1])
    return dx, dw, dres, None


_rms_norm_grads_once = torch.autograd.function.once_differentiable(_rms_norm_grads)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6, out_dtype: Optional[torch.dtype] = None):
    """``h / sqrt(mean(h^2) + eps) * weight`` over the last dimension, with
    ``h = x + residual`` (rounded to the residual's type) or ``h = x``.

    ``x`` [..., H] in bf16, fp16 or fp32 with H up to 32768, unit column stride
    and rows that are evenly spaced in memory; ``residual`` of the same shape in
    ``x.dtype`` or fp32; ``weight`` [H] in any of the three types (``None``: all
    ones). Statistics are fp32; every output is rounded once, and the norm is
    taken of ``h`` as it is stored.

    Returns ``y`` in ``x.dtype``; with ``residual`` ``(y, h)``. With
    ``out_dtype`` int8 or float8_e4m3fn ``y`` is replaced by ``q, scale``:
    ``y`` = ``q * scale[..., None]``, one fp32 scale a row (largest ``|y|`` /
    127 or 448; 1 for a row of zeros; NaN, with bytes of zero, for a row that
    holds a NaN or an infinity).

    Differentiable in ``x``, ``weight`` and ``residual`` (once) where the output
    is floating; 8-bit outputs carry no gradient and refuse inputs that ask for
    one.
    """
    dtype = x.dtype
    _check_float("x", x)
    if x.dim() == 0:
        raise ValueError("x must have shape [..., hidden]")
    hidden = x.shape[-1]
    _check_columns("x", hidden)
    if weight is not None:
        _check_float("weight", weight)
        if weight.dim() != 1 or weight.shape[0] != hidden or not weight.is_contiguous():
            raise ValueError(f"weight must be contiguous with shape ({hidden},), got {tuple(weight.shape)}")
        if weight.device != x.device:
            raise ValueError("weight and x must be on the same device")
    if residual is not None:
        if residual.dtype != dtype and residual.dtype != torch.float32:
            raise TypeError(f"residual must use {dtype} or torch.float32, got {residual.dtype}")
        if residual.shape != x.shape:
            raise ValueError(f"residual must have shape {tuple(x.shape)}, got {tuple(residual.shape)}")
        if residual.device != x.device:
            raise ValueError("residual and x must be on the same device")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if out_dtype is None:
        out_dtype = dtype
    elif out_dtype != dtype and out_dtype not in _EIGHT_BITS:
        raise TypeError(f"out_dtype must be {dtype}, torch.int8 or torch.float8_e4m3fn, got {out_dtype}")
    needs_grad = (x.requires_grad or (weight is not None and weight.requires_grad)
                  or (residual is not None and residual.requires_grad)) and torch.is_grad_enabled()
    eight_bits = out_dtype != dtype
    if eight_bits:
        if needs_grad:
            raise ValueError("an 8-bit output carries no gradient; call under torch.no_grad() or on detached inputs")
    _check_device("x", x)
    if eight_bits:
        q, scale, h, _ = K.rms_norm(x, weight, residual, eps, out_dtype)
        return (q, scale) if residual is None else (q, scale, h)
    if needs_grad:
        return _RMSNorm.apply(x, weight, residual, eps)
    y, _, h, _ = K.rms_norm(x, weight, residual, eps, out_dtype)
    return y if residual is None else (y, h)


def quantize_rows(x: torch.Tensor, dtype: torch.dtype = torch.int8):
    """``(q, scale)`` with ``x`` about ``q * scale[..., None]``: the rows of
    ``x`` [..., columns] in int8 or float8_e4m3fn with one fp32 scale each, as
    the 8-bit output of ``rms_norm``. No gradient."""
    _check_float("x", x)
    if x.dim() == 0:
        raise ValueError("x must have shape [..., columns]")
    _check_columns("x", x.shape[-1])
    if dtype not in _EIGHT_BITS:
        raise TypeError(f"dtype must be torch.int8 or torch.float8_e4m3fn, got {dtype}")
    if torch.is_grad_enabled() and x.requires_grad:
        raise ValueError("an 8-bit output carries no gradient; call under torch.no_grad() or on a detached input")
    _check_device("x", x)
    return K.quantize_rows(x, dtype)


__all__ = ["quantize_rows", "rms_norm"]
