"""Root-mean-square norm with the residual's addition, and rows in 8 bits.

``rms_norm`` makes what the layer reads: its output is the layer's
``hidden_states``, or, in 8 bits with one scale a row, the rows that
``int8_matmul`` and ``FusedMoEForward.forward_few_int8`` take.
``quantize_rows`` makes such rows of weights and of activations. The reference
has neither: its layer begins behind the norm. Checks, outputs and the autograd
node are native (csrc/torch_ops.cpp).
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _lib

MAX_HIDDEN = 32768  # columns of a row (csrc/norm.hip)


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6, out_dtype: Optional[torch.dtype] = None):
    """``h / sqrt(mean(h^2) + eps) * weight`` over the last dimension, with
    ``h = x + residual`` (rounded to the residual's type) or ``h = x``.

    ``x`` [..., H] in bf16, fp16 or fp32 with H up to 32768, unit column stride
    and rows that are evenly spaced in memory; ``residual`` of the same shape in
    ``x.dtype`` or fp32; ``weight`` [H] in any of the three types (``None``: all
    ones). Statistics and ``eps`` are fp32, over the whole range of ``h``; every
    output is rounded once, and the norm is taken of ``h`` as it is stored.

    Returns ``y`` in ``x.dtype``; with ``residual`` ``(y, h)``. With
    ``out_dtype`` int8 or float8_e4m3fn ``y`` is replaced by ``q, scale``:
    ``y`` = ``q * scale[..., None]``, one fp32 scale a row (largest ``|y|`` /
    127 or 448; 1 for a row of zeros; NaN, with bytes of zero, for a row that
    holds a NaN or an infinity).

    Differentiable in ``x``, ``weight`` and ``residual`` (once) where the output
    is floating; 8-bit outputs carry no gradient and refuse inputs that ask for
    one. A captured backward raises while a graph built on the default stream
    still uses the same leaves.
    """
    return _lib.torch_ops().rms_norm(x, weight, residual, eps, out_dtype)


def quantize_rows(x: torch.Tensor, dtype: torch.dtype = torch.int8):
    """``(q, scale)`` with ``x`` about ``q * scale[..., None]``: the rows of
    ``x`` [..., columns] in int8 or float8_e4m3fn with one fp32 scale each, as
    the 8-bit output of ``rms_norm``. No gradient."""
    return _lib.torch_ops().quantize_rows(x, dtype)


__all__ = ["quantize_rows", "rms_norm"]
