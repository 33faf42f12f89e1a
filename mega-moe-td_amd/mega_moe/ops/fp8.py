"""E4M3 with a power-of-two scale for each block of 128: blocks, products, a
trained projection, and the experts in that form.

A value is ``q * scale`` with ``q`` in float8_e4m3fn and ``scale`` in
float8_e8m0fnu (one byte, 2^k): one scale for 128 consecutive columns of a row
(activations) or for 128 x 128 (weights), as the matrix instruction takes them.
``scale`` is the smallest power of two, from 2^-126 on, for which the block's
largest value stays within 448 (1 for a block of zeros), so a quotient is exact
and ``q`` is rounded once; a block that holds a NaN or an infinity has scale NaN
and bytes 0. The last blocks of an axis hold what is left of it. ``rms_norm``
makes such rows too. The reference has no 8-bit products.

Products to float32 sum in fp32 throughout. Those to bf16 and fp16 sum in the E4M3
matrix instruction, which is twice as fast: of the 8 products of 8 neighbouring
columns it cuts each 13 bits below the largest, and adds what is left in fp32. A sum
is off by at most 7 * 2^-13 (8.5e-4) of the sum of those largest products' sizes, by
1.4e-5 of a sum of random values, but terms that are small beside others that cancel
are lost: 448 * 448 - 448 * 448 + 1 is 0. Where such sums matter ask for float32.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .. import _lib

BLOCK = 128  # values that share a scale along an axis (MM_FP8_BLOCK)


def quantize_blocks(x: torch.Tensor, rows: int = 1):
    """``(q, scale)`` of ``x`` [..., columns] in bf16, fp16 or fp32, unit column
    stride and evenly spaced. ``rows`` = 1: rows in blocks of 128 columns,
    ``scale`` [..., ceil(columns / 128)]. ``rows`` = 128: each matrix of ``x``
    [..., rows, columns] in blocks of 128 x 128, ``scale`` [..., ceil(rows /
    128), ceil(columns / 128)]. No gradient."""
    return _lib.torch_ops().quantize_blocks(x, rows)


def fp8_matmul(a: torch.Tensor, b: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor, *,
               bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``values(a) @ values(b).T + bias`` in ``out_dtype``.

    ``a`` float8_e4m3fn [..., K] with ``a_scale`` [..., ceil(K / 128)], ``b``
    [N, K] with ``b_scale`` [ceil(N / 128), ceil(K / 128)], as
    ``quantize_blocks`` makes them with ``rows`` 1 and 128; ``bias`` [N] in bf16,
    fp16 or fp32. Rows have unit column stride and are evenly spaced in memory,
    K to 2^23 elements apart, at any alignment. Results are bf16, fp16 or fp32: the
    bias is added to the sum in fp32 and the result rounded once. Only fp32 results
    are summed in fp32 throughout; for bf16 and fp16 products more than 13 bits below
    their largest neighbour are cut (above: at most 8.5e-4, typically 1.4e-5 of the
    sum). A NaN scale makes its row's outputs NaN (``a``) or those of its 128
    channels (``b``). No gradient.
    """
    return _lib.torch_ops().fp8_matmul(a, b, a_scale, b_scale, bias, out_dtype)


def fp8_linear(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """``x @ weight.T`` in ``x.dtype`` with all three products of a training step in E4M3.

    ``x`` [..., K] and ``weight`` [N, K] in bf16, fp16 or fp32 (each its own),
    unit column stride and evenly spaced rows; K, N and the number of rows at
    most 2^23. With Q1 the blocks of 128 columns and Q128 those of 128 x 128::

        y  = Q1(x) Q128(weight)^T
        dx = Q1(dy) Q128(weight)
        dweight = Q1(dy^T) Q128(Q1(x))      (blocks along the rows of x)

    Each is rounded once, ``dweight`` to the weight's type, and summed as
    ``fp8_matmul`` sums for that type: in fp32 throughout where it is fp32, otherwise
    with products more than 13 bits below their largest neighbour cut. For the
    backward ``x`` is kept in E4M3 (one byte a value and one for 128) and the
    weight's transpose likewise; both may change after the call. A row of ``y``
    and of ``dx`` depends on its own row of ``x`` and ``dy`` only. Differentiable
    once. A captured backward raises while a graph built on the default stream
    still uses the same leaves.
    """
    return _lib.torch_ops().fp8_linear(x, weight)


@dataclass(frozen=True)
class Fp8Experts:
    """Expert weights in E4M3 with a scale for each 128 x 128.

    ``gate_up`` [E, 2I, H] (gate rows, then up rows) with ``gate_up_scale``
    [E, 2I / 128, H / 128]; ``down`` [E, H, I] with ``down_scale`` [E, H / 128,
    I / 128]; all contiguous, on one device, H and I multiples of 128.
    ``quantize`` makes them from the layer's weights.
    """

    gate_up: torch.Tensor
    gate_up_scale: torch.Tensor
    down: torch.Tensor
    down_scale: torch.Tensor

    def __post_init__(self):
        if self.gate_up.dim() != 3 or self.down.dim() != 3:
            raise ValueError("gate_up must have shape [E, 2I, H] and down [E, H, I]")
        experts, two_inter, hidden = self.gate_up.shape
        if experts < 1 or two_inter < 1 or two_inter % (2 * BLOCK) or hidden < 1 or hidden % BLOCK:
            raise ValueError(f"gate_up must have shape [E, 2I, H] with I and H multiples of {BLOCK}, "
                             f"got {tuple(self.gate_up.shape)}")
        inter = two_inter // 2
        for name, dtype, shape in (
                ("gate_up", torch.float8_e4m3fn, (experts, two_inter, hidden)),
                ("gate_up_scale", torch.float8_e8m0fnu, (experts, two_inter // BLOCK, hidden // BLOCK)),
                ("down", torch.float8_e4m3fn, (experts, hidden, inter)),
                ("down_scale", torch.float8_e8m0fnu, (experts, hidden // BLOCK, inter // BLOCK))):
            t = getattr(self, name)
            if t.dtype != dtype:
                raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
            if tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous with shape {shape}, got {tuple(t.shape)}")
            if t.device != self.gate_up.device:
                raise ValueError("the expert weights and scales must be on one device")

    @classmethod
    @torch.no_grad()
    def quantize(cls, gate_up_weight: torch.Tensor, down_weight: torch.Tensor) -> "Fp8Experts":
        """From the layer's weights: ``gate_up_weight`` [E, H, 2I] and
        ``down_weight`` [E, H, I] (any strides)."""
        if gate_up_weight.dim() != 3 or down_weight.dim() != 3:
            raise ValueError("gate_up_weight must have shape [E, H, 2I] and down_weight [E, H, I]")
        experts, hidden, two_inter = gate_up_weight.shape
        if tuple(down_weight.shape) != (experts, hidden, two_inter // 2) or two_inter % 2:
            raise ValueError(f"down_weight must have shape {(experts, hidden, two_inter // 2)}, "
                             f"got {tuple(down_weight.shape)}")
        if hidden % BLOCK or two_inter % (2 * BLOCK):
            raise ValueError(f"hidden and inter must be multiples of {BLOCK}")
        made = []
        for table in (gate_up_weight.transpose(1, 2), down_weight):
            rows, cols = table.shape[1:]
            q = torch.empty(experts, rows, cols, dtype=torch.float8_e4m3fn, device=table.device)
            scale = torch.empty(experts, rows // BLOCK, cols // BLOCK, dtype=torch.float8_e8m0fnu, device=table.device)
            for e in range(experts):  # one expert's contiguous copy at a time
                part, part_scale = quantize_blocks(table[e].contiguous(), rows=BLOCK)
                q[e].view(torch.uint8).copy_(part.view(torch.uint8))
                scale[e].view(torch.uint8).copy_(part_scale.view(torch.uint8))
            made += [q, scale]
        return cls(*made)


__all__ = ["Fp8Experts", "fp8_linear", "fp8_matmul", "quantize_blocks"]
