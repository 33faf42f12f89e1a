"""Products of 8-bit integer rows, and the experts in 8 bits.

``int8_matmul`` is the dense product next to the layer (a shared expert, the
projections around it) on the rows that ``rms_norm`` and ``quantize_rows``
make; ``Int8Experts`` holds the layer's expert weights for
``FusedMoEForward.forward_few_int8``. The reference has no 8-bit products.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .. import _lib
from .norm import MAX_HIDDEN, quantize_rows


def int8_matmul(a: torch.Tensor, b: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor, *,
                bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(a * a_scale[..., None]) @ (b * b_scale[:, None]).T + bias`` in ``out_dtype``.

    ``a`` int8 [..., K] with fp32 ``a_scale`` of ``a``'s leading shape, one a
    token; ``b`` int8 [N, K] with fp32 ``b_scale`` [N], one a channel; ``bias``
    [N] in bf16, fp16 or fp32. Rows have unit column stride and are evenly
    spaced in memory, K to 2^23 elements apart. 1 <= K < 2^17: the sum is exact
    in int32; scales and bias are applied in fp32 and the result is rounded
    once to bf16, fp16 or fp32. No gradient.
    """
    return _lib.torch_ops().int8_matmul(a, b, a_scale, b_scale, bias, out_dtype)


@dataclass(frozen=True)
class Int8Experts:
    """Expert weights in int8 with one fp32 scale for each output channel.

    ``gate_up`` [E, 2I, H] (gate rows, then up rows) with ``gate_up_scale``
    [E, 2I]; ``down`` [E, H, I] with ``down_scale`` [E, H]; all contiguous, on
    one device. ``quantize`` makes them from the layer's bf16 weights.
    """

    gate_up: torch.Tensor
    gate_up_scale: torch.Tensor
    down: torch.Tensor
    down_scale: torch.Tensor

    def __post_init__(self):
        if self.gate_up.dim() != 3 or self.down.dim() != 3:
            raise ValueError("gate_up must have shape [E, 2I, H] and down [E, H, I]")
        experts, two_inter, hidden = self.gate_up.shape
        if experts < 1 or two_inter < 2 or two_inter % 2 or hidden < 1:
            raise ValueError(f"gate_up must have shape [E, 2I, H], got {tuple(self.gate_up.shape)}")
        for name, dtype, shape in (("gate_up", torch.int8, (experts, two_inter, hidden)),
                                   ("gate_up_scale", torch.float32, (experts, two_inter)),
                                   ("down", torch.int8, (experts, hidden, two_inter // 2)),
                                   ("down_scale", torch.float32, (experts, hidden))):
            t = getattr(self, name)
            if t.dtype != dtype:
                raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
            if tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous with shape {shape}, got {tuple(t.shape)}")
            if t.device != self.gate_up.device:
                raise ValueError("the expert weights and scales must be on one device")

    @classmethod
    @torch.no_grad()
    def quantize(cls, gate_up_weight: torch.Tensor, down_weight: torch.Tensor) -> "Int8Experts":
        """From the layer's weights: ``gate_up_weight`` [E, H, 2I] and
        ``down_weight`` [E, H, I] (any strides), one channel's largest value to 127."""
        if gate_up_weight.dim() != 3 or down_weight.dim() != 3:
            raise ValueError("gate_up_weight must have shape [E, H, 2I] and down_weight [E, H, I]")
        experts, hidden, two_inter = gate_up_weight.shape
        if tuple(down_weight.shape) != (experts, hidden, two_inter // 2) or two_inter % 2:
            raise ValueError(f"down_weight must have shape {(experts, hidden, two_inter // 2)}, "
                             f"got {tuple(down_weight.shape)}")
        if max(hidden, two_inter // 2) > MAX_HIDDEN:
            raise ValueError(f"hidden and inter must be at most {MAX_HIDDEN}")
        dev = gate_up_weight.device
        out = cls(torch.empty(experts, two_inter, hidden, dtype=torch.int8, device=dev),
                  torch.empty(experts, two_inter, dtype=torch.float32, device=dev),
                  torch.empty(experts, hidden, two_inter // 2, dtype=torch.int8, device=dev),
                  torch.empty(experts, hidden, dtype=torch.float32, device=dev))
        for e in range(experts):  # one expert's transposed copy at a time
            for q, scale, w in ((out.gate_up, out.gate_up_scale, gate_up_weight[e].t()),
                                (out.down, out.down_scale, down_weight[e])):
                rows, row_scale = quantize_rows(w.contiguous())
                q[e].copy_(rows)
                scale[e].copy_(row_scale)
        return out


__all__ = ["Int8Experts", "int8_matmul"]
