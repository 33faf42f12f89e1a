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

from . import _kernels as K
from .norm import MAX_HIDDEN, quantize_rows

MAX_STRIDE = 1 << 23  # of a row, 256 of which a kernel's offsets have to span
MAX_K = (1 << 17) - 1  # the int32 sum is exact below 2^17 products of two int8 values
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


def int8_matmul(a: torch.Tensor, b: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor, *,
                bias: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``(a * a_scale[..., None]) @ (b * b_scale[:, None]).T + bias`` in ``out_dtype``.

    ``a`` int8 [..., K] (rows evenly spaced in memory, unit column stride) with
    fp32 ``a_scale`` of ``a``'s leading shape, one a token; ``b`` int8 [N, K]
    (unit column stride, rows up to 2^23 elements apart, as ``a``'s) with fp32 ``b_scale`` [N], one a
    channel; ``bias`` [N] in bf16, fp16 or fp32. 1 <= K < 2^17: the sum is exact
    in int32; scales and bias are applied in fp32 and the result is rounded
    once to bf16, fp16 or fp32. No gradient.
    """
    if a.dtype != torch.int8 or b.dtype != torch.int8:
        raise TypeError(f"a and b must be torch.int8, got {a.dtype} and {b.dtype}")
    if a.dim() == 0 or b.dim() != 2:
        raise ValueError(f"a must have shape [..., K] and b [N, K], got {tuple(a.shape)} and {tuple(b.shape)}")
    n, k = b.shape
    if a.shape[-1] != k:
        raise ValueError(f"a has {a.shape[-1]} columns, b has {k}")
    if not 1 <= k <= MAX_K or n < 1:
        raise ValueError(f"b must have shape [N, K] with N >= 1 and 1 <= K <= {MAX_K}, got {tuple(b.shape)}")
    ldb, step = b.stride()
    if k > 1 and step != 1:
        raise ValueError("b must have unit column stride ([N, K], K contiguous)")
    if n > 1 and not k <= ldb <= MAX_STRIDE:
        raise ValueError(f"the rows of b must be {k} to {MAX_STRIDE} elements apart (no overlap), got {ldb}")
    if a_scale.dtype != torch.float32 or b_scale.dtype != torch.float32:
        raise TypeError(f"a_scale and b_scale must be torch.float32, got {a_scale.dtype} and {b_scale.dtype}")
    if a_scale.shape != a.shape[:-1] or not a_scale.is_contiguous():
        raise ValueError(f"a_scale must be contiguous with shape {tuple(a.shape[:-1])}, got {tuple(a_scale.shape)}")
    if b_scale.dim() != 1 or b_scale.shape[0] != n or not b_scale.is_contiguous():
        raise ValueError(f"b_scale must be contiguous with shape ({n},), got {tuple(b_scale.shape)}")
    if bias is not None:
        if bias.dtype not in _FLOATS:
            raise TypeError(f"bias must be bfloat16, float16 or float32, got {bias.dtype}")
        if bias.dim() != 1 or bias.shape[0] != n or not bias.is_contiguous():
            raise ValueError(f"bias must be contiguous with shape ({n},), got {tuple(bias.shape)}")
    device = a.device
    if b.device != device or a_scale.device != device or b_scale.device != device or (
            bias is not None and bias.device != device):
        raise ValueError("all operands must be on the device of a")
    if out_dtype not in _FLOATS:
        raise TypeError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
    if (a_scale.requires_grad or b_scale.requires_grad or (bias is not None and bias.requires_grad)) \
            and torch.is_grad_enabled():
        raise ValueError("int8_matmul carries no gradient; call under torch.no_grad() or on detached operands")
    if not a.is_cuda:
        raise ValueError("a must be a HIP device tensor")
    return K.int8_matmul(a, b, a_scale, b_scale, bias, out_dtype)


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
