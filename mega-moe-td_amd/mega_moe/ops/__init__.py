"""Operator layer: forward, five-stage backward, autograd entry, norm, 8-bit products."""

from .backward import MegaMoEBackwardFunction, moe_backward_triton
from .forward import DispatchFC1Result, FusedMoEForward, pack_gate_up_weights
from .function import MegaMoEFunction
from .int8 import Int8Experts, int8_matmul
from .norm import quantize_rows, rms_norm

__all__ = [
    "DispatchFC1Result",
    "FusedMoEForward",
    "Int8Experts",
    "MegaMoEBackwardFunction",
    "MegaMoEFunction",
    "int8_matmul",
    "moe_backward_triton",
    "pack_gate_up_weights",
    "quantize_rows",
    "rms_norm",
]
