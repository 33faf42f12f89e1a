"""Operator layer: forward, five-stage backward, autograd entry, norm, 8-bit products."""

from .backward import MegaMoEBackwardFunction, moe_backward_triton
from .forward import DispatchFC1Result, FusedMoEForward, pack_gate_up_weights
from .fp8 import Fp8Experts, fp8_linear, fp8_matmul, quantize_blocks
from .function import MegaMoEFunction
from .int8 import Int8Experts, int8_matmul
from .norm import quantize_rows, rms_norm

__all__ = [
    "DispatchFC1Result",
    "FusedMoEForward",
    "Fp8Experts",
    "Int8Experts",
    "MegaMoEBackwardFunction",
    "MegaMoEFunction",
    "fp8_linear",
    "fp8_matmul",
    "int8_matmul",
    "moe_backward_triton",
    "pack_gate_up_weights",
    "quantize_blocks",
    "quantize_rows",
    "rms_norm",
]
