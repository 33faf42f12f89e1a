"""MI355X-native Mega-MoE: public API (names of src/mega_moe/__init__.py:1-27),
with the norm in front of the layer and the 8-bit products next to it."""

from .config import MoEForwardConfig
from .ops.backward import MegaMoEBackwardFunction, moe_backward_triton
from .ops.forward import DispatchFC1Result, FusedMoEForward, pack_gate_up_weights
from .ops.fp8 import Fp8Experts, fp8_linear, fp8_matmul, quantize_blocks
from .ops.function import MegaMoEFunction
from .ops.int8 import Int8Experts, int8_matmul
from .ops.norm import quantize_rows, rms_norm
from .runtime.routing import MoERoutingPlan

__all__ = [
    "FusedMoEForward",
    "DispatchFC1Result",
    "pack_gate_up_weights",
    "MegaMoEBackwardFunction",
    "MegaMoEFunction",
    "moe_backward_triton",
    "MoEForwardConfig",
    "MoERoutingPlan",
    "Fp8Experts",
    "Int8Experts",
    "fp8_linear",
    "fp8_matmul",
    "int8_matmul",
    "quantize_blocks",
    "quantize_rows",
    "rms_norm",
]
