"""forward_few and forward_few_int8 have no backward: an operand that asks for a
gradient, or carries a tangent, is refused before any device call (a result
without one would end training silently). CPU tensors serve."""

import os

import pytest
import torch
import torch.autograd.forward_ad as fwd

import mega_moe
from mega_moe import _lib

BF, I8 = torch.bfloat16, torch.int8
pytestmark = pytest.mark.skipif(not os.path.exists(_lib.library_path()), reason="libmegamoe.so not built")


def _bf16_args(dev="cpu"):
    return dict(hidden_states=torch.zeros(2, 128, dtype=BF, device=dev),
                selected_experts=torch.zeros(2, 2, dtype=torch.int32, device=dev),
                gate_up_weight=torch.zeros(4, 128, 256, dtype=BF, device=dev),
                down_weight=torch.zeros(4, 128, 128, dtype=BF, device=dev), routing_weights=torch.ones(2, 2, device=dev))


def _int8_args(dev="cpu"):
    experts = dict(gate_up=torch.zeros(4, 256, 128, dtype=I8, device=dev), gate_up_scale=torch.ones(4, 256, device=dev),
                   down=torch.zeros(4, 128, 128, dtype=I8, device=dev), down_scale=torch.ones(4, 128, device=dev))
    return dict(tokens=torch.zeros(2, 128, dtype=I8, device=dev), token_scale=torch.ones(2, device=dev),
                selected_experts=torch.zeros(2, 2, dtype=torch.int32, device=dev),
                routing_weights=torch.ones(2, 2, device=dev)), experts


def _operator():
    return mega_moe.FusedMoEForward(None, max_tokens_per_rank=8, hidden_size=128, top_k=2, num_experts=4)


def _int8(args, experts):
    return _operator().forward_few_int8(**args, experts=mega_moe.Int8Experts(**experts))


@pytest.mark.parametrize("name", ["hidden_states", "gate_up_weight", "down_weight", "routing_weights"])
def test_bf16_operands(name):
    args = _bf16_args()
    args[name].requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        _operator().forward_few(**args)
    with torch.no_grad(), pytest.raises(ValueError, match="HIP device"):  # not for its gradient
        _operator().forward_few(**args)
    args[name].requires_grad_(False)
    with fwd.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        args[name] = fwd.make_dual(args[name], torch.ones_like(args[name]))
        _operator().forward_few(**args)


@pytest.mark.parametrize("name", ["token_scale", "routing_weights", "gate_up_scale", "down_scale"])
def test_int8_operands(name):
    args, experts = _int8_args()
    where = args if name in args else experts
    where[name].requires_grad_()
    with pytest.raises(ValueError, match="no gradient"):
        _int8(args, experts)
    with torch.no_grad(), pytest.raises(ValueError, match="HIP device"):
        _int8(args, experts)
    where[name].requires_grad_(False)
    with fwd.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        where[name] = fwd.make_dual(where[name], torch.ones_like(where[name]))
        _int8(args, experts)


@pytest.mark.gpu
def test_parameters_serve_without_a_gradient():
    """A model's parameters under no_grad and inference_mode, and refused outside."""
    args = _bf16_args("cuda")
    for name in ("gate_up_weight", "down_weight"):
        args[name] = torch.nn.Parameter(args[name])
    op = _operator()
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            assert not op.forward_few(**args).any()
    with pytest.raises(ValueError, match="no gradient"):
        op.forward_few(**args)
    small, experts = _int8_args("cuda")
    small["routing_weights"].requires_grad_()
    with torch.no_grad():
        assert not _int8(small, experts).any()
    with pytest.raises(ValueError, match="no gradient"):
        _int8(small, experts)
