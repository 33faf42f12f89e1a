"""The int8 few-token layer sums ``hidden`` products of -128 * -128 in int32: it
takes rows below 2^17 columns, as int8_matmul does, and refuses wider ones."""

import ctypes
import os

import pytest
import torch

import mega_moe
from mega_moe import _lib

I8 = torch.int8
built = pytest.mark.skipif(not os.path.exists(_lib.library_path()), reason="libmegamoe.so not built")
FAKE = ctypes.c_void_p(1 << 20)


@built
@pytest.mark.parametrize("hidden", [1 << 17, (1 << 17) + 128, 1 << 20])
def test_entry_refuses_sums_past_int32(hidden):
    lib = _lib.load()
    assert lib.mm_moe_few_scratch_bytes(1, 1, hidden, 128, 1) == 0
    assert lib.mm_moe_few_scratch_bytes(1, 1, hidden, 128, 0) > 0  # bf16 sums are fp32
    assert lib.mm_moe_few_scratch_bytes(1, 1, (1 << 17) - 128, 128, 1) > 0
    # refused by its sizes before the address of the scratch (none) counts
    rc = lib.mm_moe_few_int8(*[FAKE] * 8, 1, 1, 1, hidden, 128, 0, 1.0, 0.0, 7.0, FAKE, None, 1 << 40, None)
    assert rc == -1 and b"sizes" in lib.mm_last_error()


@pytest.mark.gpu
def test_operator_refuses_sums_past_int32():
    hidden = 1 << 17
    op = mega_moe.FusedMoEForward(None, max_tokens_per_rank=1, hidden_size=hidden, top_k=1, num_experts=1)
    full = lambda *s: torch.full(s, -128, dtype=I8, device="cuda")
    ex = mega_moe.Int8Experts(full(1, 256, hidden), torch.full((1, 256), 1e-6, device="cuda"), full(1, hidden, 128),
                              torch.full((1, hidden), 1e-3, device="cuda"))
    one = torch.ones(1, 1, device="cuda")
    with pytest.raises(ValueError, match="131072"):
        op.forward_few_int8(full(1, hidden), torch.ones(1, device="cuda"), one.int() - 1, ex, one)


@pytest.mark.gpu
def test_the_widest_row_is_exact():
    """2^17 - 128 columns of -128: the sums are 2^31 - 2^21."""
    hidden, inter = (1 << 17) - 128, 128
    op = mega_moe.FusedMoEForward(None, max_tokens_per_rank=1, hidden_size=hidden, top_k=1, num_experts=1)
    full = lambda *s: torch.full(s, -128, dtype=I8, device="cuda")
    down = torch.zeros(1, hidden, inter, dtype=I8, device="cuda")
    down[0, :, 0] = 1
    ex = mega_moe.Int8Experts(full(1, 2 * inter, hidden), torch.full((1, 2 * inter), 2.0**-30, device="cuda"), down,
                              torch.ones(1, hidden, device="cuda"))
    one = torch.ones(1, 1, device="cuda")
    out = op.forward_few_int8(full(1, hidden), torch.ones(1, device="cuda"), one.int() - 1, ex, one).double()
    pre = (2.0**31 - 2.0**21) * 2.0**-30
    want = pre * pre / (1 + 2.718281828459045**-pre)
    # the quantised activation is the group's largest value; one rounding to bf16
    assert ((out - want).abs() <= want * (2**-8 + 2**-14)).all()
