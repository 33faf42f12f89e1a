"""Argument checks of the norm, the 8-bit product and the few-token layer.

They run on the host before any device call, so CPU tensors serve: an operand
that passes every other check is refused for its device. The C entry points'
own checks are called with addresses that are never read."""

import ctypes
import os

import pytest
import torch

import mega_moe
from mega_moe import _lib

BF, F32, I8 = torch.bfloat16, torch.float32, torch.int8
built = pytest.mark.skipif(not os.path.exists(_lib.library_path()), reason="libmegamoe.so not built")


@pytest.mark.parametrize("kw,err", [
    (dict(x=torch.zeros(2, 8, dtype=torch.float64)), TypeError),
    (dict(x=torch.zeros(2, 8, dtype=I8)), TypeError),
    (dict(x=torch.zeros((), dtype=BF)), ValueError),
    (dict(x=torch.zeros(2, 0, dtype=BF)), ValueError),
    (dict(x=torch.zeros(1, 32769, dtype=BF)), ValueError),
    (dict(weight=torch.ones(7, dtype=BF)), ValueError),
    (dict(weight=torch.ones(1, 8, dtype=BF)), ValueError),
    (dict(weight=torch.ones(16, dtype=BF)[::2]), ValueError),
    (dict(weight=torch.ones(8, dtype=torch.float64)), TypeError),
    (dict(residual=torch.zeros(2, 7, dtype=BF)), ValueError),
    (dict(residual=torch.zeros(1, 8, dtype=BF)), ValueError),
    (dict(residual=torch.zeros(2, 8, dtype=torch.float16)), TypeError),
    (dict(x=torch.zeros(2, 8), residual=torch.zeros(2, 8, dtype=BF)), TypeError),
    (dict(eps=-1e-6), ValueError),
    (dict(eps=float("nan")), ValueError),
    (dict(out_dtype=F32), TypeError),
    (dict(out_dtype=torch.uint8), TypeError),
    (dict(out_dtype=I8, x=torch.zeros(2, 8, dtype=BF, requires_grad=True)), ValueError),
    (dict(out_dtype=I8, weight=torch.ones(8, dtype=BF, requires_grad=True)), ValueError),
    (dict(), ValueError),  # a CPU tensor
])
def test_rms_norm_refuses(kw, err):
    args = dict(x=torch.zeros(2, 8, dtype=BF))
    args.update(kw)
    with pytest.raises(err):
        mega_moe.rms_norm(args.pop("x"), args.pop("weight", None), **args)


@pytest.mark.parametrize("x,dtype,err", [
    (torch.zeros(2, 8, dtype=I8), I8, TypeError),
    (torch.zeros(2, 8, dtype=BF), BF, TypeError),
    (torch.zeros((), dtype=BF), I8, ValueError),
    (torch.zeros(2, 8, dtype=BF, requires_grad=True), I8, ValueError),
    (torch.zeros(2, 8, dtype=BF), I8, ValueError),
])
def test_quantize_rows_refuses(x, dtype, err):
    with pytest.raises(err):
        mega_moe.quantize_rows(x, dtype)


@pytest.mark.parametrize("kw,err", [
    (dict(a=torch.zeros(2, 16)), TypeError),
    (dict(b=torch.zeros(3, 16)), TypeError),
    (dict(a=torch.zeros(2, 15, dtype=I8)), ValueError),
    (dict(b=torch.zeros(3, 16, 1, dtype=I8)), ValueError),
    (dict(a=torch.zeros(2, 0, dtype=I8), b=torch.zeros(3, 0, dtype=I8)), ValueError),
    (dict(a=torch.zeros(2, 1 << 17, dtype=I8), b=torch.zeros(3, 1 << 17, dtype=I8)), ValueError),
    (dict(b=torch.zeros(16, 3, dtype=I8).t()), ValueError),
    (dict(b=torch.zeros(1, 16, dtype=I8).expand(3, 16)), ValueError),
    (dict(b=torch.zeros(0, 16, dtype=I8), b_scale=torch.ones(0)), ValueError),
    (dict(a_scale=torch.ones(3)), ValueError),
    (dict(a_scale=torch.ones(2, 1)), ValueError),
    (dict(a_scale=torch.ones(2, dtype=BF)), TypeError),
    (dict(b_scale=torch.ones(6)[::2]), ValueError),
    (dict(b_scale=torch.ones(3, requires_grad=True)), ValueError),
    (dict(bias=torch.ones(2)), ValueError),
    (dict(bias=torch.ones(3, dtype=torch.int32)), TypeError),
    (dict(out_dtype=torch.int32), TypeError),
    (dict(), ValueError),  # CPU tensors
])
def test_int8_matmul_refuses(kw, err):
    args = dict(a=torch.zeros(2, 16, dtype=I8), b=torch.zeros(3, 16, dtype=I8), a_scale=torch.ones(2),
                b_scale=torch.ones(3))
    args.update(kw)
    with pytest.raises(err):
        mega_moe.int8_matmul(args.pop("a"), args.pop("b"), args.pop("a_scale"), args.pop("b_scale"), **args)


@pytest.mark.parametrize("kw,err", [
    (dict(gate_up=torch.zeros(2, 256, 128)), TypeError),
    (dict(gate_up=torch.zeros(256, 128, dtype=I8)), ValueError),
    (dict(gate_up=torch.zeros(2, 255, 128, dtype=I8)), ValueError),
    (dict(gate_up=torch.zeros(2, 128, 256, dtype=I8).transpose(1, 2)), ValueError),
    (dict(gate_up_scale=torch.ones(2, 128)), ValueError),
    (dict(gate_up_scale=torch.ones(2, 256, dtype=BF)), TypeError),
    (dict(down=torch.zeros(2, 128, 127, dtype=I8)), ValueError),
    (dict(down_scale=torch.ones(128, 2).t()), ValueError),
])
def test_int8_experts_refuse(kw, err):
    args = dict(gate_up=torch.zeros(2, 256, 128, dtype=I8), gate_up_scale=torch.ones(2, 256),
                down=torch.zeros(2, 128, 128, dtype=I8), down_scale=torch.ones(2, 128))
    mega_moe.Int8Experts(**args)
    args.update(kw)
    with pytest.raises(err):
        mega_moe.Int8Experts(**args)


def test_int8_experts_quantize_refuses():
    with pytest.raises(ValueError, match="down_weight"):
        mega_moe.Int8Experts.quantize(torch.zeros(2, 128, 256), torch.zeros(2, 128, 256))
    with pytest.raises(ValueError):
        mega_moe.Int8Experts.quantize(torch.zeros(128, 256), torch.zeros(2, 128, 128))


def test_few_refuses_cpu_tensors():
    op = mega_moe.FusedMoEForward(None, max_tokens_per_rank=8, hidden_size=128, top_k=2, num_experts=4)
    sel, w = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, 2)
    with pytest.raises(ValueError, match="HIP device"):
        op.forward_few(torch.zeros(2, 128, dtype=BF), sel, torch.zeros(4, 128, 256, dtype=BF),
                       torch.zeros(4, 128, 128, dtype=BF), w)
    experts = mega_moe.Int8Experts(torch.zeros(4, 256, 128, dtype=I8), torch.ones(4, 256),
                                   torch.zeros(4, 128, 128, dtype=I8), torch.ones(4, 128))
    with pytest.raises(ValueError, match="HIP device"):
        op.forward_few_int8(torch.zeros(2, 128, dtype=I8), torch.ones(2), sel, experts, w)


FAKE = ctypes.c_void_p(1 << 20)


@built
@pytest.mark.parametrize("rows,hidden,xt,ht,yt", [
    (-1, 8, 0, 0, 0), (1 << 31, 8, 0, 0, 0), (1, 0, 0, 0, 0), (1, 32769, 0, 0, 0),
    (1, 8, 3, 3, 3), (1, 8, 0, 1, 0), (1, 8, 2, 0, 2), (1, 8, 0, 0, 1), (1, 8, 0, 0, 5), (1, 8, 5, 5, 5),
])
def test_norm_entry_refuses(rows, hidden, xt, ht, yt):
    lib = _lib.load()
    assert lib.mm_rms_norm(FAKE, 8, xt, FAKE, 8, ht, None, 0, rows, hidden, 1e-6, FAKE, FAKE, yt, FAKE, None, None) == -1
    assert b"mm_rms_norm" in lib.mm_last_error()


@built
def test_norm_entry_refuses_null_and_small_workspaces():
    lib = _lib.load()
    assert lib.mm_rms_norm(None, 8, 0, None, 0, 0, None, 0, 1, 8, 1e-6, None, FAKE, 0, None, None, None) == -1
    assert lib.mm_rms_norm(FAKE, 8, 0, FAKE, 8, 0, None, 0, 1, 8, 1e-6, None, FAKE, 0, None, None, None) == -1
    assert lib.mm_rms_norm(FAKE, 8, 0, None, 0, 0, None, 0, 1, 8, 1e-6, None, FAKE, 3, None, None, None) == -1
    assert lib.mm_quantize_rows(FAKE, 8, 0, 1, 8, FAKE, 0, FAKE, None) == -1
    assert lib.mm_quantize_rows(FAKE, 8, 0, 1, 8, FAKE, 3, None, None) == -1
    need = lib.mm_rms_norm_bwd_workspace_bytes(100, 2048)
    assert need >= 2048 * 4
    rc = lib.mm_rms_norm_bwd(FAKE, 2048, None, 0, FAKE, 2048, FAKE, 0, FAKE, 0, 0, 100, 2048, FAKE, None, FAKE, FAKE,
                             need - 1, None)
    assert rc == -2 and b"workspace" in lib.mm_last_error()
    assert lib.mm_rms_norm_bwd_workspace_bytes(1, 32769) == 0


@built
@pytest.mark.parametrize("m,n,k,lda,ldb,ldo,ot", [
    (-1, 8, 8, 8, 8, 8, 0), (8, 0, 8, 8, 8, 8, 0), (8, 8, 0, 8, 8, 8, 0), (8, 8, 1 << 17, 1 << 17, 1 << 17, 8, 0),
    (8, 8, 8, 7, 8, 8, 0), (8, 8, 8, 8, 7, 8, 0), (8, 8, 8, 8, 8, 7, 0), (8, 8, 8, 8, 8, 8, 3),
    ((1 << 31) - 1, 8, 8, 8, 8, 8, 0), ((1 << 31) - 512 - 1, (1 << 31) - 512 - 1, 8, 8, 8, 1 << 31, 0),
])
def test_int8_entry_refuses(m, n, k, lda, ldb, ldo, ot):
    lib = _lib.load()
    assert lib.mm_int8_matmul(FAKE, lda, FAKE, ldb, FAKE, FAKE, None, 0, m, n, k, FAKE, ldo, ot, None) == -1
    assert b"mm_int8_matmul" in lib.mm_last_error()


@built
@pytest.mark.parametrize("tokens,k,E,H,I,act", [
    (65, 1, 8, 128, 128, 0), (-1, 1, 8, 128, 128, 0), (1, 65, 8, 128, 128, 0), (1, 1, 0, 128, 128, 0),
    (1, 1, 32769, 128, 128, 0), (1, 1, 8, 64, 128, 0), (1, 1, 8, 128, 192, 0), (1, 1, 8, 128, 128, 3),
])
def test_few_entry_refuses(tokens, k, E, H, I, act):
    lib = _lib.load()
    big = 1 << 40
    rc = lib.mm_moe_few(FAKE, FAKE, FAKE, FAKE, FAKE, H * I, I, 1, tokens, k, E, H, I, act, 1.0, 0.0, 7.0, FAKE, FAKE,
                        big, None)
    assert rc == -1 and b"mm_moe_few" in lib.mm_last_error()
    rc = lib.mm_moe_few_int8(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, tokens, k, E, H, I, act, 1.0, 0.0, 7.0,
                             FAKE, FAKE, big, None)
    assert rc == -1 and b"mm_moe_few_int8" in lib.mm_last_error()


@built
def test_few_entry_refuses_strides_and_small_scratch():
    lib = _lib.load()
    tail = (1, 1, 8, 128, 128, 0, 1.0, 0.0, 7.0, FAKE, FAKE)
    assert lib.mm_moe_few(FAKE, FAKE, FAKE, FAKE, FAKE, 128 * 256, 256, 2, *tail, 1 << 40, None) == -1
    for int8 in (0, 1):
        assert lib.mm_moe_few_scratch_bytes(65, 1, 128, 128, int8) == 0
        assert lib.mm_moe_few_scratch_bytes(1, 1, 64, 128, int8) == 0
    need = lib.mm_moe_few_scratch_bytes(1, 1, 128, 128, 0)
    assert lib.mm_moe_few(FAKE, FAKE, FAKE, FAKE, FAKE, 128 * 128, 128, 1, *tail, need - 1, None) == -2
    assert b"scratch" in lib.mm_last_error()
    need = lib.mm_moe_few_scratch_bytes(1, 1, 128, 128, 1)
    assert lib.mm_moe_few_int8(*[FAKE] * 8, *tail, need - 1, None) == -2


@built
def test_an_operator_can_be_copied_and_pickled():
    """The native description of the few-token layer travels with the operator."""
    import copy
    import pickle

    op = mega_moe.FusedMoEForward(None, max_tokens_per_rank=8, hidden_size=128, top_k=2, num_experts=4)
    op._few_layer(torch.zeros(1, 128))
    assert op._few is not None
    for other in (copy.deepcopy(op), pickle.loads(pickle.dumps(op))):
        assert other.top_k == 2 and other._few is not None and other._few is not op._few


@built
@pytest.mark.parametrize("call", [
    lambda x: mega_moe.rms_norm(x),
    lambda x: mega_moe.rms_norm(torch.zeros_like(x), x[0]),
    lambda x: mega_moe.rms_norm(torch.zeros_like(x), residual=x),
    lambda x: mega_moe.rms_norm(x, out_dtype=I8),
    lambda x: mega_moe.quantize_rows(x),
    lambda x: mega_moe.int8_matmul(torch.zeros(2, 8, dtype=I8), torch.zeros(2, 8, dtype=I8), x[:, 0].clone(), torch.ones(2)),
    lambda x: mega_moe.int8_matmul(torch.zeros(2, 8, dtype=I8), torch.zeros(2, 8, dtype=I8), torch.ones(2), torch.ones(2),
                                   bias=x[:, 0].clone()),
])
def test_forward_mode_tangents_are_refused(call):
    """A tangent would be lost: no operator here has a forward-mode derivative."""
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        call(fwd.make_dual(torch.ones(2, 8), torch.ones(2, 8)))
