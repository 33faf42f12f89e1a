"""Argument checks of the E4M3 products with a scale for each block of 128.

They run on the host before any device call, so CPU tensors serve: an operand
that passes every other check is refused for its device. The C entry points'
own checks are called with addresses that are never read."""

import ctypes
import os

import pytest
import torch

import mega_moe
from mega_moe import _lib

BF, F32, F64, F8, E8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn, torch.float8_e8m0fnu
built = pytest.mark.skipif(not os.path.exists(_lib.library_path()), reason="libmegamoe.so not built")


def f8(*sizes):
    return torch.zeros(*sizes, dtype=torch.uint8).view(F8)


def e8(*sizes):
    return torch.full(sizes, 127, dtype=torch.uint8).view(E8)


@pytest.mark.parametrize("x,rows,err,match", [
    (torch.zeros(2, 8, dtype=F64), 1, TypeError, "x must"),
    (f8(2, 8), 1, TypeError, "x must"),
    (torch.zeros((), dtype=BF), 1, ValueError, "columns"),
    (torch.zeros(8, dtype=BF), 128, ValueError, "rows, columns"),
    (torch.zeros(2, 8, dtype=BF), 2, ValueError, "1 or 128"),
    (torch.zeros(2, 8, dtype=BF), 0, ValueError, "1 or 128"),
    (torch.zeros(2, 8, requires_grad=True), 1, ValueError, "no gradient"),
    (torch.zeros(2, 8, requires_grad=True), 128, ValueError, "no gradient"),
    (torch.zeros(2, 8, dtype=BF), 1, ValueError, "HIP device"),
    (torch.zeros(3, 2, 8, dtype=BF), 128, ValueError, "HIP device"),
])
def test_quantize_blocks_refuses(x, rows, err, match):
    with pytest.raises(err, match=match):
        mega_moe.quantize_blocks(x, rows)


@pytest.mark.parametrize("kw,err,match", [
    (dict(a=torch.zeros(2, 160, dtype=BF)), TypeError, "float8_e4m3fn"),
    (dict(b=torch.zeros(3, 160, dtype=torch.int8)), TypeError, "float8_e4m3fn"),
    (dict(a=f8(2, 159)), ValueError, "columns"),
    (dict(a=torch.zeros((), dtype=torch.uint8).view(F8)), ValueError, "shape"),
    (dict(b=f8(3, 160, 1)), ValueError, "shape"),
    (dict(a=f8(2, 0), b=f8(3, 0)), ValueError, "K"),
    (dict(b=f8(0, 160), b_scale=e8(0, 2)), ValueError, "N >= 1"),
    (dict(b=f8(160, 3).t()), ValueError, "unit column stride"),
    (dict(b=f8(1, 160).expand(3, 160)), ValueError, "overlap"),
    (dict(a_scale=torch.ones(2, 2)), TypeError, "e8m0"),
    (dict(b_scale=torch.ones(1, 2)), TypeError, "e8m0"),
    (dict(a_scale=e8(2, 1)), ValueError, "a_scale"),
    (dict(a_scale=e8(1, 2)), ValueError, "a_scale"),
    (dict(a_scale=e8(2, 2).t()), ValueError, "a_scale"),
    (dict(b_scale=e8(3, 2)), ValueError, "b_scale"),
    (dict(b_scale=e8(1, 4)[:, ::2]), ValueError, "HIP device"),  # one row of two values is not contiguous
    (dict(b_scale=e8(2, 2)), ValueError, "b_scale"),
    (dict(bias=torch.ones(2)), ValueError, "bias"),
    (dict(bias=torch.ones(6)[::2]), ValueError, "bias"),
    (dict(bias=torch.ones(3, dtype=F64)), TypeError, "bias"),
    (dict(bias=torch.ones(3, requires_grad=True)), ValueError, "no gradient"),
    (dict(out_dtype=F8), TypeError, "out_dtype"),
    (dict(out_dtype=torch.int32), TypeError, "out_dtype"),
    (dict(), ValueError, "HIP device"),
])
def test_fp8_matmul_refuses(kw, err, match):
    if match == "HIP device" and kw:
        match = "b_scale"
    args = dict(a=f8(2, 160), b=f8(3, 160), a_scale=e8(2, 2), b_scale=e8(1, 2))
    args.update(kw)
    with pytest.raises(err, match=match):
        mega_moe.fp8_matmul(args.pop("a"), args.pop("b"), args.pop("a_scale"), args.pop("b_scale"), **args)


@pytest.mark.parametrize("x,w,err,match", [
    (torch.zeros(2, 8, dtype=F64), torch.zeros(3, 8), TypeError, "x must"),
    (torch.zeros(2, 8), f8(3, 8), TypeError, "weight must"),
    (torch.zeros(()), torch.zeros(3, 8), ValueError, "shape"),
    (torch.zeros(2, 8), torch.zeros(8), ValueError, "shape"),
    (torch.zeros(2, 7), torch.zeros(3, 8), ValueError, "columns"),
    (torch.zeros(2, 0), torch.zeros(3, 0), ValueError, "K from 1"),
    (torch.zeros(2, 8), torch.zeros(0, 8), ValueError, "N and K"),
    (torch.zeros(2, 8), torch.zeros(8, 3).t(), ValueError, "unit column stride"),
    (torch.zeros(1, 1).expand((1 << 23) + 1, 1), torch.zeros(1, 1), ValueError, "at most"),
    (torch.zeros(2, 8), torch.zeros(3, 8), ValueError, "HIP device"),
    (torch.zeros(2, 8, requires_grad=True), torch.zeros(3, 8, dtype=BF), ValueError, "HIP device"),
])
def test_fp8_linear_refuses(x, w, err, match):
    with pytest.raises(err, match=match):
        mega_moe.fp8_linear(x, w)


@pytest.mark.parametrize("kw,match", [
    (dict(scale_columns=64, out_dtype=F8), "scale_columns"),
    (dict(scale_columns=128), "scale_columns"),
    (dict(scale_columns=128, out_dtype=torch.int8), "scale_columns"),
    (dict(scale_columns=128, out_dtype=F8, weight=torch.ones(8, requires_grad=True)), "no gradient|gradient"),
    (dict(scale_columns=128, out_dtype=F8), "HIP device"),
])
def test_norm_to_blocks_refuses(kw, match):
    with pytest.raises(ValueError, match=match):
        mega_moe.rms_norm(torch.zeros(2, 8), **kw)


def experts(E=4, H=128, I=128):
    return dict(gate_up=f8(E, 2 * I, H), gate_up_scale=e8(E, 2 * I // 128, H // 128), down=f8(E, H, I),
                down_scale=e8(E, H // 128, I // 128))


@pytest.mark.parametrize("kw,err,match", [
    (dict(gate_up=torch.zeros(4, 256, 128)), TypeError, "gate_up"),
    (dict(gate_up=f8(256, 128)), ValueError, "gate_up"),
    (dict(gate_up=f8(4, 255, 128)), ValueError, "multiples"),
    (dict(gate_up=f8(4, 128, 128)), ValueError, "multiples"),
    (dict(gate_up=f8(4, 256, 100)), ValueError, "multiples"),
    (dict(gate_up=f8(0, 256, 128)), ValueError, "gate_up"),
    (dict(gate_up=f8(4, 128, 256).transpose(1, 2)), ValueError, "contiguous"),
    (dict(gate_up_scale=torch.ones(4, 2, 1)), TypeError, "gate_up_scale"),
    (dict(gate_up_scale=e8(4, 256, 1)), ValueError, "gate_up_scale"),
    (dict(down=f8(128, 128)), ValueError, "down"),
    (dict(down=f8(4, 128, 256)), ValueError, "down"),
    (dict(down_scale=e8(4, 2, 1)), ValueError, "down_scale"),
    (dict(down_scale=e8(4, 1, 1).to("meta")), ValueError, "one device"),
])
def test_experts_refuse(kw, err, match):
    args = experts()
    mega_moe.Fp8Experts(**args)
    args.update(kw)
    with pytest.raises(err, match=match):
        mega_moe.Fp8Experts(**args)


def test_experts_quantize_refuses():
    make = mega_moe.Fp8Experts.quantize
    for gate_up, down, match in (
            (torch.zeros(128, 256), torch.zeros(2, 128, 128), "gate_up_weight"),
            (torch.zeros(2, 128, 256), torch.zeros(2, 128, 256), "down_weight"),
            (torch.zeros(2, 128, 255), torch.zeros(2, 128, 127), "down_weight"),
            (torch.zeros(2, 100, 256), torch.zeros(2, 100, 128), "multiples"),
            (torch.zeros(2, 128, 128), torch.zeros(2, 128, 64), "multiples")):
        with pytest.raises(ValueError, match=match):
            make(gate_up, down)


@built
@pytest.mark.parametrize("kw,err,match", [
    (dict(experts=experts()), TypeError, "Fp8Experts"),
    (dict(routing_weights=torch.ones(2, 2, requires_grad=True)), ValueError, "gradient"),
    (dict(), ValueError, "HIP device"),
])
def test_layer_refuses(kw, err, match):
    op = mega_moe.FusedMoEForward(None, max_tokens_per_rank=8, hidden_size=128, top_k=2, num_experts=4)
    args = dict(tokens=f8(2, 128), token_scale=e8(2, 1), selected=torch.zeros(2, 2, dtype=torch.int32),
                experts=mega_moe.Fp8Experts(**experts()), routing_weights=torch.ones(2, 2))
    args.update(kw)
    with pytest.raises(err, match=match):
        op.forward_fp8(*args.values())


@built
def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level():
        x = fwd.make_dual(torch.ones(2, 128), torch.ones(2, 128))
        for call in (lambda: mega_moe.quantize_blocks(x), lambda: mega_moe.quantize_blocks(x, rows=128),
                     lambda: mega_moe.rms_norm(x, out_dtype=F8, scale_columns=128),
                     lambda: mega_moe.fp8_linear(x, torch.ones(3, 128)), lambda: mega_moe.fp8_linear(torch.ones(3, 128), x),
                     lambda: mega_moe.fp8_matmul(f8(2, 128), f8(2, 128), e8(2, 1), e8(1, 1), bias=x[:, 0].clone())):
            with pytest.raises(ValueError, match="forward-mode"):
                call()


FAKE = ctypes.c_void_p(1 << 20)
BIG = 1 << 40


@built
@pytest.mark.parametrize("batch,rows,cols,block,ldq,xt", [
    (-1, 1, 8, 1, 8, 0), (1, -1, 8, 1, 8, 0), (1, 1, -8, 1, 8, 0), (1, 1 << 31, 8, 1, 8, 0), (1, 1, 1 << 31, 1, 1 << 31, 0),
    (1 << 20, 1 << 20, 8, 1, 8, 0), (1, 1 << 20, 1 << 20, 1, 1 << 20, 0), (1, 1, 8, 2, 8, 0), (1, 1, 8, 1, 7, 0),
    (1, 1, 8, 1, 129, 0), (1, 1, 8, 1, 8, 3), (1, 1, 8, 1, 8, 4), (1, 1, 8, 1, 8, -1),
])
def test_quantize_entry_refuses(batch, rows, cols, block, ldq, xt):
    lib = _lib.load()
    assert lib.mm_quantize_blocks(FAKE, cols, 0, xt, batch, rows, cols, block, FAKE, ldq, FAKE, None) == -1
    assert b"mm_quantize_blocks" in lib.mm_last_error()


@built
def test_quantize_entries_refuse_null_and_wrong_forms():
    lib = _lib.load()
    for x, q, s in ((None, FAKE, FAKE), (FAKE, None, FAKE), (FAKE, FAKE, None)):
        assert lib.mm_quantize_blocks(x, 8, 0, 0, 1, 1, 8, 1, q, 8, s, None) == -1
    turn = lib.mm_quantize_blocks_t
    assert turn(FAKE, 8, 0, None, -1, 8, 1, None, None, FAKE, FAKE, None) == -1
    assert turn(FAKE, 8, 3, None, 8, 8, 1, None, None, FAKE, FAKE, None) == -1
    assert turn(FAKE, 8, 0, None, 8, 8, 64, None, None, FAKE, FAKE, None) == -1
    assert turn(FAKE, 8, 0, None, 8, 8, 1, FAKE, None, FAKE, FAKE, None) == -1
    assert turn(FAKE, 8, 0, None, 8, 8, 1, None, None, None, FAKE, None) == -1
    assert turn(FAKE, 8, 4, None, 8, 8, 128, None, None, FAKE, FAKE, None) == -1  # E4M3 without its scales
    assert turn(FAKE, 8, 4, FAKE, 8, 8, 1, None, None, FAKE, FAKE, None) == -1
    assert turn(FAKE, 8, 4, FAKE, 8, 8, 128, FAKE, FAKE, FAKE, FAKE, None) == -1
    assert b"mm_quantize_blocks_t" in lib.mm_last_error()
    norm = lib.mm_rms_norm_blocks
    assert norm(FAKE, 8, 0, None, 0, 0, None, 0, 1, 32769, 1e-6, None, FAKE, FAKE, None) == -1
    assert norm(FAKE, 8, 4, None, 0, 4, None, 0, 1, 8, 1e-6, None, FAKE, FAKE, None) == -1
    assert norm(FAKE, 8, 2, FAKE, 8, 0, None, 0, 1, 8, 1e-6, FAKE, FAKE, FAKE, None) == -1
    assert norm(FAKE, 8, 0, FAKE, 8, 0, None, 0, 1, 8, 1e-6, None, FAKE, FAKE, None) == -1
    assert norm(FAKE, 8, 0, None, 0, 0, None, 0, 1, 8, 1e-6, None, FAKE, None, None) == -1
    assert b"mm_rms_norm_blocks" in lib.mm_last_error()


@built
@pytest.mark.parametrize("m,n,k,lda,ldb,ldo,ot", [
    (-1, 8, 8, 8, 8, 8, 0), (8, 0, 8, 8, 8, 8, 0), (8, 8, 0, 8, 8, 8, 0), (8, 8, (1 << 23) + 1, BIG, BIG, 8, 0),
    (8, 8, 8, 7, 8, 8, 0), (8, 8, 8, 8, 7, 8, 0), (8, 8, 8, 8, 8, 7, 0), (8, 8, 8, (1 << 23) + 1, 8, 8, 0),
    (8, 8, 8, 8, (1 << 23) + 1, 8, 0), (8, 8, 8, 8, 8, 8, 3), (8, 8, 8, 8, 8, 8, 4),
    ((1 << 31) - 1, 8, 8, 8, 8, 8, 0), (8, (1 << 31) - 1, 8, 8, 8, (1 << 31), 0),
])
def test_product_entry_refuses(m, n, k, lda, ldb, ldo, ot):
    lib = _lib.load()
    assert lib.mm_fp8_matmul(FAKE, lda, FAKE, FAKE, ldb, FAKE, None, 0, m, n, k, FAKE, ldo, ot, None) == -1
    assert b"mm_fp8_matmul" in lib.mm_last_error()


@built
def test_product_entry_refuses_null():
    lib = _lib.load()
    for i in range(5):
        a, sa, b, sb, out = [None if j == i else FAKE for j in range(5)]
        assert lib.mm_fp8_matmul(a, 8, sa, b, 8, sb, None, 0, 8, 8, 8, out, 8, 0, None) == -1
    assert lib.mm_fp8_matmul(FAKE, 8, FAKE, FAKE, 8, FAKE, FAKE, 3, 8, 8, 8, FAKE, 8, 0, None) == -1  # the bias's type


@built
@pytest.mark.parametrize("tokens,k,E,H,I,act", [
    (-1, 1, 8, 128, 128, 0), (1, 0, 8, 128, 128, 0), (1, 65, 8, 128, 128, 0), (1, 1, 0, 128, 128, 0),
    (1, 1, 32769, 128, 128, 0), (1, 1, 8, 64, 128, 0), (1, 1, 8, 128, 192, 0), (1, 1, 8, 128, 128, 3),
    (1 << 28, 8, 8, 128, 128, 0), (1 << 25, 1, 8, 128, 128, 0), (1, 1, 1, 1 << 16, 1 << 15, 0),
])
def test_layer_entry_refuses(tokens, k, E, H, I, act):
    lib = _lib.load()
    rc = lib.mm_moe_fp8(*[FAKE] * 8, tokens, k, E, H, I, act, 1.0, 0.0, 7.0, FAKE, FAKE, BIG, None)
    assert rc == -1 and b"mm_moe_fp8" in lib.mm_last_error()
    if act < 3:
        assert lib.mm_moe_fp8_scratch_bytes(tokens, k, E, H, I) == 0


@built
def test_layer_entry_refuses_null_alignment_and_small_scratch():
    lib = _lib.load()
    sizes = (3, 2, 8, 128, 128)
    tail = (*sizes, 0, 1.0, 0.0, 7.0)
    need = lib.mm_moe_fp8_scratch_bytes(*sizes)
    assert need > 6 * 128 * 4
    for i in range(8):
        assert lib.mm_moe_fp8(*[None if j == i else FAKE for j in range(8)], *tail, FAKE, FAKE, need, None) == -1
    odd = ctypes.c_void_p((1 << 20) + 8)
    for i in (0, 4, 6):  # x, w1, w2
        assert lib.mm_moe_fp8(*[odd if j == i else FAKE for j in range(8)], *tail, FAKE, FAKE, need, None) == -1
        assert b"aligned" in lib.mm_last_error()
    assert lib.mm_moe_fp8(*[FAKE] * 8, *tail, odd, FAKE, need, None) == -1
    assert lib.mm_moe_fp8(*[FAKE] * 8, *tail, FAKE, odd, need, None) == -1
    assert lib.mm_moe_fp8(*[FAKE] * 8, *tail, FAKE, FAKE, need - 1, None) == -2
    assert lib.mm_moe_fp8(*[FAKE] * 8, *tail, FAKE, None, need, None) == -2
    assert b"scratch" in lib.mm_last_error()
    assert lib.mm_moe_fp8(*[None] * 8, 0, *tail[1:], None, None, 0, None) == 0  # no tokens, nothing to do
