"""E4M3 products on every tile, the large ones above all: dense operands, several stages of
K and one that it cuts, rows at odd addresses, biases, all result types, NaN.

Each size is held to the tile that it is here for (``test_fp8_tiles.py`` on the CPU)."""

import pytest
import torch

import mega_moe
from tests import _fp8 as R
from tests._fp8_tiles import tile

pytestmark = pytest.mark.gpu

BF, F16, F32, F8 = torch.bfloat16, torch.float16, torch.float32, R.F8

SIZES = [  # rows, channels, K, bytes in front of a row and behind it, and the tile for 16 and for 32 bits
    (4096, 4096, 1024, 0, 0, (256, 256), (128, 128)),
    (4090, 4093, 1153, 1, 2, (256, 256), (128, 128)),  # odd addresses, a stage cut to one byte
    (4100, 3971, 385, 3, 0, (256, 256), (128, 128)),
    (4095, 4080, 255, 0, 1, (256, 256), (128, 128)),   # a cut stage and none or one behind it
    (4089, 4096, 129, 4, 0, (256, 256), (128, 128)),
    (4090, 4090, 128, 0, 0, (256, 256), (128, 128)),
    (2500, 2500, 1000, 0, 0, (128, 128), (64, 128)),   # two rounds of tiles
    (1990, 2030, 641, 1, 0, (128, 128), (64, 128)),
    (2047, 2047, 300, 0, 3, (128, 128), (64, 64)),
    (2048, 2048, 4096, 0, 0, (128, 128), (64, 128)),
]


def operands(m, n, k, before, behind, seed, low=-8, high=-4):
    gen = torch.Generator().manual_seed(seed)
    a, sa = R.rows_e4m3(gen, m, before + k + behind, low=low, high=high)
    b, sb = R.blocks_e4m3(gen, n, before + k + behind, low=low, high=high)
    kb = R.ceil(k, 128)
    return a[:, before:before + k], b[:, before:before + k], sa[:, :kb].contiguous(), sb[:, :kb].contiguous()


def check(out, a, b, sa, sb, bias):
    av, bv = R.values(a, sa, 1), R.values(b, sb, 128)
    ref, off = av @ bv.t(), R.sum_error(av, bv, wide=out.dtype == F32)
    if bias is not None:
        ref = ref + bias.double()
        off = off + 2.0 ** -23 * (ref.abs() + off)
    tiny = 2.0 ** -25 if out.dtype == F16 else 0.0  # half of fp16's smallest step
    R.near(out, ref, off + R.half_step(out.dtype) * (ref.abs() + off) + tiny)


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s[:3])))
@pytest.mark.parametrize("dtype,bias", [(BF, None), (F16, F16), (BF, F32), (F32, BF)])
def test_product_on_its_tile(size, dtype, bias):
    m, n, k, before, behind, *tiles = size
    assert tile(m, n, k, dtype == F32) == tiles[dtype == F32]
    ops = operands(m, n, k, before, behind, seed=m + k)
    add = None if bias is None else torch.randn(n, generator=torch.Generator().manual_seed(k)).to(bias).cuda()
    check(mega_moe.fp8_matmul(*ops, bias=add, out_dtype=dtype), *ops, add)


@pytest.mark.parametrize("size", [SIZES[1], SIZES[7]], ids=lambda s: "x".join(map(str, s[:3])))
@pytest.mark.parametrize("dtype", [BF, F32])
def test_nan_stays_in_its_rows_and_channels(size, dtype):
    """NaN scales in the first, a middle and the last block of K, and NaN bytes."""
    m, n, k, before, behind, *tiles = size
    assert tile(m, n, k, dtype == F32) == tiles[dtype == F32]
    a, b, sa, sb = operands(m, n, k, before, behind, seed=3)
    clean = mega_moe.fp8_matmul(a, b, sa, sb, out_dtype=dtype)
    bad = torch.zeros_like(clean, dtype=torch.bool)
    for row, block in ((0, 0), (m // 2, sa.shape[1] // 2), (m - 1, sa.shape[1] - 1)):
        sa.view(torch.uint8)[row, block] = 255
        bad[row] = True
    sb.view(torch.uint8)[3, 1] = 255
    bad[:, 3 * 128:4 * 128] = True
    a.view(torch.uint8)[7, k - 1] = 0x7F
    b.view(torch.uint8)[n - 1, 0] = 0xFF
    bad[7], bad[:, n - 1] = True, True
    out = mega_moe.fp8_matmul(a, b, sa, sb, out_dtype=dtype)
    assert torch.equal(out.isnan(), bad) and torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("m,n,k", [(4090, 3970, 4005), (4000, 4090, 3970)])
@pytest.mark.parametrize("xt,wt", [(BF, BF), (F16, F16), (BF, F32)])
def test_linear_on_large_tiles(m, n, k, xt, wt):
    """All three products of a training step on dense operands."""
    up = lambda v: R.ceil(v, 128) * 128
    assert tile(m, n, up(k), False) == tile(m, k, up(n), False) == (256, 256)
    assert tile(n, k, up(m), wt == F32) == ((128, 128) if wt == F32 else (256, 256))
    gen = torch.Generator().manual_seed(m)
    x = torch.randn(m, k, generator=gen).to(xt).cuda().requires_grad_()
    w = (torch.randn(n, k, generator=gen) * 0.05).to(wt).cuda().requires_grad_()
    dy = (torch.randn(m, n, generator=gen) * 0.1 * torch.exp(torch.randn(m, 1, generator=gen))).to(xt).cuda()
    dy[::7] = 0
    y = mega_moe.fp8_linear(x, w)
    got = (y.detach(), *torch.autograd.grad(y, (x, w), dy))
    xd, wd, dd = x.detach().double(), w.detach().double(), dy.double()
    xq, wq = R.quantized(xd, 1), R.quantized(wd, 128)
    pairs = ((xq, wq), (R.quantized(dd, 1), wq.t().contiguous()),
             (R.quantized(dd.t().contiguous(), 1), R.quantized(xq, 128).t().contiguous()))
    for out, (p, q) in zip(got, pairs):
        ref, off = p @ q.t(), R.sum_error(p, q, wide=out.dtype == F32)
        tiny = 2.0 ** -25 if out.dtype == F16 else 0.0
        R.near(out, ref, off + R.half_step(out.dtype) * (ref.abs() + off) + tiny)
