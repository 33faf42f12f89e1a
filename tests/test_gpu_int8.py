"""int8_matmul on the GPU against whole numbers and 64 bits.

The int32 sum is exact, so the result is off by its conversion to fp32, two
products with scales and the bias (each 2^-24 of what it rounds, 2^-22 in all
of the scaled sum and of the bias) and by half a step of the output's type."""

import pytest
import torch

import mega_moe
from mega_moe import _lib

pytestmark = pytest.mark.gpu

BF, F16, F32, I8 = torch.bfloat16, torch.float16, torch.float32, torch.int8


def _operands(m, n, k, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=I8)
    b = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=I8)
    sa = torch.rand(m, generator=g, device="cuda") * 1e-3 + 1e-4
    sb = torch.rand(n, generator=g, device="cuda") * 1e-2 + 1e-3
    return a, b, sa, sb


def _sums(a, b):
    return a.double() @ b.double().t()  # whole numbers below 2^31: exact


def _check(out, a, b, sa, sb, bias, dtype):
    assert out.dtype == dtype
    ref = _sums(a, b) * sa.double()[:, None] * sb.double()
    slack = ref.abs() * 2**-22
    if bias is not None:
        ref = ref + bias.double()
        slack = slack + bias.double().abs() * 2**-22
    f = torch.finfo(dtype)
    bound = ref.abs() * f.eps / 2 + slack * (1 + f.eps) + f.smallest_normal * f.eps / 2
    over = (out.double() - ref).abs() - bound
    assert not (over > 0).any(), f"{over.max().item():.3e} over the bound at {over.argmax().item()}"


SHAPES = [(1, 1, 1), (1, 16, 64), (3, 5, 7), (1, 2048, 1536), (2, 129, 300), (16, 256, 128), (17, 100, 1000),
          (31, 65, 4096), (32, 1000, 2049), (33, 512, 640), (64, 768, 2048), (65, 257, 129), (100, 300, 515),
          (127, 128, 128), (128, 128, 256), (129, 383, 1024), (255, 257, 2050), (256, 256, 896), (300, 1100, 130),
          (1021, 1793, 2309), (1024, 2048, 4096), (4097, 130, 200)]


@pytest.mark.parametrize("dtype,bias", [(BF, None), (F16, F32), (F32, BF)])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k, dtype, bias):
    a, b, sa, sb = _operands(m, n, k)
    bias = None if bias is None else torch.randn(n, device="cuda").to(bias)
    _check(mega_moe.int8_matmul(a, b, sa, sb, bias=bias, out_dtype=dtype), a, b, sa, sb, bias, dtype)


@pytest.mark.parametrize("m,n,k", [  # tiles of 256, 128, 64 and 32 rows, K whole and cut, rows on odd addresses
    (4096, 4096, 640), (4090, 4090, 3001), (2048, 3000, 517), (1500, 2000, 300), (700, 5000, 2050), (128, 4096, 4099),
    (128, 4096, 2048), (200, 2000, 260), (40, 4000, 4101), (48, 4096, 2048)])
def test_every_tile(m, n, k):
    a, b, sa, sb = _operands(m, n, k, seed=7)
    _check(mega_moe.int8_matmul(a, b, sa, sb), a, b, sa, sb, None, BF)


@pytest.mark.parametrize("m", [1, 5, 40, 130, 300])
@pytest.mark.parametrize("k", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 1023, 1025])
def test_ends_of_the_sum(m, k):
    """Whole results: scales of one, fp32 out; bytes behind a row's end are other values."""
    a, b, _, _ = _operands(m, 70, k + 40, seed=k)
    a, b = a[:, 3:3 + k], b[:, 5:5 + k]
    out = mega_moe.int8_matmul(a, b, torch.ones(m, device="cuda"), torch.ones(70, device="cuda"), out_dtype=F32)
    assert torch.equal(out.double(), _sums(a, b).float().double())


@pytest.mark.parametrize("m", [1, 64, 200])
def test_largest_sums(m):
    k = (1 << 17) - 1
    a = torch.full((m, k), -128, dtype=I8, device="cuda")
    b = torch.full((3, k), -128, dtype=I8, device="cuda")
    b[1], b[2] = 127, 0
    out = mega_moe.int8_matmul(a, b, torch.ones(m, device="cuda"), torch.ones(3, device="cuda"), out_dtype=F32)
    want = torch.tensor([16384.0 * k, -16256.0 * k, 0.0], dtype=torch.float64).float().cuda()
    assert torch.equal(out, want.expand(m, 3))


@pytest.mark.parametrize("m", [1, 30, 150])
def test_shapes_and_strides(m):
    a, b, sa, sb = _operands(m, 150, 333)
    want = mega_moe.int8_matmul(a, b, sa, sb)
    wide = torch.zeros(2 * m, 400, dtype=I8, device="cuda")
    wide[::2, 7:340] = a
    tall = torch.zeros(300, 335, dtype=I8, device="cuda")
    tall[::2, :333] = b
    assert torch.equal(mega_moe.int8_matmul(wide[::2, 7:340], tall[::2, :333], sa, sb), want)
    assert torch.equal(mega_moe.int8_matmul(a.view(1, m, 333), b, sa.view(1, m), sb), want[None])
    assert torch.equal(mega_moe.int8_matmul(a[0], b, sa[0], sb), mega_moe.int8_matmul(a[:1], b, sa[:1], sb)[0])
    assert mega_moe.int8_matmul(a[:0], b, sa[:0], sb).shape == (0, 150)


def test_scales_that_are_not_finite_stay_in_their_row_and_column():
    a, b, sa, sb = _operands(20, 40, 100)
    want = mega_moe.int8_matmul(a, b, sa, sb)
    sa[3], sb[5] = float("nan"), float("nan")
    out = mega_moe.int8_matmul(a, b, sa, sb)
    keep_r, keep_c = torch.arange(20, device="cuda") != 3, torch.arange(40, device="cuda") != 5
    assert torch.isnan(out[3]).all() and torch.isnan(out[:, 5]).all()
    assert torch.equal(out[keep_r][:, keep_c], want[keep_r][:, keep_c])


def test_refusals():
    a, b, sa, sb = _operands(4, 8, 32)
    with pytest.raises(ValueError, match="device of a"):
        mega_moe.int8_matmul(a, b.cpu(), sa, sb)
    with pytest.raises(ValueError, match="evenly spaced"):
        mega_moe.int8_matmul(torch.zeros(4, 6, 32, dtype=I8, device="cuda").transpose(0, 1), b,
                             torch.ones(6, 4, device="cuda"), sb)
    with pytest.raises(ValueError, match="unit column stride"):
        mega_moe.int8_matmul(torch.zeros(32, 4, dtype=I8, device="cuda").t(), b, sa, sb)
    with pytest.raises(ValueError, match="overlap"):
        mega_moe.int8_matmul(a[:1].expand(4, 32), b, sa, sb)


@pytest.mark.parametrize("m", [1, 48, 700])
def test_streams_and_graphs(m):
    """Calls on two streams at once, and a captured call replayed beside eager ones."""
    sets = [_operands(m, 900, 2000, seed=s) for s in range(2)]
    want = [mega_moe.int8_matmul(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, (st, s) in enumerate(zip(streams, sets)):
            with torch.cuda.stream(st):
                got[i].append(mega_moe.int8_matmul(*s))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])
    a, b, sa, sb = sets[0]
    a = a.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mega_moe.int8_matmul(a, b, sa, sb)
    for rep in range(4):
        a.copy_(sets[rep & 1][0])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mega_moe.int8_matmul(a, b, sa, sb)), rep


@pytest.mark.parametrize("dtype,code,bias", [(BF, 0, F16), (F16, 1, None), (F32, 2, F32)])
@pytest.mark.parametrize("m,n,k", [
    (9, 203, 700), (33, 203, 96), (40, 4003, 4100), (40, 4003, 4101), (130, 4003, 2052), (130, 4003, 2053), (300, 1003, 1000),
    (300, 1003, 1001), (1021, 1795, 2308), (1021, 1795, 2309), (520, 1795, 700),
    (520, 1795, 701), (120, 4095, 2052), (120, 4095, 2053), (1501, 2003, 300), (4091, 4095, 1281)])
def test_padded_outputs(m, n, k, dtype, code, bias):
    """The C entry with output rows that are padded, at odd strides: what lies
    between the rows stays as it was."""
    a, b, sa, sb = _operands(m, n, k, seed=3)
    bias = None if bias is None else torch.randn(n, device="cuda").to(bias)
    want = mega_moe.int8_matmul(a, b, sa, sb, bias=bias, out_dtype=dtype)
    _check(want, a, b, sa, sb, bias, dtype)
    for pad in (1, 6):
        out = torch.full((m + 1, n + pad), 7.0, device="cuda", dtype=dtype)
        _lib.call("mm_int8_matmul", _lib.ptr(a), k, _lib.ptr(b), k, _lib.ptr(sa), _lib.ptr(sb), _lib.ptr(bias),
                  0 if bias is None else _lib.ELEMENT_TYPES[bias.dtype], m, n, k, _lib.ptr(out), n + pad, code,
                  torch.cuda.current_stream().cuda_stream)
        assert torch.equal(out[:m, :n], want) and (out[:, n:] == 7).all() and (out[m] == 7).all()


@pytest.mark.parametrize("k", [64, 132])  # operands from memory, and the largest tiles
def test_outputs_past_32_bits(k):
    """An output of more than 2^31 elements: its last row and column."""
    m, n = 70000, 32768
    a, b, sa, sb = _operands(m, n, k)
    out = mega_moe.int8_matmul(a, b, sa, sb)
    _check(out[-5:], a[-5:], b, sa[-5:], sb, None, BF)
    _check(out[:, -3:], a, b[-3:], sa, sb[-3:], None, BF)
