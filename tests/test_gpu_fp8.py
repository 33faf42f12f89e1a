"""E4M3 with a scale for each block of 128: blocks, products and the trained
projection against their definitions in 64 bits."""

import pytest
import torch

import mega_moe
from tests import _fp8 as R

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
F8, E8 = R.F8, R.E8


def _bytes(t):
    return t.view(torch.uint8)


def _same_blocks(q, s, x, block_rows):
    """q and s bit for bit those of the definition."""
    rq, rs = R.quant(x.double(), block_rows)
    assert q.dtype == F8 and s.dtype == E8 and q.is_contiguous() and s.is_contiguous()
    assert torch.equal(q.double(), rq) and torch.equal(torch.signbit(q.float()), torch.signbit(rq.float()) & ~rs_bad(rs, q, block_rows))
    sd = s.double()
    assert torch.equal(sd.isnan(), rs.isnan()) and torch.equal(sd.nan_to_num(), rs.nan_to_num())


def rs_bad(rs, q, block_rows):
    rows, cols = q.shape
    return rs.isnan().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 127), (129, 129), (256, 384), (70, 2305), (1000, 8)])
def test_blocks(dtype, block_rows, rows, cols):
    gen = torch.Generator().manual_seed(rows * 7 + cols)
    x = (torch.randn(rows, cols, generator=gen) * torch.exp(2 * torch.randn(rows, 1, generator=gen))).to(dtype).cuda()
    q, s = mega_moe.quantize_blocks(x, rows=block_rows)
    _same_blocks(q, s, x, block_rows)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_blocks_at_the_borders(block_rows):
    """Zeros, ties, the largest and smallest values, infinities and NaN."""
    x = torch.zeros(128 * 12, 128)
    for i, top in enumerate([448.0, 449.0, 480.0, 447.9, 2.0 ** -140, 3e38, 1.0, 2.0 ** -118, 2.0 ** -119]):
        # multiples of a sixteenth step: ties of every binade, subnormal ones too
        x[i * 128:(i + 1) * 128] = torch.linspace(-1, 1, 128 * 128).view(128, 128) * top
        x[i * 128:(i + 1) * 128, 0] = top
        x[i * 128 + 1, 1:] = torch.arange(1, 128) / 128 * top
    x[9 * 128, 3], x[10 * 128 + 5, 127], x[10 * 128 + 6, 0] = float("nan"), float("inf"), float("-inf")
    x[11 * 128, 0] = -0.0
    x = x.cuda()
    q, s = mega_moe.quantize_blocks(x, rows=block_rows)
    _same_blocks(q, s, x, block_rows)
    assert _bytes(s)[9 * 128 // block_rows, 0] == 255


def test_blocks_of_strided_input():
    x = torch.randn(3, 5, 300, 260, device="cuda")
    for view in (x[..., :130], x[1:, :, ::2, 1:], x[:, 2], x[2, :, 3], x.transpose(0, 1)[1]):
        if view.dim() == 3 and view.stride(0) != 300 * 260:  # matrices apart from each other: no even rows
            with pytest.raises(ValueError, match="evenly spaced"):
                mega_moe.quantize_blocks(view)
        else:
            q, s = mega_moe.quantize_blocks(view)
            c, cs = mega_moe.quantize_blocks(view.contiguous())
            assert q.shape == view.shape and torch.equal(_bytes(q), _bytes(c)) and torch.equal(_bytes(s), _bytes(cs))
        q, s = mega_moe.quantize_blocks(view, rows=128)
        flat = view.reshape(-1, *view.shape[-2:])
        for i, m in enumerate(flat):
            _same_blocks(q.reshape(flat.shape)[i], s.reshape(-1, *s.shape[-2:])[i], m, 128)
    with pytest.raises(ValueError, match="evenly spaced"):
        mega_moe.quantize_blocks(x[:, :4, :7])
    empty, s = mega_moe.quantize_blocks(torch.empty(0, 130, device="cuda"))
    assert empty.shape == (0, 130) and s.shape == (0, 2)
    empty, s = mega_moe.quantize_blocks(torch.empty(2, 0, 130, device="cuda"), rows=128)
    assert empty.shape == (2, 0, 130) and s.shape == (2, 0, 2)


# ------------------------------------------------------------------ norm
@pytest.mark.parametrize("hidden", [1, 5, 7, 8, 9, 120, 127, 128, 129, 135, 512, 517, 2048, 4097, 7168, 16390])
@pytest.mark.parametrize("dtype,res", [(BF, BF), (BF, F32), (F16, None), (F32, F32)])
def test_norm_to_blocks(hidden, dtype, res):
    """The bytes are those of the unrounded y: a value may land on the other side
    of a rounding border if y's own error in fp32 reaches it."""
    gen = torch.Generator().manual_seed(hidden)
    rows = 9
    x = torch.randn(rows, hidden, generator=gen).to(dtype).cuda()
    w = (1 + 0.3 * torch.randn(hidden, generator=gen)).to(dtype).cuda()
    r = None if res is None else (3 * torch.randn(rows, hidden, generator=gen)).to(res).cuda()
    out = mega_moe.rms_norm(x, w, residual=r, out_dtype=F8, scale_columns=128)
    q, s = out[:2]
    h = x if r is None else (x.float() + r.float()).to(res)
    if r is not None:
        assert torch.equal(out[2], h)
    hd = h.double()
    y = hd / (hd.square().mean(dim=1, keepdim=True) + 1e-6).sqrt() * w.double()
    # fp32: the mean of H squares (a tree of at most 8 * 4 + 16 sums in a row), rsqrt, two products
    err = (48 / 2 + 6) * 2.0 ** -24
    lo, _ = R.quant(y * (1 - err), 1)
    hi, _ = R.quant(y * (1 + err), 1)
    _, rs = R.quant(y, 1)
    assert s.shape == rs.shape and torch.equal(s.double(), rs)
    v = q.double()
    assert torch.all((v - lo) * (v - hi) <= 0)
    assert (v != R.quant(y, 1)[0]).float().mean() < 1e-3


def test_norm_to_blocks_keeps_bad_values_in_their_blocks():
    x = torch.randn(4, 300, device="cuda", dtype=BF)
    x[1, 200] = float("nan")
    x[2, 5] = float("inf")
    q, s = mega_moe.rms_norm(x, out_dtype=F8, scale_columns=128)
    clean, cs = mega_moe.rms_norm(x[[0, 3]].contiguous(), out_dtype=F8, scale_columns=128)
    assert torch.equal(_bytes(q)[[0, 3]], _bytes(clean)) and torch.equal(_bytes(s)[[0, 3]], _bytes(cs))
    # a NaN spreads over its row; h / infinity is 0 but for infinity / infinity
    assert _bytes(s)[1].tolist() == [255, 255, 255] and not _bytes(q)[1].any()
    assert _bytes(s)[2].tolist() == [255, 127, 127] and not (_bytes(q)[2] & 127).any()


# ------------------------------------------------------------------ products
def _matmul(m, n, k, dtype=BF, bias=False, seed=0, nan=False):
    gen = torch.Generator().manual_seed(seed)
    a, sa = R.rows_e4m3(gen, m, k)
    b, sb = R.blocks_e4m3(gen, n, k)
    c = torch.randn(n, generator=gen).mul(1000).to(dtype).cuda() if bias else None
    if nan:
        _bytes(sa)[m // 2, -1] = 255
        _bytes(sb)[-1, 0] = 255
    return a, b, sa, sb, c


def _check_matmul(out, a, b, sa, sb, c):
    av, bv = R.values(a.cpu(), sa.cpu(), 1), R.values(b.cpu(), sb.cpu(), 128)
    ref = av @ bv.t()
    bound = R.sum_error(av, bv, wide=out.dtype == F32)
    if c is not None:
        ref = ref + c.double().cpu()
        bound = bound + 2.0 ** -24 * (ref.abs() + bound)
    near = bound + R.half_step(out.dtype) * (ref.abs() + bound)
    R.near(out, ref, near)


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 1, 128), (1, 16, 129), (2, 17, 127), (5, 130, 384), (16, 256, 2048), (17, 40, 640), (33, 129, 257),
    (64, 512, 1024), (65, 300, 131), (100, 1000, 1000), (128, 128, 128), (129, 257, 385), (256, 256, 512),
    (255, 384, 4096), (300, 1793, 769), (520, 520, 520), (700, 2048, 256), (1021, 1030, 1153),
])
@pytest.mark.parametrize("dtype,bias", [(BF, False), (F16, True), (F32, True)])
def test_matmul(m, n, k, dtype, bias):
    ops = _matmul(m, n, k, dtype, bias, seed=m + n + k)
    a, b, sa, sb, c = ops
    if dtype == F16:  # values within its range
        _bytes(sa).sub_(14)
        if c is not None:
            c.div_(1000)
    _check_matmul(mega_moe.fp8_matmul(a, b, sa, sb, bias=c, out_dtype=dtype), a, b, sa, sb, c)


@pytest.mark.parametrize("m", [3, 40, 300])
def test_matmul_nan_scales_mark_their_own(m):
    a, b, sa, sb, _ = _matmul(m, 300, 400, seed=5, nan=True)
    out = mega_moe.fp8_matmul(a, b, sa, sb, out_dtype=F32)
    _check_matmul(out, a, b, sa, sb, None)
    assert out.isnan().any() and not out.isnan().all()


@pytest.mark.parametrize("m", [4, 50, 400])
def test_matmul_extreme_scales(m):
    """Products near either end of fp32, the smallest scale byte among them."""
    gen = torch.Generator().manual_seed(3)
    for ea, eb in ((-127, 60), (-60, -60), (60, 40), (100, -127)):
        a, sa = R.rows_e4m3(gen, m, 256, low=ea, high=ea)
        b, sb = R.blocks_e4m3(gen, 144, 256, low=eb, high=eb)
        _check_matmul(mega_moe.fp8_matmul(a, b, sa, sb, out_dtype=F32), a, b, sa, sb, None)


@pytest.mark.parametrize("m", [1, 9, 30, 70, 300])
@pytest.mark.parametrize("off", [0, 1, 3, 4, 8])
def test_matmul_strides_and_alignment(m, off):
    gen = torch.Generator().manual_seed(off)
    k, n = 517, 200
    for pad in (0, 3, 16):
        base, sa = R.rows_e4m3(gen, m, k + off + pad)
        other, sb = R.blocks_e4m3(gen, n, k + off + pad)
        a, b = base[:, off:off + k], other[:, off:off + k]
        sa, sb = sa[:, :R.ceil(k, 128)].contiguous(), sb[:, :R.ceil(k, 128)].contiguous()
        _check_matmul(mega_moe.fp8_matmul(a, b, sa, sb, out_dtype=F32), a, b, sa, sb, None)


def test_matmul_leading_axes_and_no_rows():
    gen = torch.Generator().manual_seed(1)
    a, sa = R.rows_e4m3(gen, 6, 256)
    b, sb = R.blocks_e4m3(gen, 130, 256)
    flat = mega_moe.fp8_matmul(a, b, sa, sb)
    assert torch.equal(mega_moe.fp8_matmul(a.view(2, 3, 256), b, sa.view(2, 3, 2), sb), flat.view(2, 3, 130))
    assert torch.equal(mega_moe.fp8_matmul(a[0], b, sa[0], sb), mega_moe.fp8_matmul(a[:1], b, sa[:1], sb)[0])
    assert mega_moe.fp8_matmul(a[:0], b, sa[:0], sb).shape == (0, 130)


# ------------------------------------------------------------------ trained projection
def _linear_reference(x, w, dy):
    wide = [t.dtype == F32 for t in (x, x, w)]
    x, w, dy = x.detach().double().cpu(), w.detach().double().cpu(), dy.double().cpu()
    xq, wq = R.quantized(x, 1), R.quantized(w, 128)
    dyr, dyc, xc = R.quantized(dy, 1), R.quantized(dy.t().contiguous(), 1), R.quantized(xq, 128)
    pairs = ((xq, wq), (dyr, wq.t().contiguous()), (dyc, xc.t().contiguous()))
    return [(p @ q.t(), R.sum_error(p, q, u)) for (p, q), u in zip(pairs, wide)]


@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 200, 130), (5, 3, 260), (128, 128, 128), (130, 129, 127), (300, 513, 384),
                                   (1000, 72, 640)])
@pytest.mark.parametrize("xt,wt", [(BF, BF), (BF, F32), (F16, F16), (F32, F32)])
def test_linear(m, n, k, xt, wt):
    gen = torch.Generator().manual_seed(m + n * k)
    x = torch.randn(m, k, generator=gen).to(xt).cuda().requires_grad_()
    w = (torch.randn(n, k, generator=gen) * 0.05).to(wt).cuda().requires_grad_()
    dy = (torch.randn(m, n, generator=gen) * torch.exp(torch.randn(m, 1, generator=gen))).to(xt).cuda()
    dy[::7] = 0
    y = mega_moe.fp8_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert dx.dtype == xt and dw.dtype == wt and y.dtype == xt
    for got, (ref, bound) in zip((y, dx, dw), _linear_reference(x, w, dy)):
        tiny = 2.0 ** -25 if got.dtype == F16 else 0.0  # half of fp16's smallest step
        R.near(got.detach(), ref, bound + R.half_step(got.dtype) * (ref.abs() + bound) + tiny)


def test_linear_against_differences():
    """Where E4M3 holds every value, y is bilinear and differences are exact."""
    gen = torch.Generator().manual_seed(2)
    m, n, k = 9, 130, 140
    x = torch.randint(-8, 9, (m, k), generator=gen).float().cuda()
    w = torch.randint(-4, 5, (n, k), generator=gen).float().cuda()
    dy = torch.randint(-3, 4, (m, n), generator=gen).float().cuda()
    dx, dw = torch.autograd.grad(mega_moe.fp8_linear(x.requires_grad_(), w.requires_grad_()), (x, w), dy)
    with torch.no_grad():
        base = mega_moe.fp8_linear(x, w)
        for i, j in ((0, 0), (3, 127), (8, 128), (5, 139)):
            moved = x.clone()
            moved[i, j] += 1
            assert ((mega_moe.fp8_linear(moved, w) - base) * dy).sum().item() == dx[i, j].item()
        for i, j in ((0, 0), (127, 5), (128, 130), (129, 139)):
            moved = w.clone()
            moved[i, j] += 1
            assert ((mega_moe.fp8_linear(x, moved) - base) * dy).sum().item() == dw[i, j].item()


def test_linear_parts():
    """One gradient at a time, leading axes, no rows, and rows that do not see each other."""
    x = torch.randn(2, 150, 300, device="cuda", dtype=BF)
    w = torch.randn(200, 300, device="cuda", dtype=BF)
    dy = torch.randn(2, 150, 200, device="cuda", dtype=BF)
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = mega_moe.fp8_linear(a, b)
    dx, dw = torch.autograd.grad(y, (a, b), dy)
    assert torch.equal(mega_moe.fp8_linear(x, w), y.detach())
    c = x.clone().requires_grad_()
    (only,) = torch.autograd.grad(mega_moe.fp8_linear(c, w), c, dy)
    assert torch.equal(only, dx)
    d = w.clone().requires_grad_()
    (only,) = torch.autograd.grad(mega_moe.fp8_linear(x, d), d, dy)
    assert torch.equal(only, dw)
    e = x[1, 7:9].clone().requires_grad_()
    part = mega_moe.fp8_linear(e, w)
    (only,) = torch.autograd.grad(part, e, dy[1, 7:9].contiguous())
    R.near(part.detach(), y.detach()[1, 7:9], 2 * R.half_step(BF) * y.detach()[1, 7:9].abs() + 1e-4)
    R.near(only, dx[1, 7:9], 2 * R.half_step(BF) * dx[1, 7:9].abs() + 1e-4)
    none = torch.empty(0, 300, device="cuda", dtype=BF, requires_grad=True)
    z = mega_moe.fp8_linear(none, d)
    dn, dd = torch.autograd.grad(z, (none, d), torch.empty(0, 200, device="cuda", dtype=BF))
    assert z.shape == (0, 200) and dn.shape == (0, 300) and dd.shape == (200, 300) and not dd.any()


def test_linear_twice_raises():
    x = torch.randn(4, 130, device="cuda", requires_grad=True)
    w = torch.randn(20, 130, device="cuda", requires_grad=True)
    (dx,) = torch.autograd.grad(mega_moe.fp8_linear(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        dx.sum().backward()
