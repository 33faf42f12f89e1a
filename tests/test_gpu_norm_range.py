"""rms_norm on rows far from 1 on the GPU, against 64 bits.

Bounds as for rows near 1: 1 / rms is good to 2^-19 and a product with it to
2^-18, the backward's terms to 2^-17 of their absolute sum, a column's sum of a
few rows to 2^-18 more; each output is rounded once. A row's size cancels out of
all of them, as no step leaves the range of fp32."""

import pytest
import torch

import mega_moe

pytestmark = pytest.mark.gpu

BF, F32, I8 = torch.bfloat16, torch.float32, torch.int8
E4M3 = torch.float8_e4m3fn
HIDDEN = [1, 7, 64, 513, 1021, 2048, 4099, 8193, 16400, 32768]


def _near(got, ref, slack, name):
    f = torch.finfo(got.dtype)
    bound = ref.abs() * f.eps / 2 + slack * (1 + f.eps) + f.smallest_normal * f.eps / 2
    over = (got.double() - ref).abs() - bound
    assert torch.isfinite(got).all() and not (over > 0).any(), f"{name}: {over.max().item():.3e} over the bound"


def _rows(hidden, sizes, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(len(sizes), hidden, generator=g, device="cuda").double()
    x = x + torch.sign(x) * 0.1  # no row of one column is near 0
    size = torch.tensor(sizes, dtype=torch.float64, device="cuda")[:, None]
    return (x * size).to(dtype), g


def _backward(hidden, sizes, dtype, eps, residual, rel=2**-17):
    x, g = _rows(hidden, sizes, dtype, hidden)
    w = (1 + 0.3 * torch.randn(hidden, generator=g, device="cuda")).requires_grad_()
    dy = torch.randn(len(sizes), hidden, generator=g, device="cuda").to(dtype)
    x.requires_grad_()
    res = (x.detach() * 0.5).requires_grad_() if residual else None
    out = mega_moe.rms_norm(x, w, residual=res, eps=eps)
    y, h = out if residual else (out, x)
    grads = torch.autograd.grad(y, (x, w), dy)
    hd, wd, dyd = h.detach().double(), w.detach().double(), dy.double()
    r = 1 / (hd.square().mean(-1, keepdim=True) + eps).sqrt()
    t, n = dyd * wd, hd * r
    mean = (t * n).mean(-1, keepdim=True)
    _near(grads[0], r * (t - n * mean), r * (t.abs() + n.abs() * (t * n).abs().mean(-1, keepdim=True)) * rel, "dx")
    _near(grads[1], (dyd * n).sum(0), (dyd * n).abs().sum(0) * rel, "dweight")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("hidden", HIDDEN)
def test_backward_of_large_and_small_rows(hidden, residual, dtype):
    """1 / rms cubed leaves fp32 for these rows; no step of the gradient does."""
    _backward(hidden, (1.0, 1e12, 1e13, 3e15, 1e17), dtype, 1e-6, residual)
    _backward(hidden, (1.0, 1e-12, 1e-13, 1e-14), dtype, 0.0, residual)


FAR = (1.0, 1e19, 1e25, 3e37, 1e-4)       # squares past the largest fp32
NEAR = (1.0, 1e-19, 1e-25, 1e-36, 1e4)    # and below the smallest; eps = 0


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("hidden", HIDDEN)
def test_forward_where_squares_leave_the_range(hidden, dtype):
    for sizes, eps in ((FAR, 1e-6), (NEAR, 0.0), (NEAR, 1e-60)):
        x, g = _rows(hidden, sizes, dtype, hidden + 1)
        w = 1 + 0.3 * torch.randn(hidden, generator=g, device="cuda")
        for res in (None, x * 0.5):
            out = mega_moe.rms_norm(x, w, residual=res, eps=eps)
            y, h = (out, x) if res is None else out
            hd, held = h.double(), torch.tensor(eps, dtype=F32).item()  # eps is an fp32 argument: 1e-60 is 0
            ref = hd / (hd.square().mean(-1, keepdim=True) + held).sqrt() * w.double()
            _near(y, ref, ref.abs() * 2**-18, "y")


@pytest.mark.parametrize("out_dtype,most", [(I8, 127.0), (E4M3, 448.0)])
@pytest.mark.parametrize("hidden", HIDDEN)
def test_eight_bits_where_squares_leave_the_range(hidden, out_dtype, most):
    """The same bytes as the row near 1 gives that a power of two makes of it."""
    x, _ = _rows(hidden, (1.0,) * 6, BF, hidden + 2)
    k = torch.tensor([1.0, 2.0**66, 2.0**100, 2.0**124, 2.0**-66, 2.0**-100], device="cuda")[:, None]
    w = torch.rand(hidden, device="cuda").to(BF) + 0.5
    q, s = mega_moe.rms_norm(x, w, eps=0.0, out_dtype=out_dtype)
    far_q, far_s = mega_moe.rms_norm((x.float() * k).to(BF), w, eps=0.0, out_dtype=out_dtype)
    assert torch.equal(far_q.float(), q.float()) and torch.equal(far_s, s)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("hidden", HIDDEN)
def test_backward_where_squares_leave_the_range(hidden, residual, dtype):
    _backward(hidden, FAR, dtype, 1e-6, residual)
    _backward(hidden, NEAR, dtype, 0.0, residual)


def test_eps_counts_in_every_range():
    """eps of the size of the mean square, where that is near either end of fp32."""
    for size, eps in ((2.0**-60, 2.0**-120), (2.0**-70, 2.0**-139), (2.0**63, 2.0**126), (2.0**70, 2.0**127)):
        x = torch.full((3, 520), size, device="cuda")
        ref = size / (size * size + eps) ** 0.5
        y = mega_moe.rms_norm(x, eps=eps).double()
        assert ((y - ref).abs() <= ref * 2**-17).all(), (size, eps)


def test_zero_rows_and_broken_rows_keep_their_meaning():
    for hidden in (5, 300, 3000):
        x = torch.zeros(3, hidden, device="cuda")
        assert not mega_moe.rms_norm(x, eps=1e-40).any()
        assert torch.isnan(mega_moe.rms_norm(x, eps=0.0)).all()  # 0 / 0
        x[1, 2] = float("inf")
        y = mega_moe.rms_norm(x)
        assert torch.isnan(y[1, 2]) and not y[[0, 2]].any()
