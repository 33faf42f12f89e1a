"""How the E4M3 operators sum: few activations of the layer and results in 32 bits in fp32
throughout, results in 16 bits within the bound that they are documented with."""

import pytest
import torch

import mega_moe
from tests import _fp8 as R
from tests.test_gpu_fp8_layer import make, operator, reference

pytestmark = pytest.mark.gpu

# tokens, hidden, inter, experts, top_k with up to 64 rows an expert on average and up to 2^21 activations,
# and the shares of the tokens whose first slot goes to experts 0, 1, ...
UNEVEN = [
    ((500, 384, 256, 8, 1), ()),               # 62 rows on average: some above 64, some below
    ((510, 1024, 384, 8, 1), (0.25, 0.25)),    # 128 rows and few more
    ((600, 512, 256, 40, 2), (0.3, 0.2, 0.1)),  # 190, 130 and 70 rows
    ((700, 128, 256, 30, 2), (0.5,)),          # one block of K, 360 rows: two tiles, one of 160 rows and more
    ((640, 256, 128, 20, 1), (0.24, 0.2, 0.13)),  # two blocks of K
    ((900, 512, 1024, 140, 2), (0.3, 0.1)),    # 220 MB of weights, which pass the caches by
]


def uneven(size, shares, seed):
    """The layer's operands; the first slots of the given shares of the tokens go to one expert each."""
    T, H, I, E, k = size
    x, sx, sel, ex, w = make(*size, seed=seed)
    assert T * k <= 64 * E and T * k * I <= 1 << 21
    at = 0
    for e, share in enumerate(shares):
        sel[at:at + int(T * share), 0] = e
        at += int(T * share)
    assert torch.bincount(sel.flatten().long(), minlength=E).max() > 64
    return x, sx, sel, ex, w


@pytest.mark.parametrize("size,shares", UNEVEN)
@pytest.mark.parametrize("act", ["swiglu", "clamp_swiglu", "situglu"])
def test_few_activations_of_uneven_experts_are_summed_in_32_bits(size, shares, act):
    """An activation leaves its E4M3 step only where fp32 sums can carry it there, also in an expert of many rows."""
    T, H, I, E, k = size
    ops = uneven(size, shares, T * I)
    R.near(operator(T, H, k, E, act).forward_fp8(*ops), *reference(*ops, act, wide=True))


@pytest.mark.parametrize("size", [(640, 1024, 256, 20, 1), (900, 512, 1024, 140, 2),
                                  (2000, 512, 1280, 40, 1), (1500, 256, 512, 16, 6)])  # the last two: many activations
def test_a_token_does_not_see_where_the_others_go(size):
    """In a call of the same sizes: 8 tokens alone on their expert, and with 40, 100, 150 and 300 more beside them."""
    T, H, I, E, k = size
    x, sx, sel, ex, w = make(*size, seed=5)
    sel[:] = 2 + torch.arange(T * k, device="cuda", dtype=torch.int32).view(T, k) % (E - 2)
    sel[:8, 0] = 1
    op = operator(T, H, k, E)
    alone = op.forward_fp8(x, sx, sel, ex, w)
    for more in (40, 100, 150, 300):
        crowd = sel.clone()
        crowd[8:8 + more, 0] = 1
        assert torch.equal(op.forward_fp8(x, sx, crowd, ex, w)[:8], alone[:8]), more


@pytest.mark.parametrize("size,expert", [
    ((5, 256, 128, 4, 2), None), ((200, 384, 256, 16, 2), None),  # few routes; up to 64 rows an expert
    ((640, 384, 128, 20, 1), 3), ((500, 128, 256, 8, 1), 2), ((900, 512, 1024, 140, 2), 77),  # one expert has every token's first slot
    ((420, 512, 128, 3, 1), None),  # more than 64 rows on average
])
def test_few_activations_keep_what_cancels(size, expert):
    """Gate sums of 448 * 448 - 448 * 448 + 1, exact in fp32: cut 13 bits below the largest product they would be 0."""
    T, H, I, E, k = size
    x, sx, sel, ex, w = make(*size, seed=T)
    if expert is not None:
        sel[:, 0] = expert
    for t in (x, ex.gate_up):
        t.view(torch.uint8).zero_()
    for t in (sx, ex.gate_up_scale):
        t.view(torch.uint8).fill_(127)
    x[:, :3] = torch.tensor([448.0, 448.0, 1.0], device="cuda").to(R.F8)
    ex.gate_up[:, :I, :3] = torch.tensor([448.0, -448.0, 1.0], device="cuda").to(R.F8)
    ex.gate_up[:, I:, 2] = torch.tensor(1.0, device="cuda").to(R.F8)
    out = operator(T, H, k, E).forward_fp8(x, sx, sel, ex, w).double().cpu()
    ref, _ = reference(x, sx, sel, ex, w, "swiglu")
    # equal columns, on a scale of 128 and not next to a border: what is left is FC2's own sum (7 products of 8 cut at
    # 2^-13) and the result's rounding, of the sum of terms
    size_of = torch.zeros(T, H, dtype=torch.float64)
    for e in range(E):
        down = R.values(ex.down[e].cpu(), ex.down_scale[e].cpu(), 128).abs().sum(1)
        size_of += ((sel.cpu() == e) * w.cpu()).sum(1, keepdim=True).double() * 0.78 * down  # silu(1) and half an E4M3 step
    assert ref.abs().max() > 0.1 * size_of.max() / I ** 0.5
    R.near(out, ref, 2.0 ** -8 * ref.abs() + 2.0 ** -10 * size_of)


# ------------------------------------------------------------------ products
PRODUCTS = [(3, 40, 517), (40, 300, 640), (300, 260, 1000), (1000, 1900, 700), (2500, 2500, 300), (4090, 4093, 385)]


def _grouped(m, n, k, row, channel):
    """E4M3 operands whose rows repeat ``row`` and ``channel``, all scales 1."""
    make_rows = lambda r, c: torch.tensor(c, device="cuda").repeat(R.ceil(k, len(c)))[:k].expand(r, k).contiguous().to(R.F8)
    scale = lambda *s: torch.full(s, 127, dtype=torch.uint8, device="cuda").view(R.E8)
    kb = R.ceil(k, 128)
    return make_rows(m, row), make_rows(n, channel), scale(m, kb), scale(R.ceil(n, 128), kb)


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_products_to_32_bits_keep_what_cancels(m, n, k):
    """Every group of 8 holds 448 * 448 - 448 * 448 + 1: sums of whole numbers below 2^24, exact in fp32."""
    a, b, sa, sb = _grouped(m, n, k, [448.0, 448.0, 1.0, 0, 0, 0, 0, 0], [448.0, -448.0, 1.0, 0, 0, 0, 0, 0])
    want = (a[0].double() * b[0].double()).sum().item()
    assert want < 448 * 448 + 1000
    out = mega_moe.fp8_matmul(a, b, sa, sb, out_dtype=torch.float32)
    assert (out == want).all()


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("small", [3.75, 4.0, 14.0])
def test_products_to_16_bits_are_as_far_off_as_documented(m, n, k, dtype, small):
    """Seven of eight products next to the border at which they are cut: within 7 * 2^-13 of the largest."""
    a, b, sa, sb = _grouped(m, n, k, [448.0] + [small] * 7, [448.0] + [small] * 7)
    sa.view(torch.uint8).sub_(14)  # into fp16's range
    exact = (a[0].double() * b[0].double()).sum() * 2.0 ** -14
    largest = R.ceil(k, 8) * 448.0 * 448.0 * 2.0 ** -14
    out = mega_moe.fp8_matmul(a, b, sa, sb, out_dtype=dtype).double()
    off = 7 * 2.0 ** -13 * largest + (128 + R.ceil(k, 128) + 16) * 2.0 ** -23 * exact
    assert (out - exact).abs().max() <= off + R.half_step(dtype) * (exact + off)
