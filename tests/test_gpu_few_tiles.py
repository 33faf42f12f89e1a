"""forward_few in the tiles that the sizes of its other tests do not choose: 64
columns of the first product with passes of 32 rows of an expert, and with 64
rows asked for (32 columns then, as more partial sums do not fit)."""

import pytest
import torch

import mega_moe
from tests import test_gpu_few as few

pytestmark = pytest.mark.gpu

CASES = [  # T, E, k, H, F, routing: 16, 16 and 32 rows an expert in the mean, 512 tiles of 64 columns
    (64, 64, 16, 256, 512, "even"), (64, 64, 16, 384, 640, "drop"), (32, 32, 16, 256, 1024, "even"),
    (64, 64, 32, 256, 512, "even"),
]


@pytest.mark.parametrize("layout", ["natural", "contiguous"])
@pytest.mark.parametrize("T,E,k,H,F,routing", CASES)
def test_wide_tiles_of_many_rows(T, E, k, H, F, routing, layout):
    sel, w = few._routing(T, E, k, routing, T)
    gu, dn = few._weights(E, H, F, layout)
    g = torch.Generator(device="cuda").manual_seed(T + E)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    op = few._operator(E, k, H)
    out = op.forward_few(x, sel, gu, dn, w)
    few._check(out, few._reference(x, None, sel, w, gu, None, dn, None, "swiglu"))
    # a token's bits are those it has alone and in other tiles
    for a, b in ((0, 1), (3, 19), (T - 1, T)):
        assert torch.equal(op.forward_few(x[a:b], sel[a:b], gu, dn, w[a:b]), out[a:b])


@pytest.mark.parametrize("T,E,k,H,F,routing", [CASES[0], CASES[3]])
def test_the_same_in_int8(T, E, k, H, F, routing):
    sel, w = few._routing(T, E, k, routing, T)
    x, xs, ex = few._int8_inputs(T, E, H, F)
    out = few._operator(E, k, H).forward_few_int8(x, xs, sel, ex, w)
    few._check(out, few._reference(x, xs, sel, w, ex.gate_up, ex.gate_up_scale, ex.down, ex.down_scale, "swiglu"))
