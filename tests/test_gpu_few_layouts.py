"""forward_few on operands at odd addresses and with weights whose rows or
experts lie apart, overlap or repeat: the bits of packed operands."""

import pytest
import torch

import mega_moe
from tests import test_gpu_few as few

pytestmark = pytest.mark.gpu

BF, I8 = torch.bfloat16, torch.int8
T, E, K, H, F = 20, 6, 3, 256, 384


def _shifted(t, by):
    """The same contiguous values, `by` elements behind an aligned address."""
    buf = torch.empty(t.numel() + by, dtype=t.dtype, device="cuda")
    out = buf[by:].view(t.shape)
    out.copy_(t)
    return out


def _case():
    sel, w = few._routing(T, E, K, "drop", 3)
    gu, dn = few._weights(E, H, F, "contiguous")
    g = torch.Generator(device="cuda").manual_seed(8)
    return torch.randn(T, H, generator=g, device="cuda").to(BF), sel, gu, dn, w, few._operator(E, K, H)


@pytest.mark.parametrize("by", [1, 2, 3, 5])
def test_odd_addresses(by):
    x, sel, gu, dn, w, op = _case()
    want = op.forward_few(x, sel, gu, dn, w)
    odd = [_shifted(t, by) for t in (x, sel, gu, dn, w)]
    assert torch.equal(op.forward_few(*odd), want)
    odd[3] = _shifted(dn.transpose(1, 2).contiguous(), by).transpose(1, 2)
    assert torch.equal(op.forward_few(*odd), op.forward_few(x, sel, gu, dn.transpose(1, 2).contiguous().transpose(1, 2), w))
    xq, xs, ex = few._int8_inputs(T, E, H, F)
    want = op.forward_few_int8(xq, xs, sel, ex, w)
    moved = mega_moe.Int8Experts(*(_shifted(t, by) for t in (ex.gate_up, ex.gate_up_scale, ex.down, ex.down_scale)))
    assert torch.equal(op.forward_few_int8(_shifted(xq, by), _shifted(xs, by), odd[1], moved, odd[4]), want)


@pytest.mark.parametrize("pad", [1, 8, 130])
@pytest.mark.parametrize("transposed", [False, True])
def test_rows_and_experts_apart(pad, transposed):
    x, sel, gu, dn, w, op = _case()
    rows, cols = (F, H) if transposed else (H, F)
    wide = torch.full((E, rows + 2, cols + pad), float("nan"), dtype=BF, device="cuda")
    view = wide[:, 1:-1, :cols]
    view.copy_(dn.transpose(1, 2) if transposed else dn)
    view = view.transpose(1, 2) if transposed else view
    plain = dn.transpose(1, 2).contiguous().transpose(1, 2) if transposed else dn
    assert torch.equal(op.forward_few(x, sel, gu, view, w), op.forward_few(x, sel, gu, plain, w))


def test_one_expert_for_all():
    """Down weights that an expand repeats over experts and over rows."""
    x, sel, gu, dn, w, op = _case()
    one = dn[:1].expand(E, H, F)
    assert torch.equal(op.forward_few(x, sel, gu, one, w), op.forward_few(x, sel, gu, one.contiguous(), w))
    row = dn[:, :1].expand(E, H, F)
    assert torch.equal(op.forward_few(x, sel, gu, row, w), op.forward_few(x, sel, gu, row.contiguous(), w))
