"""forward_few reads the operator at every call, as forward does."""

import copy
import os

import pytest
import torch

import mega_moe
from mega_moe import _lib

BF = torch.bfloat16
built = pytest.mark.skipif(not os.path.exists(_lib.library_path()), reason="libmegamoe.so not built")
CHANGES = [dict(activation="swiglu"), dict(clamp_limit=0.25), dict(activation="situglu", situ_beta=3.0),
           dict(activation="situglu", situ_linear_beta=0.5)]


def _operator(**kw):
    cfg = mega_moe.MoEForwardConfig(activation="clamp_swiglu", clamp_limit=1.5)
    op = mega_moe.FusedMoEForward(None, max_tokens_per_rank=16, hidden_size=128, top_k=2, num_experts=4, config=cfg)
    for name, value in kw.items():
        setattr(op, name, value)
    return op


@built
@pytest.mark.parametrize("change", CHANGES + [dict(max_tokens_per_rank=5)])
def test_the_native_description_follows_the_operator(change):
    rows = torch.zeros(1, 128)
    op = _operator()
    op._few_layer(rows)
    before = op._few.__getstate__()
    other = copy.deepcopy(op)  # the copy's description is of before the change
    for o in (op, other):
        for name, value in change.items():
            setattr(o, name, value)
        o._few_layer(rows)
        fresh = _operator(**change)
        fresh._few_layer(rows)
        assert o._few.__getstate__() == fresh._few.__getstate__() != before
    kept = op._few
    op._few_layer(rows)
    assert op._few is kept  # and is built once as long as nothing changes


@pytest.mark.gpu
@pytest.mark.parametrize("change", CHANGES)
def test_outputs_follow_the_operator(change):
    g = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, gu, dn = rnd(6, 128).to(BF), (rnd(4, 128, 256) * 0.2).to(BF), (rnd(4, 128, 128) * 0.1).to(BF)
    sel = torch.rand(6, 4, generator=g, device="cuda").argsort(1)[:, :2].to(torch.int32).contiguous()
    w = torch.rand(6, 2, generator=g, device="cuda")
    ex = mega_moe.Int8Experts.quantize(gu, dn)
    xq, xs = mega_moe.quantize_rows(x)
    op = _operator()
    run = lambda o: (o.forward_few(x, sel, gu, dn, w), o.forward_few_int8(xq, xs, sel, ex, w))
    before = run(op)
    for name, value in change.items():
        setattr(op, name, value)
    after, want = run(op), run(_operator(**change))
    assert all(torch.equal(a, b) and not torch.equal(a, c) for a, b, c in zip(after, want, before))


@pytest.mark.gpu
def test_fewer_tokens_allowed_from_now_on():
    op = _operator()
    args = [torch.zeros(6, 128, dtype=BF, device="cuda"), torch.zeros(6, 2, dtype=torch.int32, device="cuda"),
            torch.zeros(4, 128, 256, dtype=BF, device="cuda"), torch.zeros(4, 128, 128, dtype=BF, device="cuda"),
            torch.zeros(6, 2, device="cuda")]
    op.forward_few(*args)
    op.max_tokens_per_rank = 5
    with pytest.raises(ValueError, match="max_tokens_per_rank=5"):
        op.forward_few(*args)
