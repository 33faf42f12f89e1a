"""NaN and infinities through the gated activations on the GPU.

The clamp of ``clamp_swiglu`` keeps NaN (torch's ``clamp`` does, and the
oracle's), so a token whose row holds one comes out NaN under every activation
and the other tokens keep their bits."""

import pytest
import torch

import mega_moe
from oracle import moe_oracle as O

pytestmark = pytest.mark.gpu

BF, F32, I8 = torch.bfloat16, torch.float32, torch.int8
NAN, INF = float("nan"), float("inf")
E, K, H, F, T = 4, 2, 256, 128, 12
ACTS = [("swiglu", {}), ("clamp_swiglu", dict(clamp_limit=1.5)), ("situglu", dict(situ_beta=2.0)),
        ("situglu", dict(situ_beta=2.0, situ_linear_beta=3.0))]


def _operator(act, kw):
    cfg = mega_moe.MoEForwardConfig(activation=act, **kw)
    return mega_moe.FusedMoEForward(None, max_tokens_per_rank=64, hidden_size=H, top_k=K, num_experts=E, config=cfg)


def _layer(seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    sel = torch.rand(T, E, generator=g, device="cuda").argsort(1)[:, :K].to(torch.int32).contiguous()
    rw = torch.rand(T, K, generator=g, device="cuda") + 0.1
    return rnd(T, H).to(BF), sel, (rnd(E, H, 2 * F) * H**-0.5).to(BF), (rnd(E, H, F) * F**-0.5).to(BF), rw


def _int8_layer(seed=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r8 = lambda *s: torch.randint(-127, 128, s, generator=g, device="cuda", dtype=I8)
    sc = lambda *s: torch.rand(*s, generator=g, device="cuda") + 0.5
    ex = mega_moe.Int8Experts(r8(E, 2 * F, H), sc(E, 2 * F) * H**-0.5 / 74, r8(E, H, F), sc(E, H) * F**-0.5 / 74)
    return r8(T, H), sc(T) / 74, ex


def _others_kept(got, want, bad):
    keep = [t for t in range(T) if t not in bad]
    assert torch.equal(got[keep], want[keep]) and torch.isfinite(want).all()
    for t in bad:
        assert torch.isnan(got[t]).all(), (t, got[t].float().abs().max())


@pytest.mark.parametrize("act,kw", ACTS)
@pytest.mark.parametrize("entry", ["forward", "forward_few"])
def test_nan_rows(entry, act, kw):
    x, sel, gu, dn, rw = _layer()
    op = _operator(act, kw)
    run = getattr(op, entry)
    want = run(x, sel, gu, dn, rw).clone()
    bad = x.clone()
    bad[5, 3], bad[7] = NAN, NAN
    _others_kept(run(bad, sel, gu, dn, rw), want, (5, 7))


@pytest.mark.parametrize("act,kw", ACTS)
def test_nan_scales(act, kw):
    _, sel, _, _, rw = _layer()
    xq, xs, ex = _int8_layer()
    op = _operator(act, kw)
    want = op.forward_few_int8(xq, xs, sel, ex, rw)
    xs[2] = NAN
    _others_kept(op.forward_few_int8(xq, xs, sel, ex, rw), want, (2,))


@pytest.mark.parametrize("act,kw", ACTS)
def test_a_broken_row_through_norm_and_layer(act, kw):
    """The norm marks a row that holds an infinity by its scale; the layer keeps the mark."""
    x, sel, _, _, rw = _layer()
    _, _, ex = _int8_layer()
    op = _operator(act, kw)
    x[4, 9] = INF
    q, s = mega_moe.rms_norm(x, out_dtype=I8)
    out = op.forward_few_int8(q, s, sel, ex, rw)
    assert torch.isnan(out[4]).all() and torch.isfinite(out[[t for t in range(T) if t != 4]]).all()


@pytest.mark.parametrize("act,kw", ACTS)
def test_nan_in_the_backward(act, kw):
    """A NaN token's gradients are NaN as the oracle's derivative pair has them;
    the other tokens' keep their bits."""
    x, sel, gu, dn, rw = _layer()
    dy = torch.randn(T, H, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").to(BF)
    op = _operator(act, kw)
    bad = x.clone()
    bad[5, 3] = NAN
    grads = []
    for rows in (x, bad):
        _, saved = op.forward(rows, sel, gu, dn, rw, return_saved=True)
        g = mega_moe.moe_backward_triton(saved, dy)
        grads.append((g["grad_hidden"].clone(), g["grad_routing_weights"].clone()))
    for want, got in zip(*grads):
        _others_kept(got, want, (5,))


@pytest.mark.parametrize("fmt", ["bf16", "fp16"])
def test_derivative_pair_keeps_nan(fmt):
    """Element for element: NaN where the oracle's clamp derivatives are NaN."""
    from mega_moe.ops import _kernels as KS

    torch.manual_seed(4)
    rows, inter, limit = 3, 128, 1.5
    dt = BF if fmt == "bf16" else torch.float16
    gu = torch.randn(rows, 2 * inter, device="cuda").mul_(2).to(dt)
    gu[0, 3], gu[1, inter + 5], gu[2, 7], gu[2, inter + 7] = NAN, NAN, NAN, NAN
    dc = torch.randn(rows, inter, device="cuda").to(BF)
    offs = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    scale = torch.ones(rows, device="cuda")
    dab, dscale = KS.swiglu_bwd(dc, gu, scale, offs, rows, "clamp_swiglu", 1.0, None, limit)
    torch.cuda.synchronize()
    g, u, d = gu[:, :inter].double().cpu(), gu[:, inter:].double().cpu(), dc.double().cpu()
    a, da, v, dv = O.gated_act_grad(g, u, "clamp_swiglu", clamp_limit=limit)
    ref = torch.cat([d * da * v, d * a * dv], dim=1)
    got = dab[:rows].double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    # exp and reciprocal good to 2^-16, one rounding to bf16; dact sums two terms of one size
    fine = ~torch.isnan(ref)
    assert ((got - ref).abs()[fine] <= ref.abs()[fine] * 2**-8 + d.abs().repeat(1, 2)[fine] * 4 * 2**-14).all()
    assert torch.isnan(dscale[:rows]).all()


@pytest.mark.parametrize("bad", [INF, -INF])
@pytest.mark.parametrize("act,kw", ACTS)
def test_infinite_scales(act, kw, bad):
    """A row's scale is finite or marks the row as broken, also where the
    activation saturates (clamp, tanh) and would hide an infinity."""
    _, sel, _, _, rw = _layer()
    xq, xs, ex = _int8_layer()
    op = _operator(act, kw)
    want = op.forward_few_int8(xq, xs, sel, ex, rw)
    xs[2], xs[9] = bad, bad
    _others_kept(op.forward_few_int8(xq, xs, sel, ex, rw), want, (2, 9))
