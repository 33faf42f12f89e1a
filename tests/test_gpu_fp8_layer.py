"""The layer on E4M3 rows and experts against its definition in 64 bits."""

import pytest
import torch

import mega_moe
from tests import _fp8 as R

pytestmark = pytest.mark.gpu

BF, F8, E8 = torch.bfloat16, R.F8, R.E8


def _act(kind, g, u):
    if kind == "swiglu":
        return g * torch.sigmoid(g) * u
    if kind == "clamp_swiglu":
        g = torch.minimum(g, torch.full_like(g, 7.0))
        return g * torch.sigmoid(g) * u.clamp(-7, 7)
    return 2.0 * torch.tanh(g / 2.0) * torch.sigmoid(g) * 3.0 * torch.tanh(u / 3.0)


def make(T, H, I, E, k, seed=0, drop=0.0, device="cuda"):
    gen = torch.Generator().manual_seed(seed)
    x, sx = R.rows_e4m3(gen, T, H, device, -8, -5)
    gu, gus = R.blocks_e4m3(gen, E * 2 * I, H, device, -12, -10)
    dn, dns = R.blocks_e4m3(gen, E * H, I, device, -12, -10)
    ex = mega_moe.Fp8Experts(gu.view(E, 2 * I, H), gus.view(E, 2 * I // 128, H // 128), dn.view(E, H, I),
                             dns.view(E, H // 128, I // 128))
    sel = torch.rand(T, E, generator=gen).argsort(dim=1)[:, :k].to(torch.int32)
    sel[torch.rand(T, k, generator=gen) < drop] = -1
    w = torch.rand(T, k, generator=gen) + 0.1
    return x, sx, sel.contiguous().to(device), ex, w.to(device)


def operator(T, H, k, E, act="swiglu"):
    extra = dict(situ_beta=2.0, situ_linear_beta=3.0) if act == "situglu" else {}
    return mega_moe.FusedMoEForward(None, max_tokens_per_rank=T, hidden_size=H, top_k=k, num_experts=E,
                                    config=mega_moe.MoEForwardConfig(activation=act, **extra))


def reference(x, sx, sel, ex, w, act, wide=False):
    """(output, bound of the error) in 64 bits on the CPU. ``wide``: gate and up are summed in fp32 throughout."""
    xv = R.values(x.cpu(), sx.cpu(), 1)
    T, H = xv.shape
    I = ex.down.shape[2]
    out = torch.zeros(T, H, dtype=torch.float64)
    bound = torch.zeros(T, H, dtype=torch.float64)
    step = R.half_step(BF)
    for e in range(ex.gate_up.shape[0]):
        token, slot = torch.nonzero(sel.cpu() == e, as_tuple=True)
        if not token.numel():
            continue
        w1 = R.values(ex.gate_up[e].cpu(), ex.gate_up_scale[e].cpu(), 128)
        w2 = R.values(ex.down[e].cpu(), ex.down_scale[e].cpu(), 128)
        rows, weight = xv[token], w.cpu().double()[token, slot][:, None]
        gu, off = rows @ w1.t(), R.sum_error(rows, w1, wide)
        g, u = gu[:, :I], gu[:, I:]
        a = _act(act, g, u) * weight
        # gate's factor has a slope of at most 1.2 (SiTU-GLU: beta tanh(g / beta) <= g), up's of 1; 16 steps for the function itself
        da = weight * (1.2 * u.abs() * off[:, :I] + (g.abs() + off[:, :I]) * off[:, I:]) + 2.0 ** -20 * a.abs()
        q, s = R.quant(a, 1)
        av = R.values(q, s, 1)
        # rounding is monotone: what the kernel holds lies between the bytes of both ends, on the same scale
        sc = s.repeat_interleave(128, 1)
        ends = [R.round_e4m3(((a + d) / sc).clamp(-448, 448)) * sc for d in (-da, da)]
        dq = torch.maximum((ends[0] - av).abs(), (ends[1] - av).abs())
        y = av @ w2.t()
        dy = dq @ w2.abs().t() + R.sum_error(av, w2)
        out.index_add_(0, token, y)
        bound.index_add_(0, token, dy)
    k = sel.shape[1]
    return out, bound + step * (out.abs() + bound) + k * 2.0 ** -23 * out.abs()


SIZES = [  # tokens, hidden, inter, experts, top_k
    (1, 128, 128, 1, 1), (1, 256, 128, 8, 2), (3, 384, 256, 16, 4), (17, 128, 384, 4, 2), (40, 640, 128, 3, 3),
    (64, 256, 256, 40, 8), (150, 256, 128, 2, 2), (333, 384, 256, 2, 1), (500, 128, 128, 8, 6), (700, 256, 512, 2, 2),
]


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("act,drop", [("swiglu", 0.0), ("clamp_swiglu", 0.2), ("situglu", 0.0)])
def test_layer(size, act, drop):
    T, H, I, E, k = size
    ops = make(T, H, I, E, k, seed=T + H, drop=drop)
    out = operator(T, H, k, E, act).forward_fp8(*ops)
    assert out.dtype == BF and out.shape == (T, H)
    R.near(out, *reference(*ops, act))


def test_layer_routes_of_no_expert():
    """Ids out of range carry no expert; a token with none has zeros."""
    x, sx, sel, ex, w = make(20, 256, 128, 4, 2, seed=9)
    sel[0], sel[5, 1], sel[7, 0], sel[9] = -1, 4, -7, 1000
    op = operator(20, 256, 2, 4)
    out = op.forward_fp8(x, sx, sel, ex, w)
    R.near(out, *reference(x, sx, torch.where((sel >= 0) & (sel < 4), sel, -1), ex, w, "swiglu"))
    assert not out[0].any() and not out[9].any()
    assert not op.forward_fp8(x, sx, torch.full_like(sel, -1), ex, w).any()
    same = torch.full_like(sel, 2)  # one expert has every route, twice a token
    R.near(op.forward_fp8(x, sx, same, ex, w), *reference(x, sx, same, ex, w, "swiglu"))
    none = op.forward_fp8(x[:0], sx[:0], sel[:0], ex, w[:0])
    assert none.shape == (0, 256) and none.dtype == BF


@pytest.mark.parametrize("T", [6, 200])
def test_layer_keeps_nan_to_its_token(T):
    x, sx, sel, ex, w = make(T, 256, 128, 4, 2, seed=3)
    op = operator(T, 256, 2, 4)
    clean = op.forward_fp8(x, sx, sel, ex, w)
    bad, other = sx.clone(), sel.clone()
    bad.view(torch.uint8)[4, 1] = 255
    bad.view(torch.uint8)[5, 0] = 255
    other[5] = -1
    out = op.forward_fp8(x, bad, other, ex, w)
    assert out[4].isnan().all() and not out[5].any()
    rest = [i for i in range(T) if i not in (4, 5)]
    assert torch.equal(out[rest], clean[rest])


def test_layer_from_weights_and_norm():
    """Norm to E4M3 rows, experts from bf16 weights: near the bf16 layer, within what E4M3 rounds."""
    T, H, I, E, k = 96, 512, 256, 8, 2
    gen = torch.Generator().manual_seed(4)
    gate_up = (torch.randn(E, H, 2 * I, generator=gen) * 0.05).to(BF).cuda()
    down = (torch.randn(E, I, H, generator=gen) * 0.05).to(BF).cuda().transpose(1, 2)
    x = torch.randn(T, H, generator=gen).to(BF).cuda()
    sel = torch.rand(T, E, generator=gen).argsort(dim=1)[:, :k].to(torch.int32).contiguous().cuda()
    w = torch.softmax(torch.randn(T, k, generator=gen), dim=1).cuda()
    ex = mega_moe.Fp8Experts.quantize(gate_up, down)
    q, s = mega_moe.rms_norm(x, out_dtype=F8, scale_columns=128)
    op = operator(T, H, k, E)
    out = op.forward_fp8(q, s, sel, ex, w)
    R.near(out, *reference(q, s, sel, ex, w, "swiglu"))
    bf = op.forward(mega_moe.rms_norm(x), sel, gate_up, down, w)
    # each factor is off by up to 2^-4, as if at random: a few of them in a row
    assert (out.float() - bf.float()).norm() / bf.float().norm() < 0.1
