"""forward_few and forward_few_int8 on the GPU against the layer in 64 bits.

The bounds carry, for every element, the errors of the steps in front of it:
  * a dot product of n terms in fp32 is off by at most n 2^-23 of the sum of
    its absolute terms, in whatever order (2^-23: the matrix instructions
    promise no rounding to nearest of each step);
  * the activation's slopes are at most L in gate (1.1, or 1 + beta / 4 for
    situglu) and 1 in up, its own exp and reciprocal are good to 2^-16;
  * bf16: the activation is rounded to half a step, 2^-8; the output again;
  * int8: sums are whole; an activation within 2^-7 of a step of a rounding
    border may land on either side, a full step away.
"""

import pytest
import torch

import mega_moe

pytestmark = pytest.mark.gpu

BF, F32, I8 = torch.bfloat16, torch.float32, torch.int8
BETA, LBETA, LIMIT = 2.0, 3.0, 1.5


def _operator(E, k, H, act="swiglu"):
    kw = dict(situ_beta=BETA, situ_linear_beta=LBETA) if act == "situglu" else {}
    cfg = mega_moe.MoEForwardConfig(activation=act, clamp_limit=LIMIT, **kw)
    return mega_moe.FusedMoEForward(None, max_tokens_per_rank=64, hidden_size=H, top_k=k, num_experts=E, config=cfg)


def _routing(T, E, k, kind, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    sel = torch.rand(T, E, generator=g, device="cuda").argsort(1)[:, :k].to(torch.int32)
    if sel.shape[1] < k:
        sel = sel[:, torch.arange(k, device="cuda") % E]
    if kind == "one":
        sel.fill_(E - 1)
    elif kind == "repeat":
        sel[:, 1:] = sel[:, :1]
    elif kind == "drop":
        sel[torch.rand(T, k, generator=g, device="cuda") < 0.4] = -1
        sel[0] = E + 7
    elif kind == "none":
        sel.fill_(-5)
    w = torch.rand(T, k, generator=g, device="cuda") - 0.2
    return sel.contiguous(), w


def _weights(E, H, F, layout, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    gu = (torch.randn(E, H, 2 * F, generator=g, device="cuda") * H**-0.5).to(BF)
    dn = (torch.randn(E, H, F, generator=g, device="cuda") * F**-0.5).to(BF)
    if layout == "natural":
        dn = dn.transpose(1, 2).contiguous().transpose(1, 2)
    return gu, dn


def _act(kind, g, u):
    if kind == "swiglu":
        return g * torch.sigmoid(g), u, 1.1
    if kind == "clamp_swiglu":
        gc = g.clamp(max=LIMIT)
        return gc * torch.sigmoid(gc), u.clamp(-LIMIT, LIMIT), 1.1
    return BETA * torch.tanh(g / BETA) * torch.sigmoid(g), LBETA * torch.tanh(u / LBETA), 1 + BETA / 4


def _reference(x, xs, sel, w, gu, gus, dn, dns, kind):
    """(out, bound) in 64 bits; xs, gus, dns None: bf16."""
    int8 = xs is not None
    T, k = sel.shape
    E = gu.shape[0]
    H = x.shape[1]
    out = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    xd = x.double() if not int8 else x.double() * xs.double()[:, None]
    for e in sel.unique().tolist():
        if not 0 <= e < E:
            continue
        t, j = torch.nonzero(sel == e, as_tuple=True)
        w1 = gu[e].double() if not int8 else (gu[e].double() * gus[e].double()[:, None]).t()
        w2 = dn[e].double() if not int8 else dn[e].double() * dns[e].double()[:, None]
        F = w2.shape[1]
        pre, mag = xd[t] @ w1, xd[t].abs() @ w1.abs()
        # int8: whole sums, three roundings of scales
        err = pre.abs() * 2**-21 if int8 else mag * (H * 2**-23)
        a, v, slope = _act(kind, pre[:, :F], pre[:, F:])
        wt = w[t, j].double()[:, None]
        act = a * v * wt
        da = (slope * v.abs() * err[:, :F] + a.abs() * err[:, F:]) * wt.abs() * (1 + 2**-8) + act.abs() * 2**-16
        da = da + slope * err[:, :F] * err[:, F:] * wt.abs()
        if int8:
            r = act.view(len(t), F // 32, 32)
            top = r.abs().amax(-1, keepdim=True)
            s = torch.where(top > 0, top / 127, torch.ones_like(top))
            q = (r / s).round()
            near = ((r / s - (r / s).floor() - 0.5).abs() < 2**-7)
            step = (q * s)
            da = (step.abs() * 2**-15 + near * s).view(len(t), F)
            act = step.view(len(t), F)
        else:
            da = da + (act.abs() + da) * 2**-8 + 2.0**-133
        y, ymag = act @ w2.t(), act.abs() @ w2.abs().t()
        ye = da @ w2.abs().t() + ymag * ((F + 64) * 2**-23)
        out.index_add_(0, t, y)
        bound.index_add_(0, t, ye + y.abs() * 2**-20)
    return out, bound + (out.abs() + bound) * 2**-8 + 2.0**-133


def _check(got, ref):
    out, bound = ref
    assert got.dtype == BF and got.shape == out.shape
    over = (got.double() - out).abs() - bound
    assert not (over > 0).any(), f"{over.max().item():.3e} over the bound, largest value {out.abs().max().item():.3e}"


CASES = [  # T, E, k, H, F, routing
    (1, 8, 1, 128, 128, "even"), (1, 128, 8, 512, 256, "even"), (2, 4, 2, 256, 128, "even"), (3, 40, 5, 384, 384, "drop"),
    (5, 3, 3, 256, 640, "even"), (8, 64, 8, 1024, 512, "even"), (16, 2, 2, 256, 256, "even"), (16, 16, 4, 512, 128, "one"),
    (17, 8, 2, 256, 256, "even"), (17, 200, 6, 384, 256, "drop"), (32, 128, 8, 512, 384, "even"),
    (33, 1, 1, 256, 128, "one"), (40, 5, 4, 128, 256, "repeat"), (64, 8, 2, 256, 128, "even"), (64, 300, 16, 256, 256, "even"),
    (64, 2, 8, 128, 128, "even"), (64, 64, 64, 128, 128, "drop"), (64, 20000, 4, 128, 128, "drop"), (9, 6, 2, 256, 128, "none"),
    (1, 8, 2, 128, 128, "none"), (6, 5, 64, 128, 128, "one"),
]


@pytest.mark.parametrize("layout", ["natural", "contiguous"])
@pytest.mark.parametrize("T,E,k,H,F,routing", CASES)
def test_few(T, E, k, H, F, routing, layout):
    sel, w = _routing(T, E, k, routing, T)
    gu, dn = _weights(E, H, F, layout)
    x = torch.randn(T, H, device="cuda").to(BF)
    out = _operator(E, k, H).forward_few(x, sel, gu, dn, w)
    _check(out, _reference(x, None, sel, w, gu, None, dn, None, "swiglu"))


def _int8_inputs(T, E, H, F, seed=2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r8 = lambda *s: torch.randint(-127, 128, s, generator=g, device="cuda", dtype=I8)
    sc = lambda *s: torch.rand(*s, generator=g, device="cuda") + 0.5
    x, xs = r8(T, H), sc(T) / 74
    return x, xs, mega_moe.Int8Experts(r8(E, 2 * F, H), sc(E, 2 * F) * H**-0.5 / 74, r8(E, H, F), sc(E, H) * F**-0.5 / 74)


@pytest.mark.parametrize("T,E,k,H,F,routing", CASES)
def test_few_int8(T, E, k, H, F, routing):
    sel, w = _routing(T, E, k, routing, T)
    x, xs, ex = _int8_inputs(T, E, H, F)
    out = _operator(E, k, H).forward_few_int8(x, xs, sel, ex, w)
    _check(out, _reference(x, xs, sel, w, ex.gate_up, ex.gate_up_scale, ex.down, ex.down_scale, "swiglu"))


@pytest.mark.parametrize("act", ["swiglu", "situglu", "clamp_swiglu"])
@pytest.mark.parametrize("T", [2, 20])
def test_activations(T, act):
    E, k, H, F = 12, 3, 256, 256
    sel, w = _routing(T, E, k, "even", 5)
    gu, dn = _weights(E, H, F, "natural")
    gu = (gu.float() * 3).to(BF)  # gates and ups on both sides of the clamp
    x = torch.randn(T, H, device="cuda").to(BF)
    op = _operator(E, k, H, act)
    _check(op.forward_few(x, sel, gu, dn, w), _reference(x, None, sel, w, gu, None, dn, None, act))
    xq, xs, ex = _int8_inputs(T, E, H, F)
    xs = xs * 3
    _check(op.forward_few_int8(xq, xs, sel, ex, w),
           _reference(xq, xs, sel, w, ex.gate_up, ex.gate_up_scale, ex.down, ex.down_scale, act))


@pytest.mark.parametrize("T", [1, 16, 17, 64])
def test_agrees_with_forward(T):
    """The same layer as ``forward``, which rounds gate, up and the expert outputs too."""
    E, k, H, F = 32, 4, 512, 256
    sel, w = _routing(T, E, k, "drop", 3)
    gu, dn = _weights(E, H, F, "natural")
    x = torch.randn(T, H, device="cuda").to(BF)
    op = _operator(E, k, H)
    few, full = op.forward_few(x, sel, gu, dn, w).double(), op.forward(x, sel, gu, dn, w).double()
    ref, _ = _reference(x, None, sel, w, gu, None, dn, None, "swiglu")
    assert (few - ref).norm() <= (full - ref).norm() * 1.01


def test_a_token_does_not_see_the_others():
    """NaN and infinities of one token, or its scale, leave the others' bits alone."""
    E, k, H, F, T = 4, 2, 256, 128, 12
    sel, w = _routing(T, E, k, "even", 4)
    gu, dn = _weights(E, H, F, "contiguous")
    x = torch.randn(T, H, device="cuda").to(BF)
    op = _operator(E, k, H)
    want = op.forward_few(x, sel, gu, dn, w)
    bad = x.clone()
    bad[5, 3], bad[7, 0] = float("nan"), float("inf")
    got = op.forward_few(bad, sel, gu, dn, w)
    keep = [t for t in range(T) if t not in (5, 7)]
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[5]).all()
    xq, xs, ex = _int8_inputs(T, E, H, F)
    want = op.forward_few_int8(xq, xs, sel, ex, w)
    xs[2] = float("nan")
    got = op.forward_few_int8(xq, xs, sel, ex, w)
    keep = [t for t in range(T) if t != 2]
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[2]).all()


@pytest.mark.parametrize("int8", [False, True])
def test_bits_do_not_depend_on_the_batch(int8):
    """A token's output is the same alone and with others, whatever tiles the
    sizes choose (16, 32 and 64 rows of an expert, 32 and 64 columns)."""
    for E, k, F in ((24, 3, 256), (4, 4, 256), (64, 8, 1024)):
        H, T = 384, 64
        sel, w = _routing(T, E, k, "drop", 8)
        op = _operator(E, k, H)
        if int8:
            x, xs, ex = _int8_inputs(T, E, H, F)
            run = lambda a, b: op.forward_few_int8(x[a:b], xs[a:b], sel[a:b], ex, w[a:b])
        else:
            gu, dn = _weights(E, H, F, "natural")
            x = torch.randn(T, H, device="cuda").to(BF)
            run = lambda a, b: op.forward_few(x[a:b], sel[a:b], gu, dn, w[a:b])
        full = run(0, T)
        for a, b in ((0, 1), (5, 21), (7, 40), (63, 64)):
            assert torch.equal(run(a, b), full[a:b]), (E, a, b)


def test_experts_past_32_bits():
    """Weight offsets beyond 2^31 elements: the last experts of a large table."""
    E, k, H, F = 260, 2, 4096, 1024
    gu = torch.zeros(E, H, 2 * F, dtype=BF, device="cuda")
    dn = torch.zeros(E, H, F, dtype=BF, device="cuda")
    small, sdn = _weights(2, H, F, "contiguous")
    gu[-2:], dn[-2:] = small, sdn
    x = torch.randn(3, H, device="cuda").to(BF)
    w = torch.rand(3, k, device="cuda")
    sel = torch.tensor([[0, 1], [1, 0], [0, 0]], dtype=torch.int32, device="cuda")
    got = _operator(E, k, H).forward_few(x, sel + (E - 2), gu, dn, w)
    assert torch.equal(got, _operator(2, k, H).forward_few(x, sel, small, sdn, w))
    del gu, dn
    q = mega_moe.Int8Experts.quantize(small, sdn)
    big = mega_moe.Int8Experts(*(torch.zeros(E, *t.shape[1:], dtype=t.dtype, device="cuda")
                                 for t in (q.gate_up, q.gate_up_scale, q.down, q.down_scale)))
    for name in ("gate_up", "gate_up_scale", "down", "down_scale"):
        getattr(big, name)[-2:] = getattr(q, name)
    xq, xs = mega_moe.quantize_rows(x)
    got = _operator(E, k, H).forward_few_int8(xq, xs, sel + (E - 2), big, w)
    assert torch.equal(got, _operator(2, k, H).forward_few_int8(xq, xs, sel, q, w))


def test_quantized_experts():
    """Int8Experts.quantize: every weight within half a step of its channel's scale."""
    E, H, F = 3, 256, 128
    for layout in ("natural", "contiguous"):
        gu, dn = _weights(E, H, F, layout)
        q = mega_moe.Int8Experts.quantize(gu, dn)
        for w, v, s in ((gu.transpose(1, 2), q.gate_up, q.gate_up_scale), (dn, q.down, q.down_scale)):
            assert torch.equal(s, (w.float().abs().amax(-1) / 127)) or \
                ((s - w.float().abs().amax(-1) / 127).abs() <= s * 2**-22).all()
            assert ((v.double() * s.double()[..., None] - w.double()).abs() <= s.double()[..., None] * 0.501).all()


def test_refusals():
    E, k, H, F = 4, 2, 256, 128
    sel, w = _routing(3, E, k, "even", 0)
    gu, dn = _weights(E, H, F, "natural")
    x = torch.randn(3, H, device="cuda").to(BF)
    op = mega_moe.FusedMoEForward(None, max_tokens_per_rank=80, hidden_size=H, top_k=k, num_experts=E)
    with pytest.raises(ValueError, match="at most 64"):
        op.forward_few(torch.zeros(65, H, dtype=BF, device="cuda"), torch.zeros(65, k, dtype=torch.int32, device="cuda"),
                       gu, dn, torch.zeros(65, k, device="cuda"))
    for args, err in (((x.float(), sel, gu, dn, w), TypeError), ((x[:, :128], sel, gu, dn, w), ValueError),
                      ((x, sel.long(), gu, dn, w), TypeError), ((x, sel, gu[:2], dn, w), ValueError),
                      ((x, sel, gu, dn[:, :, ::2], w), ValueError), ((x, sel, gu, dn, w.to(BF)), ValueError)):
        with pytest.raises(err):
            op.forward_few(*args)
    xq, xs, ex = _int8_inputs(3, E, H, F)
    other = _int8_inputs(3, E + 1, H, F)[2]
    for args, err in (((xq.float(), xs, sel, ex, w), TypeError), ((xq[:2], xs, sel, ex, w), ValueError),
                      ((xq, xs[:2], sel, ex, w), ValueError), ((xq, xs, sel, gu, w), TypeError),
                      ((xq, xs, sel, other, w), ValueError), ((xq, xs, sel, ex, w[:2]), ValueError)):
        with pytest.raises(err):
            op.forward_few_int8(*args)
    none = torch.zeros(0, k, dtype=torch.int32, device="cuda")
    assert op.forward_few(x[:0], none, gu, dn, w[:0]).shape == (0, H)
    assert op.forward_few_int8(xq[:0], xs[:0], none, ex, w[:0]).shape == (0, H)


def _block(op, s, ex, x, res, sel, w):
    """One decoding step's second half: norm, routed experts, a shared expert in int8."""
    q, sq, h = mega_moe.rms_norm(x, s["norm"], residual=res, out_dtype=I8)
    routed = op.forward_few_int8(q, sq, sel, ex, w)
    g, u = mega_moe.int8_matmul(q, s["up"], sq, s["up_scale"]).chunk(2, dim=-1)
    a, sa = mega_moe.quantize_rows(torch.nn.functional.silu(g) * u)
    return routed + mega_moe.int8_matmul(a, s["down"], sa, s["down_scale"]), h


def test_block_runs_together_and_in_graphs():
    """The operators as a decoding step runs them, against 64 bits; two graphs
    of different sizes replayed in turn, on streams of their own, beside eager work."""
    E, k, H, F, T = 16, 4, 512, 256, 24
    gu, dn = _weights(E, H, F, "natural")
    ex = mega_moe.Int8Experts.quantize(gu, dn)
    up, up_scale = mega_moe.quantize_rows((torch.randn(2 * F, H, device="cuda") * H**-0.5).to(BF))
    down, down_scale = mega_moe.quantize_rows((torch.randn(H, F, device="cuda") * F**-0.5).to(BF))
    s = dict(norm=torch.rand(H, device="cuda").to(BF) + 0.5, up=up, up_scale=up_scale, down=down, down_scale=down_scale)
    op = _operator(E, k, H)
    x, res = torch.randn(T, H, device="cuda").to(BF), torch.randn(T, H, device="cuda").to(BF)
    sel, w = _routing(T, E, k, "drop", 6)
    out, h = _block(op, s, ex, x, res, sel, w)
    # unquantised, in 64 bits: the 8-bit steps leave a relative error of about a percent
    hd = h.double()
    y = hd / (hd.square().mean(-1, keepdim=True) + 1e-6).sqrt() * s["norm"].double()
    ref, _ = _reference(y, None, sel, w, gu, None, dn, None, "swiglu")
    g, u = (y @ (up.double() * up_scale.double()[:, None]).t()).chunk(2, dim=-1)
    ref = ref + (g * torch.sigmoid(g) * u) @ (down.double() * down_scale.double()[:, None]).t()
    assert (out.double() - ref).norm() <= 0.05 * ref.norm()

    graphs = []
    for n in (T, 3):
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        args = [t[:n].clone() for t in (x, res, sel, w)]
        with torch.cuda.stream(st):
            _block(op, s, ex, *args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            got = _block(op, s, ex, *args)
        graphs.append((graph, st, args, got))
    for rep in range(4):
        for graph, st, args, got in graphs:
            args[0].copy_(torch.randn(args[0].shape, device="cuda"))
            args[2].copy_(_routing(args[2].shape[0], E, k, "drop", 20 + rep)[0])
        torch.cuda.synchronize()
        for graph, st, args, got in graphs:
            with torch.cuda.stream(st):
                graph.replay()
        eager = [_block(op, s, ex, *args) for _, _, args, _ in graphs]
        torch.cuda.synchronize()
        for (_, _, _, got), want in zip(graphs, eager):
            assert all(torch.equal(a, b) for a, b in zip(got, want)), rep


def test_few_between_forward_and_backward():
    """forward_few neither supersedes a saved pass nor touches its tables, on any stream."""
    E, k, H, F, T = 8, 2, 256, 128, 48
    sel, w = _routing(T, E, k, "even", 2)
    gu, dn = _weights(E, H, F, "natural")
    x, dy = torch.randn(T, H, device="cuda").to(BF), torch.randn(T, H, device="cuda").to(BF)
    op = _operator(E, k, H)
    _, saved = op.forward(x, sel, gu, dn, w, return_saved=True)
    want = {n: v.clone() for n, v in mega_moe.moe_backward_triton(saved, dy).items() if isinstance(v, torch.Tensor)}
    leaves = [x.requires_grad_(), w.requires_grad_()]
    out = mega_moe.MegaMoEFunction.apply(op, x, w, sel, gu, dn, torch.empty(0, device="cuda"), None)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        op.forward_few(x.detach(), sel, gu, dn, w.detach())
    grads = torch.autograd.grad(out, leaves, dy)
    torch.cuda.synchronize()
    assert torch.equal(grads[0], want["grad_hidden"]) and torch.equal(grads[1], want["grad_routing_weights"])
