"""rms_norm and quantize_rows on the GPU against the same functions in 64 bits.

Tolerances (relative to the sums of absolute terms, counted in 64 bits):
  * a row's sum of squares is at most 32 products in one thread, then joined
    over at most 2^10 threads in a tree: under 64 roundings of 2^-24, so the
    mean is off by at most 2^-18 of itself and 1 / rms by 2^-19, plus a few
    2^-24 of the root, the products with weight and row: 2^-18 in all;
  * the backward's dot product has the same depth on terms of either sign: its
    error is 2^-18 of the sum of the absolute terms; with the products around
    it 2^-17 of |r w dy| + |h| r^3 mean|w dy h| + |dh|;
  * dweight adds a thread's rows (under 2^10 here), 4 waves, 32 of a share and 32 shares:
    2^-13 of the sum of the absolute terms bounds it;
  * each output is rounded once: half a step, or half the smallest subnormal.
"""

import pytest
import torch

import mega_moe

pytestmark = pytest.mark.gpu

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
E4M3 = torch.float8_e4m3fn
EPS = 1e-6


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _check(got, ref, slack, dtype, name):
    assert got.dtype == dtype, name
    bound = ref.abs() * _half(dtype) + slack * (1 + _half(dtype)) + _tiny(dtype)
    over = (got.double() - ref).abs() - bound
    assert not (over > 0).any(), f"{name}: {over.max().item():.3e} over the bound at {over.argmax().item()}"


def _make(rows, hidden, dtype, residual, weight, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, hidden, generator=g, device="cuda") * scale).to(dtype)
    res = None
    if residual is not None:
        res = (torch.randn(rows, hidden, generator=g, device="cuda") * 4 * scale).to(residual)
    w = None if weight is None else (1 + 0.3 * torch.randn(hidden, generator=g, device="cuda")).to(weight)
    return x, res, w, g


def _reference(x, res, w):
    h = x if res is None else (x.double() + res.double()).float().to(res.dtype)
    hd = h.double()
    r = 1 / (hd.square().mean(-1, keepdim=True) + EPS).sqrt()
    return h, hd, r, hd * r * (1.0 if w is None else w.double())


SHAPES = [(1, 1), (1, 7), (3, 8), (5, 63), (2, 512), (9, 513), (4, 1024), (7, 1021), (1, 2048), (65, 2048), (6, 2049),
          (3, 4099), (2, 8192), (3, 8193), (2, 16384), (1, 16391), (1, 32768)]


@pytest.mark.parametrize("dtype,residual,weight", [(BF, None, BF), (BF, BF, F32), (BF, F32, None), (F16, F16, F16),
                                                   (F16, F32, F32), (F32, F32, F32), (F32, None, BF)])
@pytest.mark.parametrize("rows,hidden", SHAPES)
def test_forward(rows, hidden, dtype, residual, weight):
    x, res, w, _ = _make(rows, hidden, dtype, residual, weight)
    out = mega_moe.rms_norm(x, w, residual=res, eps=EPS)
    h, _, _, y = _reference(x, res, w)
    if res is not None:
        out, got_h = out
        # x + residual is one fp32 addition, rounded to the residual's type: bit for bit
        assert torch.equal(got_h, (x.float() + res.float()).to(residual))
    _check(out, y, y.abs() * 2**-18, dtype, "y")


@pytest.mark.parametrize("out_dtype,most", [(torch.int8, 127.0), (E4M3, 448.0)])
@pytest.mark.parametrize("dtype,residual", [(BF, None), (BF, BF), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 7), (5, 513), (4, 2048), (2, 4099), (2, 8193), (1, 32768)])
def test_eight_bits(rows, hidden, dtype, residual, out_dtype, most):
    x, res, w, _ = _make(rows, hidden, dtype, residual, F32)
    got = mega_moe.rms_norm(x, w, residual=res, eps=EPS, out_dtype=out_dtype)
    h, _, _, y = _reference(x, res, w)
    _check_rows8(got[0], got[1], y, out_dtype, most)
    if res is not None:
        assert torch.equal(got[2], (x.float() + res.float()).to(residual))


def _check_rows8(q, scale, y, out_dtype, most):
    assert q.dtype == out_dtype and scale.dtype == F32 and scale.shape == y.shape[:-1]
    top = y.abs().amax(-1)
    want = torch.where(top > 0, top / most, torch.ones_like(top))
    assert ((scale.double() - want).abs() <= want * 2**-17).all()
    s = scale.double()[..., None]
    back = q.double() * s
    # half a step of the format, the step's place moved by y's own 2^-17
    step = s if out_dtype == torch.int8 else torch.maximum(y.abs() * 2.0**-3, s * 2.0**-9)
    assert ((back - y).abs() <= step * 0.5 * (1 + 2**-10) + y.abs() * 2**-16).all()
    if out_dtype == torch.int8:
        assert int(q.to(torch.int32).abs().max()) == (127 if (top > 0).any() else 0)


@pytest.mark.parametrize("dtype", [torch.int8, E4M3])
@pytest.mark.parametrize("shape", [(1, 1), (5, 300), (3, 5, 1030), (2, 20000)])
def test_quantize_rows(shape, dtype):
    x = torch.randn(*shape, device="cuda").to(BF)
    x[0] = 0
    q, scale = mega_moe.quantize_rows(x, dtype)
    assert q.shape == x.shape and scale.shape == x.shape[:-1]
    assert (scale[0] == 1).all() and not q[0].float().any()
    _check_rows8(q, scale, x.double(), dtype, 127.0 if dtype == torch.int8 else 448.0)


@pytest.mark.parametrize("hidden", [7, 64, 515, 2048, 7168, 16384])
@pytest.mark.parametrize("weight", [None, BF, F32])
def test_borders_round_to_even(hidden, weight):
    """Quotients that lie on a rounding border exactly, whatever the row's rms:
    whole numbers up to 254 in int8 (a scale of 2 times the row's), up to 448 in
    E4M3 (of 1). The weight's 1.5 is in every value and drops out."""
    g = torch.Generator(device="cuda").manual_seed(hidden)
    rows = 33
    w = None if weight is None else torch.full((hidden,), 1.5, dtype=weight, device="cuda")
    scale = 2.0 ** torch.randint(-9, 9, (rows, 1), generator=g, device="cuda")  # another rms a row
    for out, top, want in ((torch.int8, 254, lambda n: (n / 2).round()), (E4M3, 448, lambda n: n.to(E4M3).float())):
        n = torch.randint(-top, top + 1, (rows, hidden), generator=g, device="cuda").float()
        if out == E4M3:
            n = n.to(BF).float().clamp(-top, top)  # 8 bits: borders of 4 among them
        n[:, hidden // 2] = -top
        q, s = mega_moe.rms_norm((n * scale).to(BF), w, eps=EPS, out_dtype=out)
        assert torch.equal(q.float(), want(n))
        q, s = mega_moe.quantize_rows((n * scale).to(BF), out)
        assert torch.equal(q.float(), want(n)) and torch.equal(s, scale[:, 0] * (2 if out == torch.int8 else 1))


def test_tiny_rows_keep_their_scale_normal():
    x = torch.full((2, 64), 1e-37, device="cuda")
    x[1] = 1e-28
    q, scale = mega_moe.quantize_rows(x)
    assert torch.equal(scale[0], torch.tensor(1e-30 / 127, device="cuda")) and not q[0].any()
    assert (q[1] == 127).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_not_finite_rows(bad):
    x = torch.randn(4, 1000, device="cuda", dtype=BF)
    x[1, 999] = bad
    clean = x.clone()
    clean[1] = 0
    y, ref = mega_moe.rms_norm(x), mega_moe.rms_norm(clean)
    assert torch.equal(y[[0, 2, 3]], ref[[0, 2, 3]]) and torch.isnan(y[1, 999])
    for dtype in (torch.int8, E4M3):
        for q, s in (mega_moe.quantize_rows(x, dtype), mega_moe.rms_norm(x, out_dtype=dtype)):
            assert torch.isnan(s[1]) and torch.isfinite(s[[0, 2, 3]]).all() and not q[1].float().any()


def test_zero_rows_and_zero_row_calls():
    y, h = mega_moe.rms_norm(torch.zeros(2, 40, device="cuda", dtype=BF), residual=torch.zeros(2, 40, device="cuda", dtype=BF))
    assert not y.any() and not h.any()
    x = torch.empty(0, 40, device="cuda", dtype=BF, requires_grad=True)
    w = torch.ones(40, device="cuda", requires_grad=True)
    out = mega_moe.rms_norm(x, w)
    assert out.shape == (0, 40)
    dx, dw = torch.autograd.grad(out, (x, w), torch.empty(0, 40, device="cuda", dtype=BF))
    assert dx.shape == (0, 40) and not dw.any()
    q, s = mega_moe.quantize_rows(x.detach())
    assert q.shape == (0, 40) and s.shape == (0,)


@pytest.mark.parametrize("hidden", [129, 1024, 5000])
def test_strided_rows(hidden):
    base = torch.randn(6, hidden + 3, device="cuda").to(BF)
    x, res = base[::2, 1:hidden + 1], torch.randn(3, hidden + 5, device="cuda")[:, :hidden]
    w = torch.randn(hidden + 1, device="cuda").to(BF)[1:]
    got = mega_moe.rms_norm(x, w, residual=res)
    want = mega_moe.rms_norm(x.contiguous(), w.clone(), residual=res.contiguous())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    three = torch.randn(2, 3, hidden, device="cuda").to(BF)
    assert torch.equal(mega_moe.rms_norm(three, w).view(6, hidden), mega_moe.rms_norm(three.view(6, hidden), w))
    assert torch.equal(mega_moe.rms_norm(three[0, 0], w), mega_moe.rms_norm(three[0], w)[0])
    row = torch.randn(1, hidden, device="cuda").to(BF)
    assert torch.equal(mega_moe.rms_norm(row.expand(4, hidden), w), mega_moe.rms_norm(row, w).expand(4, hidden))


def test_refuses_layouts():
    x = torch.randn(4, 6, 64, device="cuda").to(BF)
    for bad in (x.transpose(0, 1), x.transpose(1, 2), x[..., ::2]):
        with pytest.raises(ValueError):
            mega_moe.rms_norm(bad)
    with pytest.raises(ValueError, match="same device"):
        mega_moe.rms_norm(x, torch.ones(64))


TRAIN = [(1, 1), (1, 8), (3, 13), (33, 512), (5, 1030), (70, 2048), (4100, 96), (9, 2305), (5, 8192), (3, 8195),
         (2, 32768), (5000, 640)]


@pytest.mark.parametrize("dtype,residual,weight", [(BF, None, BF), (BF, BF, BF), (BF, F32, F32), (F16, F16, F32),
                                                   (F16, F32, F16), (F32, F32, F32), (F32, None, F32)])
@pytest.mark.parametrize("rows,hidden", TRAIN)
def test_backward(rows, hidden, dtype, residual, weight):
    x, res, w, g = _make(rows, hidden, dtype, residual, weight, seed=3)
    dy = torch.randn(rows, hidden, generator=g, device="cuda").to(dtype)
    leaves = [t.requires_grad_() for t in (x, w, res) if t is not None]
    out = mega_moe.rms_norm(x, w, residual=res, eps=EPS)
    dh = None
    if res is None:
        grads = torch.autograd.grad(out, leaves, dy)
    else:
        dh = torch.randn(rows, hidden, generator=g, device="cuda").to(residual)
        grads = torch.autograd.grad(out, leaves, (dy, dh))
    with torch.no_grad():
        _, hd, r, _ = _reference(x, res, w)
        dyd, wd = dy.double(), w.double()
        t = dyd * wd
        c = r.pow(3) * (t * hd).mean(-1, keepdim=True)
        dx = r * t - hd * c + (0 if dh is None else dh.double())
        slack = (r * t).abs() + hd.abs() * r.pow(3) * (t * hd).abs().mean(-1, keepdim=True)
        slack = (slack + (0 if dh is None else dh.double().abs())) * 2**-17
        dw = (dyd * hd * r).sum(0)
        dw_slack = (dyd * hd * r).abs().sum(0) * 2**-13
    _check(grads[0], dx, slack, dtype, "dx")
    _check(grads[1], dw, dw_slack, weight, "dweight")
    if res is not None:
        _check(grads[2], dx, slack, residual, "dresidual")


def test_backward_against_differences():
    """fp32 operands; a difference of 2 d is off by d^2 of the third derivative
    (under 10 here: d = 2^-8 gives 2e-4) and by 2^-23 of the loss over d."""
    torch.manual_seed(1)
    x, res = torch.randn(3, 40, device="cuda"), torch.randn(3, 40, device="cuda")
    w, a, b = torch.rand(40, device="cuda") + 0.5, torch.randn(3, 40, device="cuda"), torch.randn(3, 40, device="cuda")
    leaves = [t.requires_grad_() for t in (x, w, res)]

    def loss():
        y, h = mega_moe.rms_norm(x, w, residual=res)
        return (y.double() * a.double()).sum() + (h.double() * b.double()).sum()

    grads = torch.autograd.grad(loss(), leaves)
    d = 2.0**-8
    with torch.no_grad():
        for leaf, grad in zip(leaves, grads):
            flat, gflat = leaf.view(-1), grad.reshape(-1)
            for i in (0, 7, flat.numel() - 1):
                keep = flat[i].item()
                flat[i] = keep + d
                up = loss().item()
                flat[i] = keep - d
                down = loss().item()
                flat[i] = keep
                assert abs((up - down) / (2 * d) - gflat[i].item()) < 5e-3 * (1 + abs(gflat[i].item()))


def test_partial_gradients():
    """Gradients that are absent, expanded, or of one output only."""
    x = torch.randn(6, 136, device="cuda", dtype=BF, requires_grad=True)
    w = torch.rand(136, device="cuda", requires_grad=True)
    res = torch.randn(6, 136, device="cuda", requires_grad=True)
    y, h = mega_moe.rms_norm(x, w, residual=res)
    gx, gr = torch.autograd.grad(h.sum(), (x, res), retain_graph=True)
    assert (gx == 1).all() and (gr == 1).all() and gx.dtype == BF and gr.dtype == F32
    ones = torch.autograd.grad(y, (x, w), torch.ones_like(y), retain_graph=True)
    summed = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)   # an expanded scalar
    assert all(torch.equal(a, b) for a, b in zip(ones, summed))
    turned = torch.autograd.grad(y, (x, w), torch.ones(136, 6, device="cuda", dtype=BF).t())
    assert all(torch.equal(a, b) for a, b in zip(ones, turned))
    # no weight, and the same tensor as x and residual
    z = torch.randn(4, 72, device="cuda", requires_grad=True)
    yz, hz = mega_moe.rms_norm(z, residual=z)
    (gz,) = torch.autograd.grad((yz, hz), z, (torch.ones_like(yz), torch.ones_like(hz)))
    z2 = (2 * z.detach()).double().requires_grad_()
    yref = z2 / (z2.square().mean(-1, keepdim=True) + EPS).sqrt()
    (gref,) = torch.autograd.grad((yref, z2 * 1), z2, (torch.ones_like(yref), torch.ones_like(yref)))
    assert ((gz.double() - 2 * gref).abs() <= 2**-14 * (1 + gref.abs())).all()
    with pytest.raises(RuntimeError):  # differentiable once
        (gy,) = torch.autograd.grad(mega_moe.rms_norm(z).sum(), z, create_graph=True)
        gy.sum().backward()


def test_repeats_bit_for_bit_and_in_a_graph():
    x, res, w, g = _make(700, 1500, BF, BF, BF, seed=9)
    dy, dh = torch.randn_like(x), torch.randn_like(x)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, res)]
        y, h = mega_moe.rms_norm(leaves[0], leaves[1], residual=leaves[2])
        q, s, _ = mega_moe.rms_norm(x, w, residual=res, out_dtype=torch.int8)
        return [y, h, q, s, *torch.autograd.grad((y, h), leaves, (dy, dh))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = [t.clone() for t in step()]
        again = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    del again
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    for rep in range(4):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), rep


def test_norm_and_layer_train_together():
    """norm -> layer -> residual, forward and backward, as a decoder block chains
    them: the block's gradients are the norm's backward of the layer's own, and a
    captured step repeats them."""
    T, E, k, H, F = 130, 6, 2, 256, 128
    x, res, w, g = _make(T, H, BF, BF, BF, seed=11)
    sel = torch.rand(T, E, generator=g, device="cuda").argsort(1)[:, :k].to(torch.int32).contiguous()
    rw = torch.rand(T, k, generator=g, device="cuda")
    gu = (torch.randn(E, H, 2 * F, generator=g, device="cuda") * H**-0.5).to(BF)
    dn = (torch.randn(E, H, F, generator=g, device="cuda") * F**-0.5).to(BF)
    dy = torch.randn(T, H, generator=g, device="cuda").to(BF)
    none = torch.empty(0, device="cuda")
    side = torch.cuda.Stream()

    def step(op):
        leaves = [t.detach().requires_grad_() for t in (x, w, res, rw, gu, dn)]
        y, h = mega_moe.rms_norm(leaves[0], leaves[1], residual=leaves[2], eps=EPS)
        out = h + mega_moe.MegaMoEFunction.apply(op, y, leaves[3], sel, *leaves[4:], none, None)
        return [out, *torch.autograd.grad(out, leaves, dy)]

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        op = mega_moe.FusedMoEForward(None, max_tokens_per_rank=T, hidden_size=H, top_k=k, num_experts=E,
                                      config=mega_moe.MoEForwardConfig())
        first = [t.detach().clone() for t in step(op)]
        # the same in two pieces: the layer's gradients from its own call, the norm's in 64 bits
        y, h = mega_moe.rms_norm(x, w, residual=res, eps=EPS)
        leaves = [t.detach().requires_grad_() for t in (y, rw, gu, dn)]
        out = mega_moe.MegaMoEFunction.apply(op, leaves[0], leaves[1], sel, *leaves[2:], none, None)
        part = torch.autograd.grad(out, leaves, dy)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first[4:], part[1:]))
    _, hd, r, _ = _reference(x, res, w)
    t, dyd = part[0].double() * w.double(), part[0].double()
    dx = r * t - hd * r.pow(3) * (t * hd).mean(-1, keepdim=True) + dy.double()
    slack = ((r * t).abs() + hd.abs() * r.pow(3) * (t * hd).abs().mean(-1, keepdim=True) + dy.double().abs()) * 2**-17
    _check(first[1], dx, slack, BF, "dx")
    _check(first[3], dx, slack, BF, "dresidual")
    _check(first[2], (dyd * hd * r).sum(0), (dyd * hd * r).abs().sum(0) * 2**-13, BF, "dweight")
    del out, leaves, y, h, part
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step(op)
    for rep in range(3):
        x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = [t.detach().clone() for t in step(op)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), rep


def test_a_captured_backward_beside_an_eager_graph_is_refused():
    """A graph built on the default stream keeps its leaves' nodes on that stream,
    which no capture can reach: the backward raises before the hand-over, the
    capture stays whole, and without that graph the same steps are captured."""
    x = torch.randn(5, 264, device="cuda", requires_grad=True)
    w = torch.rand(264, device="cuda", requires_grad=True)
    dy = torch.randn(5, 264, device="cuda")
    alive = mega_moe.rms_norm(x, w)
    want = [alive.detach().clone(), *torch.autograd.grad(alive, (x, w), dy, retain_graph=True)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = mega_moe.rms_norm(x, w)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            torch.autograd.grad(y, (x, w), dy)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want[0])
    del alive, y, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = mega_moe.rms_norm(x, w)
        got = [y, *torch.autograd.grad(y, (x, w), dy)]
    for _ in range(3):
        for t in got:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # not refused: no capture, and the eager graph alive
    alive = mega_moe.rms_norm(x, w)
    with torch.cuda.stream(side):
        y = mega_moe.rms_norm(x, w)
        got = torch.autograd.grad(y, (x, w), dy)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1:]))


def test_rows_past_32_bits():
    """Row offsets beyond 2^31 elements: the last rows of a 4.3 GB input."""
    rows, hidden = (1 << 20) + 3, 2056
    x = torch.zeros(rows, hidden, dtype=BF, device="cuda")
    x[-2:] = torch.randn(2, hidden, device="cuda").to(BF)
    y = mega_moe.rms_norm(x)
    assert torch.equal(y[-2:], mega_moe.rms_norm(x[-2:].clone())) and not y[-4:-2].any()
