"""The E4M3 operators as they are used: run together, captured, from several
streams at once, past 32-bit offsets, and the layer's refusals and long runs of tiles."""

import threading

import pytest
import torch

import mega_moe
from tests import _fp8 as R
from tests.test_gpu_fp8_layer import make, operator, reference

pytestmark = pytest.mark.gpu

BF, F32, F8, E8 = torch.bfloat16, torch.float32, R.F8, R.E8


# ------------------------------------------------------------------ together
def _serving(seed, T=40, H=384, I=256, E=8, k=2, N=520):
    """Inputs, and one block of a model on them: a norm to E4M3 rows, a projection
    of them, the experts, and blocks of what comes out."""
    x, sx, sel, ex, w = make(T, H, I, E, k, seed=seed, drop=0.1)
    gen = torch.Generator().manual_seed(seed + 50)
    hidden = torch.randn(T, H, generator=gen).to(BF).cuda()
    stream = torch.randn(T, H, generator=gen).cuda()
    weight, scale = mega_moe.quantize_blocks((torch.randn(N, H, generator=gen) * 0.1).to(BF).cuda(), rows=128)
    bias = torch.randn(N, generator=gen).cuda()
    op = operator(T, H, k, E)

    def step():
        q, s, h = mega_moe.rms_norm(hidden, residual=stream, out_dtype=F8, scale_columns=128)
        y = mega_moe.fp8_matmul(q, weight, s, scale, bias=bias)
        wide = mega_moe.fp8_matmul(q, weight, s, scale, out_dtype=F32)
        out = op.forward_fp8(q, s, sel, ex, w)
        return [q.view(torch.uint8), s.view(torch.uint8), h, y, wide, out,
                *(t.view(torch.uint8) for t in mega_moe.quantize_blocks(out))]

    return step, hidden, (stream, weight, scale, bias, sel, ex, w)


def test_a_block_of_a_model():
    step, hidden, (stream, weight, scale, bias, sel, ex, w) = _serving(1)
    q, s, h, y, wide, out, q2, s2 = step()
    h64 = (hidden.float() + stream).double().cpu()
    assert torch.equal(h.double().cpu(), h64)
    normed = h64 / (h64.square().mean(1, keepdim=True) + 1e-6).sqrt()
    q, s = q.view(F8), s.view(E8)
    held = R.values(q.cpu(), s.cpu(), 1)
    # a scale is a power of two up to twice what would do, E4M3 steps are 2^-3 and the smallest 2^-9: the
    # fp32 norm moves a value by less than 2^-20, which may carry it over a border to the step next to it
    top = normed.abs().unflatten(1, (-1, 128)).amax(2).repeat_interleave(128, 1)
    R.near(held, normed, 2.0 ** -4 * (1 + 2.0 ** -15) * normed.abs() + 2.0 ** -10 * top / 224)
    b = R.values(weight.cpu(), scale.cpu(), 128)
    ref, off = held @ b.t(), R.sum_error(held, b)
    biased = ref + bias.double().cpu()
    R.near(y, biased, off + R.half_step(BF) * (biased.abs() + off) + 2.0 ** -23 * biased.abs())
    off = R.sum_error(held, b, wide=True)
    R.near(wide, ref, off + R.half_step(F32) * (ref.abs() + off))
    R.near(out, *reference(q, s, sel, ex, w, "swiglu"))
    want = R.quant(out.double().cpu(), 1)
    assert torch.equal(q2.view(F8).double().cpu(), want[0]) and torch.equal(s2.view(E8).double().cpu(), want[1])


def _training(seed, m=150, k=260, n=200):
    """A norm in front of two projections of its output, one in the norm's type and
    one with its weight in 32 bits, and their sum's gradients."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, scale, a, b = rnd(m, k).to(BF), rnd(k).to(BF), (rnd(n, k) * 0.1).to(BF), rnd(n, k) * 0.1
    dy = rnd(m, n).to(BF)

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, scale, a, b)]
        h = mega_moe.rms_norm(leaves[0], leaves[1])
        y = mega_moe.fp8_linear(h, leaves[2]) + mega_moe.fp8_linear(h, leaves[3])
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    return step, x, (scale, a, b, dy)


def test_norm_and_projections_train_together():
    """The chain's gradients are those of its parts."""
    step, x, (scale, a, b, dy) = _training(3)
    y, dx, ds, da, db = step()
    h = mega_moe.rms_norm(x, scale).requires_grad_()
    parts = []
    for w in (a, b):
        leaf = w.detach().requires_grad_()
        out = mega_moe.fp8_linear(h, leaf)
        parts.append((out.detach(), *torch.autograd.grad(out, (h, leaf), dy)))
    assert torch.equal(y, parts[0][0] + parts[1][0])
    assert torch.equal(da, parts[0][2]) and torch.equal(db, parts[1][2])
    leaves = [t.detach().requires_grad_() for t in (x, scale)]
    # autograd adds the two in bf16, in either order
    want = torch.autograd.grad(mega_moe.rms_norm(*leaves), leaves, parts[0][1] + parts[1][1])
    assert torch.equal(dx, want[0]) and torch.equal(ds, want[1])


def test_gradients_accumulate_and_follow_updates():
    """Weight and input may change behind the call: what the backward reads is kept."""
    x = torch.randn(70, 150, device="cuda", requires_grad=True)
    w = torch.randn(90, 150, device="cuda", requires_grad=True)
    dy = torch.randn(70, 90, device="cuda")
    want = torch.autograd.grad(mega_moe.fp8_linear(x, w), (x, w), dy)
    for _ in range(2):
        y = mega_moe.fp8_linear(x, w)
        y.backward(dy)
    assert torch.equal(x.grad, want[0] + want[0]) and torch.equal(w.grad, want[1] + want[1])
    y = mega_moe.fp8_linear(x, w)
    with torch.no_grad():
        x.mul_(2)
        w.zero_()
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(y, (x, w), dy), want))


@pytest.mark.parametrize("layout", ["expanded", "transposed", "strided"])
def test_incoming_gradients_of_any_layout(layout):
    x = torch.randn(70, 150, device="cuda", dtype=BF, requires_grad=True)
    w = torch.randn(90, 150, device="cuda", dtype=BF, requires_grad=True)
    dy = {"expanded": lambda: torch.tensor(0.5, device="cuda", dtype=BF).expand(70, 90),
          "transposed": lambda: torch.randn(90, 70, device="cuda").to(BF).t(),
          "strided": lambda: torch.randn(70, 180, device="cuda").to(BF)[:, ::2]}[layout]()
    got = torch.autograd.grad(mega_moe.fp8_linear(x, w), (x, w), dy)
    want = torch.autograd.grad(mega_moe.fp8_linear(x, w), (x, w), dy.contiguous())
    assert all(torch.equal(p, q) for p, q in zip(got, want))


# ------------------------------------------------------------------ captured
@pytest.mark.parametrize("make_step", [_serving, _training])
def test_captured_and_replayed(make_step):
    step, x, _ = make_step(5)
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
        x.copy_(torch.randn(x.shape, device="cuda"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), rep


def test_two_graphs_of_different_sizes():
    """Each capture holds workspaces of its own: replays in turn do not meet."""
    made = [_serving(7), _serving(8, T=3), _serving(9, T=200, E=4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for step, *_ in made:
            step()
    torch.cuda.synchronize()
    graphs = []
    for step, *_ in made:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            graphs.append((graph, step()))
    for rep in range(3):
        for _, x, _ in made:
            x.copy_(torch.randn(x.shape, device="cuda"))
        torch.cuda.synchronize()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (step, *_), (_, outs) in zip(made, graphs):
            assert all(torch.equal(a, b) for a, b in zip(outs, step())), rep


def test_a_captured_backward_beside_an_eager_graph_is_refused():
    x = torch.randn(5, 264, device="cuda", requires_grad=True)
    w = torch.randn(70, 264, device="cuda", requires_grad=True)
    dy = torch.randn(5, 70, device="cuda")
    alive = mega_moe.fp8_linear(x, w)
    want = [alive.detach().clone(), *torch.autograd.grad(alive, (x, w), dy, retain_graph=True)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = mega_moe.fp8_linear(x, w)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            torch.autograd.grad(y, (x, w), dy)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want[0])
    del alive, y, graph
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = mega_moe.fp8_linear(x, w)
        got = [y, *torch.autograd.grad(y, (x, w), dy)]
    for _ in range(3):
        for t in got:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ------------------------------------------------------------------ at once
def test_threads_on_streams_of_their_own():
    steps = [_serving(s)[0] for s in (11, 12)] + [_training(s)[0] for s in (13, 14)]
    want = [step() for step in steps]
    torch.cuda.synchronize()
    got, errors = [[] for _ in steps], []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(8):
                    got[i].append(steps[i]())
            stream.synchronize()
        except Exception as e:  # reported by the test's own thread
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(steps))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for outs, ref in zip(got, want):
        assert len(outs) == 8
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_one_operator_on_two_streams():
    """The layer keeps nothing between calls: one operator serves two streams at once."""
    x, sx, sel, ex, w = make(150, 256, 128, 4, 2, seed=21)
    op = operator(150, 256, 2, 4)
    sizes = (150, 1, 64, 17)
    want = [op.forward_fp8(x[:t], sx[:t], sel[:t], ex, w[:t]) for t in sizes]
    streams = [torch.cuda.Stream() for _ in sizes]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        for t, s in zip(sizes, streams):
            with torch.cuda.stream(s):
                got.append(op.forward_fp8(x[:t], sx[:t], sel[:t], ex, w[:t]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 4]) for i, g in enumerate(got))


# ------------------------------------------------------------------ the layer
LAYERS = [  # tokens, hidden, inter, experts, top_k
    (1300, 256, 512, 128, 2),  # 512 tiles of FC1: two for each workgroup
    (800, 128, 128, 40, 1),    # one block of K in either product, a workgroup for a tile
    (1100, 384, 1152, 30, 3),  # 9 and 2 runs of channels, the last one of H half full
    (640, 512, 896, 130, 4),   # 20 rows an expert
    (640, 512, 1024, 140, 4),  # 220 MB of weights, which pass the caches by
    (150, 512, 1024, 140, 4),  # the same for few rows
    (1500, 256, 512, 16, 6),   # 560 rows an expert
    (2000, 256, 256, 12, 1),   # 167 rows an expert: two tiles each
]


@pytest.mark.parametrize("size", LAYERS)
def test_layer_over_many_tiles(size):
    T, H, I, E, k = size
    ops = make(T, H, I, E, k, seed=T + I, drop=0.05)
    R.near(operator(T, H, k, E).forward_fp8(*ops), *reference(*ops, "swiglu"))


FEW = [  # one for each way in which few activations are summed, and one past a tile's part of 64 rows
    (1, 256, 128, 8, 2), (30, 1024, 384, 16, 4), (16, 640, 256, 2, 2),
    (300, 384, 256, 60, 4), (900, 256, 384, 24, 2),
    (200, 384, 256, 6, 4), (420, 512, 128, 3, 1), (700, 256, 256, 2, 2),
]


@pytest.mark.parametrize("size", FEW)
@pytest.mark.parametrize("act", ["swiglu", "clamp_swiglu", "situglu"])
def test_few_activations_are_summed_in_32_bits(size, act):
    """An activation leaves its E4M3 step only where fp32 sums can carry it there."""
    T, H, I, E, k = size
    ops = make(T, H, I, E, k, seed=T * I)
    R.near(operator(T, H, k, E, act).forward_fp8(*ops), *reference(*ops, act, wide=True))


def test_layer_of_uneven_experts():
    """Experts of no row, one row and hundreds in one call, and rows of zeros."""
    T, H, I, E, k = 900, 256, 256, 20, 2
    x, sx, sel, ex, w = make(T, H, I, E, k, seed=31)
    sel[:] = torch.randint(5, 8, sel.shape, generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    sel[0, 0], sel[1, 1], sel[2:40, 0] = 0, 19, 9
    x[3:9] = 0
    w[50] = 0
    out = operator(T, H, k, E).forward_fp8(x, sx, sel, ex, w)
    R.near(out, *reference(x, sx, sel, ex, w, "swiglu"))
    assert not out[50].any()


def test_layer_refuses():
    x, sx, sel, ex, w = make(6, 128, 128, 4, 2)
    op = operator(8, 128, 2, 4)
    other = make(6, 256, 128, 4, 2)[3]
    few = make(6, 128, 128, 3, 2)[3]
    flat = torch.zeros(6 * 128 + 16, dtype=torch.uint8, device="cuda").view(F8)
    big = make(9, 128, 128, 4, 2)
    for args, err, match in (
            ((x.to(BF), sx, sel, ex, w), TypeError, "float8_e4m3fn"),
            ((x[:5], sx, sel, ex, w), ValueError, "tokens"),
            ((x.t().contiguous().t(), sx, sel, ex, w), ValueError, "tokens"),
            ((x, torch.ones(6, 1, device="cuda"), sel, ex, w), ValueError, "token_scale"),
            ((x, sx[:5], sel, ex, w), ValueError, "token_scale"),
            ((x, sx, sel, other, w), ValueError, "experts hold"),
            ((x, sx, sel, few, w), ValueError, "experts hold"),
            ((x, sx, sel.long(), ex, w), TypeError, "int32|Int32|INT32"),
            ((x, sx, sel, ex, w[:, :1]), ValueError, "routing_weights"),
            ((x, sx, sel, ex, w.to(BF)), ValueError, "routing_weights"),
            ((x, sx, sel, ex, w.cpu()), ValueError, "routing_weights"),
            ((x.cpu(), sx, sel, ex, w), ValueError, "same device"),
            ((flat[8:8 + 6 * 128].view(6, 128), sx, sel, ex, w), ValueError, "aligned"),
            ((*big[:3], ex, big[4]), ValueError, "max_tokens|exceed|at most")):
        with pytest.raises(err, match=match):
            op.forward_fp8(*args)
    R.near(op.forward_fp8(x, sx, sel, ex, w), *reference(x, sx, sel, ex, w, "swiglu"))


# ------------------------------------------------------------------ large
def test_blocks_past_32_bits():
    """Offsets beyond 2^31 elements: the last rows of a 4.6 GB input."""
    x = torch.zeros(280003, 8200, dtype=BF, device="cuda")
    x[-3:] = torch.randn(3, 8200, device="cuda").to(BF)
    want = mega_moe.quantize_blocks(x[-3:].clone())
    q, s = mega_moe.quantize_blocks(x)
    assert torch.equal(q[-3:].view(torch.uint8), want[0].view(torch.uint8))
    assert torch.equal(s[-3:].view(torch.uint8), want[1].view(torch.uint8))
    assert not q[-300:-3].view(torch.uint8).any() and (s[-300:-3].view(torch.uint8) == 127).all()
    want = mega_moe.quantize_blocks(x[-67:].clone(), rows=128)  # 280003 = 67 more than whole blocks
    q, s = mega_moe.quantize_blocks(x, rows=128)
    assert torch.equal(q[-67:].view(torch.uint8), want[0].view(torch.uint8))
    assert torch.equal(s[-1:].view(torch.uint8), want[1].view(torch.uint8))


def test_products_past_32_bits():
    """Rows and columns behind 2^31 bytes of an operand, and outputs behind 2^31."""
    gen = torch.Generator().manual_seed(41)
    K, M = 8192, 270003
    a = torch.zeros(M, K, dtype=torch.uint8, device="cuda").view(F8)
    sa = torch.full((M, K // 128), 127, dtype=torch.uint8, device="cuda").view(E8)
    tail, tail_scale = R.rows_e4m3(gen, 5, K)
    a.view(torch.uint8)[-5:] = tail.view(torch.uint8)
    sa.view(torch.uint8)[-5:] = tail_scale.view(torch.uint8)
    b, sb = R.blocks_e4m3(gen, 130, K)
    want = mega_moe.fp8_matmul(tail, b, tail_scale, sb, out_dtype=F32)
    got = mega_moe.fp8_matmul(a, b, sa, sb, out_dtype=F32)
    rv, bv = R.values(tail.cpu(), tail_scale.cpu(), 1), R.values(b.cpu(), sb.cpu(), 128)
    off = R.sum_error(rv, bv, wide=True)
    R.near(want, rv @ bv.t(), off + R.half_step(F32) * ((rv @ bv.t()).abs() + off))
    R.near(got[-5:], rv @ bv.t(), off + R.half_step(F32) * ((rv @ bv.t()).abs() + off))
    assert not got[:-5].any()
    # the same rows as channels: a tensor of scales for the last block of 128
    square = torch.full((R.ceil(M, 128), K // 128), 127, dtype=torch.uint8, device="cuda").view(E8)
    rows, rows_scale = R.rows_e4m3(gen, 3, K)
    got = mega_moe.fp8_matmul(rows, a, rows_scale, square)
    xv, cv = R.values(rows.cpu(), rows_scale.cpu(), 1), tail.double().cpu()
    off = R.sum_error(xv, cv)
    R.near(got[:, -5:], xv @ cv.t(), off + R.half_step(BF) * ((xv @ cv.t()).abs() + off))
    assert not got[:, :-5].any()


def test_linear_past_32_bits():
    """A training step on 2.4e9 values: only the last block's rows are not zero."""
    m, k, n = 128 * 4700 + 3, 4096, 8
    x = torch.zeros(m, k, dtype=BF, device="cuda")
    dy = torch.zeros(m, n, dtype=BF, device="cuda")
    x[-3:], dy[-3:] = torch.randn(3, k, device="cuda").to(BF), torch.randn(3, n, device="cuda").to(BF)
    w = (torch.randn(n, k, device="cuda") * 0.1).to(BF).requires_grad_()
    few = x[-3:].clone().requires_grad_()
    few_y = mega_moe.fp8_linear(few, w)
    want = torch.autograd.grad(few_y, (few, w), dy[-3:].clone())
    x.requires_grad_()
    y = mega_moe.fp8_linear(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    # tiles may differ, and with them the order of fp32 sums and the side on which a result is rounded
    y = y.detach()
    off = R.half_step(BF) * 2
    R.near(y[-3:], few_y.detach(), off * few_y.detach().abs() + 1e-3 * few_y.detach().abs().max())
    R.near(dx[-3:], want[0], off * want[0].abs() + 1e-3 * want[0].abs().max())
    R.near(dw, want[1], off * want[1].abs() + 1e-3 * want[1].abs().max())
    assert not y[:-3].any() and not dx[:-3].any()


def test_layer_past_32_bits():
    """Expert outputs of 5.1 GB and rows behind 2^29 bytes: the last tokens."""
    T, H, I, E, k = 78000, 8192, 128, 8, 2
    x, sx, sel, ex, w = make(64, H, I, E, k, seed=51)
    reps = R.ceil(T, 64)
    many = [t.view(torch.uint8) if t.dtype in (F8, E8) else t for t in (x, sx, sel, w)]
    many = [t.repeat(reps, 1)[:T].contiguous() for t in many]
    out = operator(T, H, k, E).forward_fp8(many[0].view(F8), many[1].view(E8), many[2], ex, many[3])
    ref, bound = reference(x, sx, sel, ex, w, "swiglu")
    at = torch.arange(T - 64, T) % 64
    R.near(out[-64:], ref[at], bound[at])
    assert torch.equal(out[: 64 * (reps - 1)].view(reps - 1, 64, H), out[:64].expand(reps - 1, 64, H))


# ------------------------------------------------------------------ what is not a number, and nothing
@pytest.mark.parametrize("size", [(6, 256, 128, 4, 2), (400, 384, 256, 16, 2), (640, 512, 896, 130, 4), (200, 256, 128, 4, 2),
                                  (1500, 256, 512, 16, 6)])
def test_layer_keeps_bad_tokens_to_themselves(size):
    """A NaN byte, a NaN scale and infinite weights in a token, on each of the layer's ways."""
    T, H, I, E, k = size
    x, sx, sel, ex, w = make(T, H, I, E, k, seed=61)
    op = operator(T, H, k, E)
    clean = op.forward_fp8(x, sx, sel, ex, w)
    x.view(torch.uint8)[1, 77] = 0x7F
    sx.view(torch.uint8)[2, 1] = 255
    w[3, 0] = float("nan")
    w[4, k - 1] = float("inf")
    out = op.forward_fp8(x, sx, sel, ex, w)
    assert out[1].isnan().all() and out[2].isnan().all() and out[3].isnan().all() and out[4].isnan().all()
    rest = [0, *range(5, T)]
    assert torch.equal(out[rest], clean[rest])


def test_layer_keeps_a_bad_expert_to_its_tokens():
    T, H, I, E, k = 300, 256, 256, 8, 2
    x, sx, sel, ex, w = make(T, H, I, E, k, seed=62)
    op = operator(T, H, k, E)
    clean = op.forward_fp8(x, sx, sel, ex, w)
    ex.down_scale.view(torch.uint8)[3, 1, 0] = 255  # columns 128-255 of what expert 3 gives
    out = op.forward_fp8(x, sx, sel, ex, w)
    hit = (sel == 3).any(1)
    assert out[hit][:, 128:].isnan().all() and torch.equal(out[hit][:, :128], clean[hit][:, :128])
    assert torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("m", [5, 40, 400])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_product_of_nan_bytes(m, dtype):
    gen = torch.Generator().manual_seed(63)
    a, sa = R.rows_e4m3(gen, m, 300)
    b, sb = R.blocks_e4m3(gen, 200, 300)
    clean = mega_moe.fp8_matmul(a, b, sa, sb, out_dtype=dtype)
    a.view(torch.uint8)[2, 299] = 0xFF
    b.view(torch.uint8)[7, 0] = 0x7F
    out = mega_moe.fp8_matmul(a, b, sa, sb, out_dtype=dtype)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[2], bad[:, 7] = True, True
    assert torch.equal(out.isnan(), bad) and torch.equal(out[~bad], clean[~bad])


def test_nothing():
    """No rows, no columns, no matrices."""
    empty = lambda *s: torch.empty(*s, dtype=BF, device="cuda")
    for shape, rows, scales in (((0, 300), 1, (0, 3)), ((5, 0), 1, (5, 0)), ((0, 300), 128, (0, 3)), ((300, 0), 128, (3, 0)),
                                ((0, 4, 300), 128, (0, 1, 3)), ((2, 0, 7), 1, (2, 0, 1))):
        q, s = mega_moe.quantize_blocks(empty(*shape), rows)
        assert q.shape == shape and s.shape == scales and q.dtype == F8 and s.dtype == E8
    q, s = mega_moe.rms_norm(empty(0, 300), out_dtype=F8, scale_columns=128)
    assert q.shape == (0, 300) and s.shape == (0, 3)
    gen = torch.Generator().manual_seed(64)
    b, sb = R.blocks_e4m3(gen, 200, 300)
    assert mega_moe.fp8_matmul(q, b, s, sb, out_dtype=F32).shape == (0, 200)
    assert mega_moe.fp8_linear(empty(0, 300), empty(40, 300)).shape == (0, 40)
    assert mega_moe.fp8_linear(empty(300), empty(40, 300)).shape == (40,)


# ------------------------------------------------------------------ products in tiles of 64 x 128
@pytest.mark.parametrize("m,n,k", [(1000, 1900, 2100), (1000, 1899, 2101), (1793, 2305, 1000), (960, 1920, 257)])
@pytest.mark.parametrize("dtype,bias", [(BF, None), (torch.float16, F32), (F32, BF)])
def test_product_of_a_thousand_rows(m, n, k, dtype, bias):
    gen = torch.Generator().manual_seed(m + k)
    a, sa = R.rows_e4m3(gen, m, k, low=-8, high=-4)
    b, sb = R.blocks_e4m3(gen, n, k, low=-8, high=-4)
    add = None if bias is None else torch.randn(n, generator=gen).to(bias).cuda()
    av, bv = R.values(a, sa, 1), R.values(b, sb, 128)
    ref, off = av @ bv.t(), R.sum_error(av, bv, wide=dtype == F32)
    if bias is not None:
        ref = ref + add.double()
        off = off + 2.0 ** -23 * (ref.abs() + off)
    got = mega_moe.fp8_matmul(a, b, sa, sb, bias=add, out_dtype=dtype)
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    R.near(got, ref, off + R.half_step(dtype) * (ref.abs() + off) + tiny)
