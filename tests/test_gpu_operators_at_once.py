"""The operators next to the layer from several threads at once, and the norm's
backward past 2^31 elements."""

import threading

import pytest
import torch

import mega_moe

pytestmark = pytest.mark.gpu

BF, F32, I8 = torch.bfloat16, torch.float32, torch.int8


def _work(op, seed):
    """Inputs on the caller's stream, and one pass through every operator."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    T, H, F, E, k = 12, 512, 256, 8, 2
    x, res, w = rnd(300, 1000).to(BF), rnd(300, 1000), rnd(1000)
    dy = rnd(300, 1000).to(BF)
    rows, gu, dn = rnd(T, H).to(BF), (rnd(E, H, 2 * F) * H**-0.5).to(BF), (rnd(E, H, F) * F**-0.5).to(BF)
    sel = torch.rand(T, E, generator=g, device="cuda").argsort(1)[:, :k].to(torch.int32).contiguous()
    rw = torch.rand(T, k, generator=g, device="cuda")
    w8, w8_scale = mega_moe.quantize_rows(rnd(700, 1000).to(BF))

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, res)]
        y, h = mega_moe.rms_norm(leaves[0], leaves[1], residual=leaves[2])
        grads = torch.autograd.grad((y, h), leaves, (dy, torch.ones_like(h)))
        q, s, _ = mega_moe.rms_norm(x, w, residual=res, out_dtype=I8)
        return [y.detach(), *grads, q, s, mega_moe.int8_matmul(q, w8, s, w8_scale),
                op.forward_few(rows, sel, gu, dn, rw)]

    return step


def test_threads_on_streams_of_their_own():
    op = mega_moe.FusedMoEForward(None, max_tokens_per_rank=64, hidden_size=512, top_k=2, num_experts=8)
    steps = [_work(op, s) for s in range(4)]
    want = [step() for step in steps]
    torch.cuda.synchronize()
    got, errors = [[] for _ in steps], []

    def run(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
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
        assert len(outs) == 10
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_errors_stay_with_their_thread():
    """A refused call's message is its own thread's, beside calls that succeed."""
    from mega_moe import _lib

    x = torch.randn(4, 64, device="cuda").to(BF)
    wrong = []

    def run(code):
        fake = torch.empty(16, device="cuda")
        for _ in range(200):
            rc = _lib.load().mm_quantize_rows(_lib.ptr(fake), 8, code, 1, 8, _lib.ptr(fake), 3, None, None)
            if rc != -1 or b"null" not in _lib.load().mm_last_error():
                wrong.append(rc)
            mega_moe.quantize_rows(x)

    threads = [threading.Thread(target=run, args=(c,)) for c in (0, 1, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_norm_backward_past_32_bits():
    """Row offsets beyond 2^31 elements in the backward: only the last rows of a
    4.3 GB input have a gradient. dweight: two rows' terms and zeros."""
    rows, hidden = (1 << 20) + 3, 2056
    x = torch.zeros(rows, hidden, dtype=BF, device="cuda")
    dy = torch.zeros_like(x)
    g = torch.Generator(device="cuda").manual_seed(5)
    x[-2:] = torch.randn(2, hidden, generator=g, device="cuda").to(BF)
    dy[-2:] = torch.randn(2, hidden, generator=g, device="cuda").to(BF)
    w = torch.rand(hidden, generator=g, device="cuda") + 0.5
    few = [t[-2:].clone() for t in (x, dy)]
    leaves = [x.requires_grad_(), w.requires_grad_()]
    dx, dw = torch.autograd.grad(mega_moe.rms_norm(x, w), leaves, dy)
    small = [few[0].requires_grad_(), w]
    want = torch.autograd.grad(mega_moe.rms_norm(few[0], w), small, few[1])
    assert torch.equal(dx[-2:], want[0]) and not dx[-4:-2].any() and not dx[:2].any()
    # one addition of two terms, in fp32 whatever the order of the zeros
    assert ((dw - want[1]).abs() <= want[1].abs() * 2**-23).all()
