"""Products in 8-bit floating point with a scale for each block of 128: the calls whose time is measured.

A value is held as E4M3 times its block's scale, a power of two in one byte:
blocks are 128 columns of a row (activations) or 128 x 128 (weights). Every
case is one pass through a public entry point (``own``) or the same mathematics
in elementary torch operations in 32 bits. Sizes are those of the layer
configurations in ``mega_moe/bench_configs.py`` and of the tests, or generic
ones between them.

Kinds of case:
  quant        quantize_blocks: rows or 128 x 128 blocks to E4M3
  matmul       fp8_matmul on rows and weights that are in E4M3
  linear       fp8_linear forward and backward: a training step's projection,
               whose input is kept in E4M3 and read again by the weight gradient
  moe          FusedMoEForward.forward_fp8: the expert layer on E4M3 rows
  block        rms_norm with a residual to E4M3 rows, then the expert layer
"""

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mega-moe-td_amd")
_EPS = 1e-6
_B = 128  # values of a block along a row
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_F8, _E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _quant(name, rows, cols, block_rows, dtype="bf16"):
    c = dict(kind="quant", rows=rows, cols=cols, block_rows=block_rows, dtype=dtype)
    return dict(c, name=name) if name else c


def _matmul(name, rows, k, n, dtype="bf16", bias=False):
    c = dict(kind="matmul", rows=rows, k=k, n=n, dtype=dtype, bias=bias)
    return dict(c, name=name) if name else c


def _linear(name, rows, k, n, dtype="bf16", weight="same"):
    c = dict(kind="linear", rows=rows, k=k, n=n, dtype=dtype, weight=weight)
    return dict(c, name=name) if name else c


def _moe(name, kind, tokens, hidden, inter, experts, top_k, act="swiglu", drop=0.0):
    c = dict(kind=kind, tokens=tokens, hidden=hidden, inter=inter, experts=experts, top_k=top_k, act=act, drop=drop)
    return dict(c, name=name) if name else c


def listed():
    return [
        # a prompt chunk of a wide layer into 8 bits
        _quant("quant_prompt", 8192, 7168, 1),
        # a weight of odd sizes, kept in 32 bits by its optimizer
        _quant("quant_weight_ragged", 2305, 1793, 128, dtype="fp32"),
        # generation for one user: a projection of a wide layer
        _matmul("matmul_token", 1, 7168, 4096),
        # generation for a batch of users
        _matmul("matmul_batch", 64, 7168, 4096),
        # a short prompt, sizes that no block divides
        _matmul("matmul_ragged", 1021, 2309, 1793, dtype="fp16", bias=True),
        # a prompt chunk
        _matmul("matmul_prompt", 8192, 7168, 4096),
        # training: a projection's forward and both gradients, a full micro-batch
        _linear("linear_train", 8192, 4096, 4096),
        # training on odd sizes, the weight in 32 bits
        _linear("linear_train_ragged", 1021, 2305, 1793, weight="fp32"),
        # generation for one user: the expert layer
        _moe("moe_one", "moe", 1, 2048, 768, 128, 8),
        # several short prompts: some 30 rows an expert, a tenth of the routes dropped
        _moe("moe_mid", "moe", 512, 2048, 768, 128, 8, act="clamp_swiglu", drop=0.1),
        # generation for a batch on a wide layer, from the residual stream
        _moe("block_batch", "block", 32, 7168, 2048, 64, 8),
        # a prompt chunk on a wide layer of many experts, from the residual stream
        _moe("block_prompt", "block", 4096, 7168, 2048, 256, 8),
    ]


_MOST_QUANT = 8192 * 7168
_MOST_MATMUL = 8192 * 7168 * 4096
_MOST_LINEAR = 8192 * 4096 * 4096
_MOST_WEIGHTS = 256 * 7168 * 2048
_MOST_ROUTED = 4096 * 8 * 7168 * 2048


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["quant", "matmul", "matmul", "linear", "moe", "moe", "block"])
        if kind == "quant":
            rows, cols = _log_int(rng, 1, 16384), _log_int(rng, 64, 8192)
            if rows * cols > _MOST_QUANT:
                continue
            return _quant(None, rows, cols, rng.choice([1, 128]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        if kind in ("matmul", "linear"):
            rows, k, n = _log_int(rng, 1, 8192), _log_int(rng, 256, 8192), _log_int(rng, 256, 8192)
            if rng.random() < 0.5:
                k, n = _B * -(-k // _B), _B * -(-n // _B)
            if rows * k * n > (_MOST_MATMUL if kind == "matmul" else _MOST_LINEAR):
                continue
            if kind == "linear":
                return _linear(None, rows, k, n, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                               weight=rng.choice(["same", "fp32"]))
            return _matmul(None, rows, k, n, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                           bias=rng.random() < 0.3)
        experts = _log_int(rng, 8, 256)
        top_k = rng.choice([v for v in (1, 2, 4, 6, 8, 16) if v <= experts])
        hidden, inter, tokens = 256 * _log_int(rng, 1, 28), 128 * _log_int(rng, 1, 16), _log_int(rng, 1, 4096)
        if experts * hidden * inter > _MOST_WEIGHTS or tokens * top_k * hidden * inter > _MOST_ROUTED:
            continue
        return _moe(None, kind, tokens, hidden, inter, experts, top_k,
                    act=rng.choice(["swiglu", "swiglu", "situglu", "clamp_swiglu"]), drop=rng.choice([0.0, 0.0, 0.1]))


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _ceil(n, d):
    return -(-n // d)


def _stream(gen, rows, hidden, dtype):
    """Rows of a residual stream: normal, with a few channels much larger than the others."""
    loud = 1.0 + 15.0 * (torch.rand(hidden, generator=gen, device="cuda") < 0.01).float()
    return (_randn(gen, rows, hidden) * loud).to(dtype)


def _e4m3(gen, *shape):
    """Normal values as the quantiser leaves them: a block's largest between 224 and 448."""
    out = torch.empty(*shape, dtype=_F8, device="cuda")
    flat = out.view(-1)
    step = 1 << 28
    for i in range(0, flat.numel(), step):
        part = flat[i:i + step]
        part.copy_(_randn(gen, part.numel()).mul_(90.0).clamp_(-448.0, 448.0))
    return out


def _e8m0(gen, low, *shape):
    """Powers of two from 2^low to 2^(low + 2)."""
    return (torch.randint(0, 3, shape, generator=gen, device="cuda") + (127 + low)).to(torch.uint8).view(_E8)


def prepare(case, seed):
    c, gen = case, _gen(seed)
    kind = c["kind"]
    s = dict(case=case)
    if kind == "quant":
        s["x"] = _stream(gen, c["rows"], c["cols"], _DT[c["dtype"]])
    elif kind == "matmul":
        kb = _ceil(c["k"], _B)
        s.update(a=_e4m3(gen, c["rows"], c["k"]), sa=_e8m0(gen, -8, c["rows"], kb),
                 b=_e4m3(gen, c["n"], c["k"]), sb=_e8m0(gen, -13, _ceil(c["n"], _B), kb), dtype=_DT[c["dtype"]],
                 bias=_randn(gen, c["n"]).to(_DT[c["dtype"]]) if c["bias"] else None)
    elif kind == "linear":
        dtype = _DT[c["dtype"]]
        s["x"] = _stream(gen, c["rows"], c["k"], dtype).requires_grad_()
        s["weight"] = (_randn(gen, c["n"], c["k"]) * 0.02).to(torch.float32 if c["weight"] == "fp32" else dtype)
        s["weight"].requires_grad_()
        # gradients differ in size from token to token, and padding has none
        size = torch.exp(_randn(gen, c["rows"], 1)) * (torch.rand(c["rows"], 1, generator=gen, device="cuda") > 0.05)
        s["dy"] = (_randn(gen, c["rows"], c["n"]) * size * 1e-2).to(dtype)
    else:
        s.update(_experts_state(c, gen))
    return s


def _experts_state(c, gen):
    T, H, F, E, k = c["tokens"], c["hidden"], c["inter"], c["experts"], c["top_k"]
    w, idx = torch.topk(torch.softmax(_randn(gen, T, E), dim=-1), k, dim=-1)
    w = (w / w.sum(dim=-1, keepdim=True)).contiguous()
    sel = idx.to(torch.int32)
    sel[torch.rand(T, k, generator=gen, device="cuda") < c["drop"]] = -1
    s = dict(sel=sel.contiguous(), w=w, gate_up=_e4m3(gen, E, 2 * F, H),
             gate_up_scale=_e8m0(gen, -13, E, 2 * F // _B, H // _B), down=_e4m3(gen, E, H, F),
             down_scale=_e8m0(gen, -13, E, H // _B, F // _B))
    # rows that the fullest expert gets, for the size of the plain form's batches
    s["most"] = max(1, int(torch.bincount(sel[sel >= 0].long(), minlength=E).max()))
    if c["kind"] == "block":
        s.update(x=_randn(gen, T, H).to(torch.bfloat16), residual=_stream(gen, T, H, torch.bfloat16),
                 weight=(1.0 + 0.2 * _randn(gen, H)).to(torch.bfloat16))
    else:
        s.update(x=_e4m3(gen, T, H), sx=_e8m0(gen, -8, T, H // _B))
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import mega_moe

    c, kind = s["case"], s["case"]["kind"]
    if kind == "quant":
        return mega_moe.quantize_blocks(s["x"], rows=c["block_rows"])
    if kind == "matmul":
        return mega_moe.fp8_matmul(s["a"], s["b"], s["sa"], s["sb"], bias=s["bias"], out_dtype=s["dtype"])
    if kind == "linear":
        y = mega_moe.fp8_linear(s["x"], s["weight"])
        return (y, *torch.autograd.grad(y, (s["x"], s["weight"]), s["dy"]))
    if "op" not in s:
        # what a program builds once and keeps: the operator, and its experts in 8 bits
        extra = dict(situ_beta=2.0, situ_linear_beta=3.0) if c["act"] == "situglu" else {}
        s["op"] = mega_moe.FusedMoEForward(
            None, max_tokens_per_rank=4096, hidden_size=c["hidden"], top_k=c["top_k"], num_experts=c["experts"],
            config=mega_moe.MoEForwardConfig(activation=c["act"], **extra))
        s["experts"] = mega_moe.Fp8Experts(s["gate_up"], s["gate_up_scale"], s["down"], s["down_scale"])
    if kind == "moe":
        return s["op"].forward_fp8(s["x"], s["sx"], s["sel"], s["experts"], s["w"])
    q, sq, h = mega_moe.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=_EPS, out_dtype=_F8,
                                 scale_columns=_B)
    return s["op"].forward_fp8(q, sq, s["sel"], s["experts"], s["w"]), h


def _power(k):
    """2^k in 32 bits, from its bits."""
    return (k + 127).to(torch.int32).bitwise_left_shift(23).view(torch.float32)


def _plain_quant(x, block_rows):
    """(E4M3 values in 32 bits, scales in 32 bits) of x [..., rows, columns] in blocks."""
    rows, cols = x.shape[-2:]
    br = block_rows
    x = torch.nn.functional.pad(x, (0, -cols % _B, 0, -rows % br))
    g = x.reshape(*x.shape[:-2], x.shape[-2] // br, br, x.shape[-1] // _B, _B)
    top = g.abs().amax(dim=(-3, -1), keepdim=True)
    m, e = torch.frexp(top)
    k = torch.where(m <= 0.875, e - 9, e - 8).clamp_min(-126)
    k = torch.where(top == 0, torch.zeros_like(k), k)
    q = (g * _power(-k)).to(_F8).float().reshape(x.shape)[..., :rows, :cols]
    return q, _power(k)[..., 0, :, 0]


def _plain_values(q, scale, block_rows):
    """Values in 32 bits of E4M3 values in blocks."""
    rows, cols = q.shape[-2:]
    if rows % block_rows == 0 and cols % _B == 0:
        g = q.float().view(*q.shape[:-2], rows // block_rows, block_rows, cols // _B, _B)
        return g.mul_(scale.float()[..., :, None, :, None]).view(q.shape)
    s = scale.float().repeat_interleave(block_rows, dim=-2)[..., :rows, :].repeat_interleave(_B, dim=-1)[..., :cols]
    return q.float() * s


@torch.no_grad()
def _run_plain(s):
    c, kind = s["case"], s["case"]["kind"]
    if kind == "quant":
        q, scale = _plain_quant(s["x"].float(), c["block_rows"])
        return q.to(_F8), scale.to(_E8)
    if kind == "matmul":
        out = _plain_values(s["a"], s["sa"], 1) @ _plain_values(s["b"], s["sb"], _B).t()
        if s["bias"] is not None:
            out = out + s["bias"].float()
        return out.to(s["dtype"])
    if kind == "linear":
        x, w, dy = s["x"].float(), s["weight"].float(), s["dy"].float()
        xv = _plain_values(*_plain_quant(x, 1), 1)
        wv = _plain_values(*_plain_quant(w, _B), _B)
        y = xv @ wv.t()
        dx = _plain_values(*_plain_quant(dy, 1), 1) @ wv
        dw = _plain_values(*_plain_quant(dy.t().contiguous(), 1), 1) @ _plain_values(*_plain_quant(xv, _B), _B)
        return y.to(s["x"].dtype), dx.to(s["x"].dtype), dw.to(s["weight"].dtype)
    h = None
    if kind == "moe":
        x = _plain_values(s["x"], s["sx"], 1)
    else:
        h = (s["x"].float() + s["residual"].float()).to(s["residual"].dtype)
        h32 = h.float()
        y = h32 * torch.rsqrt(h32.square().mean(dim=-1, keepdim=True) + _EPS) * s["weight"].float()
        x = _plain_values(*_plain_quant(y, 1), 1)
    out = _plain_layer(s, c, x)
    return out if h is None else (out, h)


def _plain_layer(s, c, x):
    T, k = s["sel"].shape
    H, F, E = c["hidden"], c["inter"], c["experts"]
    flat = s["sel"].reshape(-1).long()
    live = (flat >= 0) & (flat < E)
    at = torch.where(live, flat, torch.zeros_like(flat))
    weight = s["w"].reshape(-1, 1)
    if T * k <= E:  # few routes: each with its own expert's weights
        xr = x.repeat_interleave(k, dim=0)
        gu = torch.bmm(_plain_values(s["gate_up"].view(torch.uint8)[at].view(_F8), s["gate_up_scale"].view(torch.uint8)[at].view(_E8), _B),
                       xr[:, :, None])[:, :, 0]
        act = _activation(c["act"], *gu.chunk(2, dim=-1)) * weight
        act = _plain_values(*_plain_quant(act, 1), 1)
        y = torch.bmm(_plain_values(s["down"].view(torch.uint8)[at].view(_F8), s["down_scale"].view(torch.uint8)[at].view(_E8), _B),
                      act[:, :, None])[:, :, 0]
    else:  # every expert with its routes, filled up to those of the fullest
        cap = s["most"]
        key = torch.where(live, flat, torch.full_like(flat, E))
        order = torch.argsort(key, stable=True)
        first = torch.searchsorted(key[order].contiguous(), torch.arange(E + 1, device=key.device))
        place = torch.empty_like(key)
        place[order] = torch.arange(T * k, device=key.device) - first[key[order]]
        slot = torch.where(live, key * cap + place, torch.full_like(key, E * cap))
        xp = torch.zeros(E * cap + 1, H, device=x.device)
        xp[slot] = x.repeat_interleave(k, dim=0)
        wp = torch.zeros(E * cap + 1, 1, device=x.device)
        wp[slot] = weight
        xt = xp[:-1].view(E, cap, H).transpose(1, 2).contiguous()
        gu = torch.bmm(_plain_values(s["gate_up"], s["gate_up_scale"], _B), xt).transpose(1, 2)
        act = _activation(c["act"], *gu.chunk(2, dim=-1)) * wp[:-1].view(E, cap, 1)
        act = _plain_values(*_plain_quant(act.reshape(E * cap, F), 1), 1).view(E, cap, F)
        y = torch.bmm(_plain_values(s["down"], s["down_scale"], _B), act.transpose(1, 2).contiguous())
        y = torch.cat([y.transpose(1, 2).reshape(E * cap, H), torch.zeros(1, H, device=x.device)])[slot]
    y = torch.where(live[:, None], y, torch.zeros_like(y))
    return y.reshape(T, k, -1).sum(dim=1).to(torch.bfloat16)


def _activation(kind, g, u):
    if kind == "swiglu":
        return g * torch.sigmoid(g) * u
    if kind == "clamp_swiglu":
        g, u = g.clamp(max=7.0), u.clamp(-7.0, 7.0)
        return g * torch.sigmoid(g) * u
    return 2.0 * torch.tanh(g / 2.0) * torch.sigmoid(g) * (3.0 * torch.tanh(u / 3.0))


# ------------------------------------------------------------------ bytes and flops
def work(case):
    c, kind = case, case["kind"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if kind == "quant":
        n = c["rows"] * c["cols"]
        scales = _ceil(c["rows"], c["block_rows"]) * _ceil(c["cols"], _B)
        return {"bytes": n * (size[c["dtype"]] + 1) + scales, "flops": 3 * n}
    if kind == "matmul":
        m, k, n = c["rows"], c["k"], c["n"]
        kb = _ceil(k, _B)
        total = (m + n) * k + (m + _ceil(n, _B)) * kb + m * n * size[c["dtype"]]
        return {"bytes": total + (n * size[c["dtype"]] if c["bias"] else 0), "flops": 2 * m * n * k}
    if kind == "linear":
        m, k, n, x = c["rows"], c["k"], c["n"], size[c["dtype"]]
        w = 4 if c["weight"] == "fp32" else x
        return {"bytes": 2 * x * m * (k + n) + 2 * w * n * k, "flops": 6 * m * n * k}
    T, H, F, E, k = c["tokens"], c["hidden"], c["inter"], c["experts"], c["top_k"]
    routes = T * k * (1.0 - c["drop"])
    distinct = E * (1.0 - (1.0 - k * (1.0 - c["drop"]) / E) ** T)  # experts that an even draw of T tokens reaches
    weights = 3 * H * F * (1.0 + 1.0 / (_B * _B))
    return {"bytes": distinct * weights + T * H * ((6 if kind == "block" else 1) + 2) + 8 * T * k,
            "flops": 6 * routes * H * F}


# ------------------------------------------------------------------ 64 bits
def _exact_quant(x, block_rows):
    """(values before and after rounding to E4M3, exponents of the scales), block by block of rows."""
    rows, cols = x.shape
    nr, nc = _ceil(rows, block_rows), _ceil(cols, _B)
    full = torch.zeros(nr * block_rows, nc * _B, dtype=torch.float64, device=x.device)
    full[:rows, :cols] = x
    blocks = full.view(nr, block_rows, nc, _B).permute(0, 2, 1, 3)
    top = blocks.abs().flatten(2).max(dim=2).values
    k = torch.ceil(torch.log2(torch.clamp(top, min=1e-300) / 448.0))
    k = torch.where(top > 448.0 * torch.exp2(k), k + 1, k)  # log2's own rounding
    k = torch.where(top <= 448.0 * torch.exp2(k - 1), k - 1, k)
    k = torch.clamp(k, min=-126.0)
    k[top == 0] = 0.0
    scale = torch.exp2(k)
    v = blocks / scale[:, :, None, None]
    # a normal value has 3 bits behind its first, one below 2^-6 steps of 2^-9
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(v.abs(), min=2.0 ** -30))), min=-6.0) - 3.0)
    q = torch.round(v / step) * step
    back = q.permute(0, 2, 1, 3).reshape(full.shape)[:rows, :cols]
    return back, scale


def _exact_values(q, scale, block_rows):
    rows, cols = q.shape
    r = torch.arange(rows, device=q.device) // block_rows
    k = torch.arange(cols, device=q.device) // _B
    return q.double() * scale.double()[r][:, k]


@torch.no_grad()
def exact(case, seed):
    s, c, kind = prepare(case, seed), case, case["kind"]
    if kind == "quant":
        return list(_exact_quant(s["x"].double(), c["block_rows"]))
    if kind == "matmul":
        out = _exact_values(s["a"], s["sa"], 1) @ _exact_values(s["b"], s["sb"], _B).t()
        return out if s["bias"] is None else out + s["bias"].double()
    if kind == "linear":
        x, w, dy = s["x"].detach().double(), s["weight"].detach().double(), s["dy"].double()
        xv = _exact_values(*_exact_quant(x, 1), 1)
        wv = _exact_values(*_exact_quant(w, _B), _B)
        dyr = _exact_values(*_exact_quant(dy, 1), 1)
        dyc = _exact_values(*_exact_quant(dy.t(), 1), 1)
        xc = _exact_values(*_exact_quant(xv, _B), _B)
        return [xv @ wv.t(), dyr @ wv, dyc @ xc]
    h = None
    if kind == "moe":
        x = _exact_values(s["x"], s["sx"], 1)
    else:
        h = (s["x"].double() + s["residual"].double()).to(torch.bfloat16).double()
        y = h / torch.sqrt((h * h).sum(dim=1, keepdim=True) / h.shape[1] + _EPS) * s["weight"].double()
        x = _exact_values(*_exact_quant(y, 1), 1)
    F = c["inter"]
    out = torch.zeros(c["tokens"], c["hidden"], dtype=torch.float64, device=x.device)
    for e in range(c["experts"]):
        token, place = torch.nonzero(s["sel"] == e, as_tuple=True)
        if not token.numel():
            continue
        gu = x[token] @ _exact_values(s["gate_up"][e], s["gate_up_scale"][e], _B).t()
        g, u = gu[:, :F], gu[:, F:]
        if c["act"] == "clamp_swiglu":
            g, u = torch.minimum(g, torch.full_like(g, 7.0)), u.clamp(-7.0, 7.0)
        sig = 1.0 / (1.0 + torch.exp(-g))
        if c["act"] == "situglu":
            act = 2.0 * torch.tanh(0.5 * g) * sig * 3.0 * torch.tanh(u / 3.0)
        else:
            act = g * sig * u
        act = act * s["w"][token, place].double()[:, None]
        act = _exact_values(*_exact_quant(act, 1), 1)
        out.index_add_(0, token, act @ _exact_values(s["down"][e], s["down_scale"][e], _B).t())
    return out if h is None else [out, h]
