"""The operators around the layer whose time is measured: norm, 8-bit product, and the layer for a few tokens.

Every case is one pass through an operator's public entry point (``own``) or
the same mathematics in elementary torch operations in 32 bits. Sizes are those
of the layer configurations in ``mega_moe/bench_configs.py`` and of the tests,
or generic ones between them.

Kinds of case:
  norm         rms_norm, with or without a residual; output as the input's
               type, or e4m3 with one scale a row
  norm_train   rms_norm forward and backward
  product      int8_matmul: int8 rows with scales, int8 weights with scales
  project      rms_norm with a residual to int8 rows, then int8_matmul on them
  few          the expert layer for a few tokens, bf16 weights
  few_int8     the same on int8 rows and int8 experts
  block_int8   rms_norm with a residual to int8 rows, then few_int8 on them
"""

import math
import os
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mega-moe-td_amd")
_EPS = 1e-6
_GROUP = 32  # columns of the activation that share a scale in the int8 layer
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _norm(name, rows, hidden, dtype="bf16", residual="same", weight="same", out="same", train=False):
    c = dict(kind="norm_train" if train else "norm", rows=rows, hidden=hidden, dtype=dtype, residual=residual,
             weight=weight, out=out)
    return dict(c, name=name) if name else c


def _product(name, rows, k, n, dtype="bf16", bias=False, norm=False):
    c = dict(kind="project" if norm else "product", rows=rows, k=k, n=n, dtype=dtype, bias=bias)
    return dict(c, name=name) if name else c


def _few(name, kind, tokens, hidden, inter, experts, top_k, act="swiglu", down="natural", drop=0.0):
    c = dict(kind=kind, tokens=tokens, hidden=hidden, inter=inter, experts=experts, top_k=top_k, act=act, down=down,
             drop=drop)
    return dict(c, name=name) if name else c


def listed():
    return [
        # generation for one user: the norm in front of the layer
        _norm("norm_token", 1, 2048),
        # a prompt chunk on a wide layer, normed into 8 bits
        _norm("norm_prompt_e4m3", 8192, 7168, out="e4m3"),
        # training: a full micro-batch
        _norm("norm_train", 8192, 2048, train=True),
        # training on an odd number of odd rows, the residual stream and the weight in 32 bits
        _norm("norm_train_ragged", 1021, 2305, residual="fp32", weight="fp32", train=True),
        # generation for one user: a shared expert's first product
        _product("product_token", 1, 2048, 1536),
        # generation for a batch of users on a wide layer
        _product("product_batch", 32, 7168, 4096),
        # a short prompt, sizes that no tile divides
        _product("product_ragged", 1021, 2309, 1793, dtype="fp16", bias=True),
        # a prompt chunk on a wide layer
        _product("product_prompt", 8192, 7168, 4096),
        # generation for a batch: the norm and the projection behind it
        _product("project_batch", 64, 4096, 2048, norm=True),
        # generation for one user: the whole expert layer
        _few("few_one", "few", 1, 2048, 768, 128, 8),
        # generation for a few users on a wide layer: nearly every route has an expert of its own
        _few("few_wide", "few", 8, 7168, 2048, 64, 8, down="contiguous"),
        # generation for a batch in 8 bits: the norm and the expert layer behind it
        _few("block_int8", "block_int8", 32, 2048, 768, 128, 8, down="contiguous"),
    ]


_MOST_NORM = 8192 * 7168
_MOST_TRAIN = 8192 * 2048
_MOST_PRODUCT = 8192 * 7168 * 4096
_MOST_WEIGHTS = 64 * 7168 * 2048
_MOST_ROUTED = 64 * 7168 * 2048


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["norm", "norm_train", "product", "product", "project", "few", "few", "few_int8",
                           "block_int8"])
        if kind in ("norm", "norm_train"):
            train = kind == "norm_train"
            rows, hidden = _log_int(rng, 1, 16384), _log_int(rng, 64, 8192)
            if rows * hidden > (_MOST_TRAIN if train else _MOST_NORM):
                continue
            return _norm(None, rows, hidden, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                         residual=rng.choice(["same", "none", "fp32"]), weight=rng.choice(["same", "fp32"]),
                         out="same" if train else rng.choice(["same", "e4m3"]), train=train)
        if kind in ("product", "project"):
            norm = kind == "project"
            rows, k, n = _log_int(rng, 1, 8192), _log_int(rng, 256, 8192), _log_int(rng, 256, 8192)
            if rng.random() < 0.5:
                k, n = 128 * -(-k // 128), 128 * -(-n // 128)
            if rows * k * n > _MOST_PRODUCT:
                continue
            return _product(None, rows, k, n, dtype=rng.choice(["bf16", "bf16", "fp16"] if norm else ["bf16", "bf16", "fp16", "fp32"]),
                            bias=rng.random() < 0.3, norm=norm)
        experts = _log_int(rng, 8, 256)
        top_k = rng.choice([v for v in (1, 2, 4, 6, 8, 16) if v <= experts])
        hidden, inter, tokens = 256 * _log_int(rng, 1, 28), 128 * _log_int(rng, 1, 16), _log_int(rng, 1, 64)
        weights = experts * hidden * inter
        if weights > _MOST_WEIGHTS or tokens * top_k * hidden * inter > _MOST_ROUTED:
            continue
        return _few(None, kind, tokens, hidden, inter, experts, top_k,
                    act=rng.choice(["swiglu", "swiglu", "situglu", "clamp_swiglu"]),
                    down=rng.choice(["natural", "contiguous"]) if kind == "few" else "contiguous",
                    drop=rng.choice([0.0, 0.0, 0.1]))


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _int8(gen, *shape):
    """Normal values as a quantiser leaves them: the largest of a row near 127."""
    out = torch.empty(*shape, dtype=torch.int8, device="cuda")
    flat = out.view(-1)
    step = 1 << 28
    for i in range(0, flat.numel(), step):
        part = flat[i:i + step]
        part.copy_(_randn(gen, part.numel()).mul_(36.0).round_().clamp_(-127, 127))
    return out


def _scales(gen, *shape):
    return torch.rand(*shape, generator=gen, device="cuda").mul_(0.01).add_(0.005)


def _stream(gen, rows, hidden, dtype):
    """Rows of a residual stream: normal, with a few channels much larger than the others."""
    loud = 1.0 + 15.0 * (torch.rand(hidden, generator=gen, device="cuda") < 0.01).float()
    return (_randn(gen, rows, hidden) * loud).to(dtype)


def _norm_state(c, gen, rows, hidden, dtype):
    res = c.get("residual", "same")
    wdt = torch.float32 if c.get("weight") == "fp32" else dtype
    s = dict(x=_randn(gen, rows, hidden).to(dtype), weight=(1.0 + 0.2 * _randn(gen, hidden)).to(wdt), residual=None)
    if res != "none":
        s["residual"] = _stream(gen, rows, hidden, torch.float32 if res == "fp32" else dtype)
    return s


def prepare(case, seed):
    c, gen = case, _gen(seed)
    kind = c["kind"]
    s = dict(case=case)
    if kind in ("norm", "norm_train"):
        dtype = _DT[c["dtype"]]
        s.update(_norm_state(c, gen, c["rows"], c["hidden"], dtype))
        if kind == "norm_train":
            s["dy"] = _randn(gen, c["rows"], c["hidden"]).to(dtype)
            s["leaves"] = [s["x"].requires_grad_(), s["weight"].requires_grad_()]
            if s["residual"] is not None:
                s["dh"] = _randn(gen, c["rows"], c["hidden"]).to(s["residual"].dtype)
                s["leaves"].append(s["residual"].requires_grad_())
    elif kind in ("product", "project"):
        if kind == "project":
            s.update(_norm_state(c, gen, c["rows"], c["k"], torch.bfloat16))
        else:
            s.update(a=_int8(gen, c["rows"], c["k"]), sa=_scales(gen, c["rows"]))
        s.update(b=_int8(gen, c["n"], c["k"]), sb=_scales(gen, c["n"]), dtype=_DT[c["dtype"]],
                 bias=_randn(gen, c["n"]).to(_DT[c["dtype"]]) if c["bias"] else None)
    else:
        s.update(_experts_state(c, gen))
    return s


def _experts_state(c, gen):
    T, H, F, E, k = c["tokens"], c["hidden"], c["inter"], c["experts"], c["top_k"]
    w, idx = torch.topk(torch.softmax(_randn(gen, T, E), dim=-1), k, dim=-1)
    w = (w / w.sum(dim=-1, keepdim=True)).contiguous()
    sel = idx.to(torch.int32)
    sel[torch.rand(T, k, generator=gen, device="cuda") < c["drop"]] = -1
    s = dict(sel=sel.contiguous(), w=w)
    if c["kind"] == "few":
        s["x"] = _randn(gen, T, H).to(torch.bfloat16)
        tables = []
        for shape in ((E, H, 2 * F), (E, F, H) if c["down"] == "natural" else (E, H, F)):
            table = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
            for e in range(E):
                table[e].copy_(_randn(gen, *shape[1:]).mul_(0.02))
            tables.append(table)
        s.update(gate_up=tables[0], down=tables[1].transpose(1, 2) if c["down"] == "natural" else tables[1])
        return s
    s.update(gate_up=_int8(gen, E, 2 * F, H), gate_up_scale=_scales(gen, E, 2 * F).mul_(0.06),
             down=_int8(gen, E, H, F), down_scale=_scales(gen, E, H).mul_(0.06))
    if c["kind"] == "block_int8":
        s.update(_norm_state({}, gen, T, H, torch.bfloat16))
    else:
        s.update(x=_int8(gen, T, H), sx=_scales(gen, T))
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import mega_moe

    c, kind = s["case"], s["case"]["kind"]
    if kind == "norm":
        out = torch.float8_e4m3fn if c["out"] == "e4m3" else None
        return mega_moe.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=_EPS, out_dtype=out)
    if kind == "norm_train":
        if s["residual"] is None:
            y = mega_moe.rms_norm(s["x"], s["weight"], eps=_EPS)
            return (y, *torch.autograd.grad(y, s["leaves"], s["dy"]))
        y, h = mega_moe.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=_EPS)
        return (y, h, *torch.autograd.grad((y, h), s["leaves"], (s["dy"], s["dh"])))
    if kind == "product":
        return mega_moe.int8_matmul(s["a"], s["b"], s["sa"], s["sb"], bias=s["bias"], out_dtype=s["dtype"])
    if kind == "project":
        q, sq, h = mega_moe.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=_EPS, out_dtype=torch.int8)
        return mega_moe.int8_matmul(q, s["b"], sq, s["sb"], bias=s["bias"], out_dtype=s["dtype"]), h
    if "op" not in s:
        # what a program builds once and keeps: the operator, and its experts in 8 bits
        extra = dict(situ_beta=2.0, situ_linear_beta=3.0) if c["act"] == "situglu" else {}
        s["op"] = mega_moe.FusedMoEForward(
            None, max_tokens_per_rank=64, hidden_size=c["hidden"], top_k=c["top_k"], num_experts=c["experts"],
            config=mega_moe.MoEForwardConfig(activation=c["act"], **extra))
        if kind != "few":
            s["experts"] = mega_moe.Int8Experts(s["gate_up"], s["gate_up_scale"], s["down"], s["down_scale"])
    if kind == "few":
        return s["op"].forward_few(s["x"], s["sel"], s["gate_up"], s["down"], s["w"])
    if kind == "few_int8":
        return s["op"].forward_few_int8(s["x"], s["sx"], s["sel"], s["experts"], s["w"])
    q, sq, h = mega_moe.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=_EPS, out_dtype=torch.int8)
    return s["op"].forward_few_int8(q, sq, s["sel"], s["experts"], s["w"]), h


def _plain_norm(s):
    """(y in 32 bits, the sum as it is stored, the sum in 32 bits, 1 / rms)"""
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["residual"].dtype)
    h32 = h.float()
    r = torch.rsqrt(h32.square().mean(dim=-1, keepdim=True) + _EPS)
    return h32 * r * s["weight"].float(), h, h32, r


def _plain_rows8(y, most):
    """(values / scale, scale) of rows in 8 bits whose largest value is `most`."""
    top = y.abs().amax(dim=-1, keepdim=True)
    scale = torch.where(top > 0, top.clamp_min(1e-30) / most, torch.ones_like(top))
    return y / scale, scale


@torch.no_grad()
def _run_plain(s):
    c, kind = s["case"], s["case"]["kind"]
    if kind == "norm":
        y, h, _, _ = _plain_norm(s)
        if c["out"] == "e4m3":
            v, scale = _plain_rows8(y, 448.0)
            out = (v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn), scale[:, 0])
        else:
            out = (y.to(s["x"].dtype),)
        if s["residual"] is not None:
            out += (h,)
        return out if len(out) > 1 else out[0]
    if kind == "norm_train":
        y, h, h32, r = _plain_norm(s)
        wdy = s["dy"].float() * s["weight"].float()
        dx = r * wdy - h32 * (r.pow(3) * (wdy * h32).mean(dim=-1, keepdim=True))
        dw = (s["dy"].float() * h32 * r).sum(dim=0).to(s["weight"].dtype)
        if s["residual"] is None:
            return y.to(s["x"].dtype), dx.to(s["x"].dtype), dw
        dx = dx + s["dh"].float()
        return y.to(s["x"].dtype), h, dx.to(s["x"].dtype), dw, dx.to(s["residual"].dtype)
    if kind in ("product", "project"):
        if kind == "project":
            y, h, _, _ = _plain_norm(s)
            v, scale = _plain_rows8(y, 127.0)
            v = v.round()
        else:
            v, scale = s["a"].float(), s["sa"][:, None]
        out = (v @ s["b"].float().t()) * scale * s["sb"]
        if s["bias"] is not None:
            out = out + s["bias"].float()
        out = out.to(s["dtype"])
        return (out, h) if kind == "project" else out
    h = None
    if kind == "few":
        x = s["x"].float()
    elif kind == "few_int8":
        x = s["x"].float() * s["sx"][:, None]
    else:
        y, h, _, _ = _plain_norm(s)
        v, scale = _plain_rows8(y, 127.0)
        x = v.round() * scale
    T, k = s["sel"].shape
    flat = s["sel"].reshape(-1).long()
    live = (flat >= 0) & (flat < c["experts"])
    at = torch.where(live, flat, torch.zeros_like(flat))
    xr = x.repeat_interleave(k, dim=0)
    if kind == "few":
        gu = torch.bmm(xr[:, None, :], s["gate_up"][at].float())[:, 0]
    else:
        gu = torch.bmm(s["gate_up"][at].float(), xr[:, :, None])[:, :, 0] * s["gate_up_scale"][at]
    act = _activation(c["act"], *gu.chunk(2, dim=-1)) * s["w"].reshape(-1, 1)
    if kind != "few":
        v, scale = _plain_rows8(act.reshape(act.shape[0], -1, _GROUP), 127.0)
        act = (v.round() * scale).reshape(act.shape)
    y = torch.bmm(s["down"][at].float(), act[:, :, None])[:, :, 0]
    if kind != "few":
        y = y * s["down_scale"][at]
    y = torch.where(live[:, None], y, torch.zeros_like(y))
    out = y.reshape(T, k, -1).sum(dim=1).to(torch.bfloat16)
    return out if h is None else (out, h)


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
    if kind in ("norm", "norm_train"):
        n, x = c["rows"] * c["hidden"], size[c["dtype"]]
        r = {"same": x, "none": 0, "fp32": 4}[c["residual"]]
        w = 4 if c["weight"] == "fp32" else x
        total = n * (x + 2 * r + (1 if c["out"] == "e4m3" else x)) + c["hidden"] * w
        if kind == "norm_train":  # dy, dh and h in (h is an output of the forward), dx and dresidual out
            total += n * (2 * x + (2 * r if r else x)) + 2 * c["hidden"] * w
            return {"bytes": total + (n * r if r else 0), "flops": 16 * n}
        return {"bytes": total, "flops": 6 * n}
    if kind in ("product", "project"):
        m, k, n = c["rows"], c["k"], c["n"]
        total = n * k + m * n * size[c["dtype"]] + 4 * n
        total += (6 * m * k + 2 * k) if kind == "project" else (m * k + 4 * m)
        return {"bytes": total, "flops": 2 * m * n * k}
    T, H, F, E, k = c["tokens"], c["hidden"], c["inter"], c["experts"], c["top_k"]
    routes = T * k * (1.0 - c["drop"])
    distinct = E * (1.0 - (1.0 - k * (1.0 - c["drop"]) / E) ** T)  # experts that an even draw of T tokens reaches
    weights = 3 * H * F * (2 if kind == "few" else 1) + (0 if kind == "few" else 4 * (2 * F + H))
    rows = {"few": 2, "few_int8": 1, "block_int8": 6}[kind]
    return {"bytes": distinct * weights + T * H * (rows + 2) + 8 * T * k, "flops": 6 * routes * H * F}


# ------------------------------------------------------------------ 64 bits
def _exact_norm(s):
    h = s["x"]
    if s["residual"] is not None:
        h = (s["x"].double() + s["residual"].double()).to(s["residual"].dtype)
    hd = h.detach().double()
    ms = (hd * hd).sum(dim=1, keepdim=True) / hd.shape[1]
    return hd, (ms + _EPS) ** -0.5


def _exact_rows8(y, most):
    top = y.abs().max(dim=-1, keepdim=True).values
    scale = torch.where(top == 0, torch.ones_like(top), torch.clamp(top, min=1e-30) / most)
    return y / scale, scale


@torch.no_grad()
def exact(case, seed):
    s, c, kind = prepare(case, seed), case, case["kind"]
    if kind == "norm":
        hd, r = _exact_norm(s)
        y = hd * r * s["weight"].double()
        if c["out"] == "e4m3":
            v, scale = _exact_rows8(y, 448.0)
            out = [v.clamp(-448, 448).to(torch.float8_e4m3fn).double(), scale.flatten()]
        else:
            out = [y]
        if s["residual"] is not None:
            out.append(hd)
        return out if len(out) > 1 else out[0]
    if kind == "norm_train":
        hd, r = _exact_norm(s)
        w, dy = s["weight"].double(), s["dy"].double()
        unit = hd * r
        t = dy * w
        dx = r * (t - unit * (t * unit).sum(dim=1, keepdim=True) / hd.shape[1])
        dw = (dy * unit).sum(dim=0)
        if s["residual"] is None:
            return [unit * w, dx, dw]
        dx = dx + s["dh"].double()
        return [unit * w, hd, dx, dw, dx]
    if kind in ("product", "project"):
        if kind == "project":
            hd, r = _exact_norm(s)
            v, scale = _exact_rows8(hd * r * s["weight"].double(), 127.0)
            rows = torch.round(v) * scale
        else:
            rows = s["a"].double() * s["sa"].double()[:, None]
        out = rows @ (s["b"].double() * s["sb"].double()[:, None]).t()
        if s["bias"] is not None:
            out += s["bias"].double()
        return [out, hd] if kind == "project" else out
    return _exact_layer(s, c, kind)


def _exact_layer(s, c, kind):
    """The layer expert by expert: each one's routes through its two products."""
    hd = None
    if kind == "few":
        x = s["x"].double()
    elif kind == "few_int8":
        x = s["x"].double() * s["sx"].double()[:, None]
    else:
        hd, r = _exact_norm(s)
        v, scale = _exact_rows8(hd * r * s["weight"].double(), 127.0)
        x = torch.round(v) * scale
    F = c["inter"]
    out = torch.zeros(c["tokens"], c["hidden"], dtype=torch.float64, device=x.device)
    for e in range(c["experts"]):
        token, slot = torch.nonzero(s["sel"] == e, as_tuple=True)
        if not token.numel():
            continue
        if kind == "few":
            w1, w2 = s["gate_up"][e].double(), s["down"][e].double().t()
        else:
            w1 = (s["gate_up"][e].double() * s["gate_up_scale"][e].double()[:, None]).t()
            w2 = (s["down"][e].double() * s["down_scale"][e].double()[:, None]).t()
        gu = x[token] @ w1
        g, u = gu[:, :F], gu[:, F:]
        if c["act"] == "clamp_swiglu":
            g, u = torch.minimum(g, torch.full_like(g, 7.0)), u.clamp(-7.0, 7.0)
        sig = 1.0 / (1.0 + torch.exp(-g))
        if c["act"] == "situglu":
            act = 2.0 * torch.tanh(0.5 * g) * sig * 3.0 * torch.tanh(u / 3.0)
        else:
            act = g * sig * u
        act = act * s["w"][token, slot].double()[:, None]
        if kind != "few":
            v, scale = _exact_rows8(act.view(act.shape[0], F // _GROUP, _GROUP), 127.0)
            act = (torch.round(v) * scale).view(act.shape[0], F)
        out.index_add_(0, token, act @ w2)
    return out if hd is None else [out, hd]
