"""E4M3 blocks and their products in 64 bits, from the definitions."""

import torch

F8, E8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
BLOCK = 128


def ceil(n, d):
    return -(-n // d)


def round_e4m3(v):
    """The nearest E4M3 value of |v| <= 448, ties to even, in 64 bits."""
    _, e = torch.frexp(v)  # v = m 2^e, 0.5 <= m < 1: 4 significant bits, or steps of 2^-9
    step = torch.exp2((e - 4).clamp_min(-9).double())
    return torch.round(v / step) * step


def quant(x, block_rows):
    """(values of q, scales) in 64 bits of a matrix in 64 bits; NaN scales and zero bytes for blocks that are not finite."""
    rows, cols = x.shape
    full = torch.zeros(ceil(rows, block_rows) * block_rows, ceil(cols, BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    full[:rows, :cols] = x
    g = full.view(full.shape[0] // block_rows, block_rows, full.shape[1] // BLOCK, BLOCK)
    top = g.abs().amax(dim=(1, 3))
    good = torch.isfinite(top)
    m, e = torch.frexp(torch.where(good, top, torch.ones_like(top)))
    k = torch.where(m <= 0.875, e - 9, e - 8).clamp_min(-126)  # 448 = 0.875 * 2^9
    scale = torch.where(top == 0, torch.ones_like(top), torch.exp2(k.double()))
    q = round_e4m3(torch.where(good[:, None, :, None], g / scale[:, None, :, None], torch.zeros_like(g)))
    return q.reshape(full.shape)[:rows, :cols], torch.where(good, scale, torch.full_like(scale, float("nan")))


def values(q, scale, block_rows):
    """q * scale in 64 bits."""
    rows, cols = q.shape
    s = scale.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    return q.double() * s


def quantized(x, block_rows):
    return values(*quant(x, block_rows), block_rows)


def sum_error(a, b, wide=False):
    """Bound of a product's error before it is rounded, for a [M, K] and b [N, K].

    A term takes part in at most 128 additions of its block and then in one for
    each block behind it (and 16 where waves are joined), each off by at most one
    unit of 2^-23 of the sum of the terms' sizes (truncation included). The E4M3
    instruction first cuts each of 8 neighbouring products 13 bits below the
    exponents of the largest: 7 products, each off by less than 2^-13 of the
    largest, which is at most the product of either side's largest. ``wide``:
    results in 32 bits, summed in fp32 throughout."""
    err = (128 + ceil(a.shape[1], BLOCK) + 16) * 2.0 ** -23 * (a.abs() @ b.abs().t())
    if wide:
        return err
    tops = [torch.nn.functional.pad(t.abs(), (0, -t.shape[1] % 8)).unflatten(1, (-1, 8)).amax(dim=2) for t in (a, b)]
    return err + 7 * 2.0 ** -13 * (tops[0] @ tops[1].t())


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def near(got, ref, bound):
    """`got` within `bound` of `ref`, NaN where it is."""
    got = got.double().cpu()
    ref, bound = ref.double().cpu(), bound.double().cpu()
    assert got.shape == ref.shape
    assert torch.equal(got.isnan(), ref.isnan())
    off = (got - ref).abs()
    off, bound = off[~ref.isnan()], bound[~ref.isnan()]
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert worst <= 0, f"off by {worst} more than its bound; largest difference {off.max().item()}"


def rows_e4m3(gen, rows, cols, device="cuda", low=-3, high=3):
    """Random E4M3 rows with scales of 2^low .. 2^high."""
    q = (torch.randn(rows, cols, generator=gen) * 80).clamp(-448, 448).to(F8)
    s = (torch.randint(low, high + 1, (rows, ceil(cols, BLOCK)), generator=gen) + 127).to(torch.uint8).view(E8)
    return q.to(device), s.to(device)


def blocks_e4m3(gen, rows, cols, device="cuda", low=-3, high=3):
    """A random E4M3 matrix with scales for 128 x 128."""
    q = (torch.randn(rows, cols, generator=gen) * 80).clamp(-448, 448).to(F8)
    s = torch.randint(low, high + 1, (ceil(rows, BLOCK), ceil(cols, BLOCK)), generator=gen) + 127
    return q.to(device), s.to(torch.uint8).view(E8).to(device)
