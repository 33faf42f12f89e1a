"""8-bit rows of fp16 inputs with fp16 weights: products of 22 bits, whose
multiple by 127 or 448 no longer fits fp32. Quotients that lie on a rounding
border exactly still round to even."""

import pytest
import torch

import mega_moe

pytestmark = pytest.mark.gpu

F16 = torch.float16


@pytest.mark.parametrize("hidden", [7, 64, 515, 2048, 7168, 16384])
@pytest.mark.parametrize("weight", [2047, 1999, 1365, 1025])
@pytest.mark.parametrize("out_dtype,part,whole,quotient,want", [
    (torch.int8, 1, 2, 63.5, 64.0),            # y / s = 127 / 2
    (torch.int8, 5, 254, 2.5, 2.0),            # 127 * 5 / 254
    (torch.float8_e4m3fn, 3, 64, 21.0, 20.0),  # 448 * 3 / 64, between 20 and 22
    (torch.float8_e4m3fn, 5, 64, 35.0, 35.0),  # between 32 and 36: no border
    (torch.float8_e4m3fn, 9, 448, 9.0, 9.0),
    (torch.float8_e4m3fn, 17, 448, 17.0, 16.0),
])
def test_exact_quotients(hidden, weight, out_dtype, part, whole, quotient, want):
    """Row r holds `part` * m_r and, once, `whole` * m_r: the quotient is the
    same in all of them, whatever m_r and the weight's 11 bits."""
    if out_dtype == torch.float8_e4m3fn:
        want = torch.tensor(quotient).to(out_dtype).float().item()  # round to nearest even
    rows = 64
    m = torch.arange(2047 // part, 2047 // part - rows, -1, device="cuda").clamp(min=1).double()
    x = (m[:, None] * part).expand(rows, hidden).clone()
    x[:, hidden // 2] = m * whole
    assert x[:, 0].max() < 2048
    scale = 2.0 ** -(torch.arange(rows, device="cuda") % 7).double()[:, None] / 4096
    rows16 = (x * scale).to(F16)
    # both are held exactly, or the case says nothing
    exact = (rows16.double() == x * scale).all(1)
    w = torch.full((hidden,), weight / 1024, dtype=F16, device="cuda")
    q, _ = mega_moe.rms_norm(rows16, w, out_dtype=out_dtype)
    q = q.float()[exact]
    assert exact.any()
    top = 127.0 if out_dtype == torch.int8 else 448.0
    ref = torch.full_like(q, want)
    ref[:, hidden // 2] = top
    assert torch.equal(q, ref), (q != ref).sum().item()
