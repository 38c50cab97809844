"""The products' GELU (tanh form) against 64 bits, negative arguments included, where 0.5 v (1 + tanh z) would cancel.

Codes of zero make the argument the bias itself.  Tolerance: the exponent t = -2 z log2(e), |t| < 72 for |v| <= 8, is
formed with roundings of at most 3.5 * 2^-24 of it (1.1e-5 of the exponential), the hardware's exponential is good to
2^-22, its reciprocal to 2^-23, a sum and a product add 2^-23: below 2^-16 of the value in all; then one rounding to
bf16, 2^-8 of the value."""
import math

import pytest
import torch

from k2q import ops

pytestmark = pytest.mark.gpu


def arguments():
    v = torch.cat((torch.linspace(-8, 8, 1001), torch.linspace(-5, -1, 500), torch.tensor([0.0, -0.0, 1e-20, -1e-20, 30.0])))
    return torch.cat((v, torch.full(((-v.numel()) % 16,), -3.0)))


def expected(v):
    z = math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)
    return v / (1.0 + torch.exp(-2.0 * z))


def product(kind, m, bias, rank):
    n, k = bias.numel(), 256
    xq, sx = torch.zeros(m, k, dtype=torch.int8, device="cuda"), torch.ones(m, device="cuda")
    kw = dict(act="gelu_tanh")
    if rank:                                                     # an adapter term of zero: the other epilogues
        kw |= dict(u=torch.zeros(m, rank, device="cuda"), bm=torch.ones(n, rank, device="cuda"), lora_scale=1.0)
    if kind == 8:
        wq, sw = torch.ones(n, k, dtype=torch.int8, device="cuda"), torch.ones(n, device="cuda")
        y = ops.gemm_w8a8(xq, sx, wq, sw, bias, **kw)
    else:
        wq = torch.full((n, k // 2), 0x11, dtype=torch.uint8, device="cuda")
        sw = torch.ones(n, k // 128, dtype=torch.bfloat16, device="cuda")
        y = ops.gemm_w4a8(xq, sx, wq, sw, bias, **kw)
    ops.check_status()
    return y


@pytest.mark.parametrize("rank", [0, 8, 24])
@pytest.mark.parametrize("kind,m", [(4, 1), (4, 13), (4, 40), (8, 5), (8, 300), (8, 8200)])
def test_gelu_of_every_product(kind, m, rank):
    """4 bits: the few-row kernel up to 16 rows, the large product beyond; 8 bits: one CTA, CTA pairs, the adapter
    term on the fp32 pipe."""
    v = arguments().cuda()
    y = product(kind, m, v, rank).double()
    want = expected(v.double())
    assert ((y - want).abs() <= (2.0 ** -8 + 2.0 ** -16) * want.abs()).all(), float(((y - want).abs() / want.abs().clamp(min=1e-30)).max())


@pytest.mark.parametrize("kind,m", [(4, 2), (4, 40), (8, 300)])
def test_gelu_of_infinities_and_nan(kind, m):
    v = torch.tensor([float("inf"), float("nan"), float("-inf"), -1e30, 1e30, -200.0] + [1.0] * 10, device="cuda")
    y = product(kind, m, v, 0).double()
    assert (y[:, 0] == math.inf).all() and y[:, 1].isnan().all()
    assert y[:, 2].isnan().all()                                 # -inf times a zero, as the formula has it
    assert (y[:, 3] == 0).all() and (y[:, 4] == torch.tensor(1e30).bfloat16().double().item()).all() and (y[:, 5] == 0).all()
