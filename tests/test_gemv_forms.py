"""Few-row W4A8 product: every form that the dispatch reaches against the large product and the CPU oracle, long
contractions, and the large product itself at few rows."""
import ctypes as C

import pytest
import torch

from k2q import _lib, ops
from oracle import convrot_ref as R

pytestmark = pytest.mark.gpu


def make(m, n, k, seed, bias=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    xq = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8, device="cuda")
    wq = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8, device="cuda")
    sx = torch.rand(m, generator=g, device="cuda") * 0.05 + 1e-3
    sw = ((torch.rand(n, k // 128, generator=g, device="cuda") - 0.1) * 0.01).bfloat16()
    b = torch.randn(n, generator=g, device="cuda") if bias else None
    return xq, sx, wq, sw, b


def same_bits(a, b):
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


def large(xq, sx, wq, sw, b, u=None, bm=None, lora_scale=0.0, act=None):
    """``k2q_gemm_w4a8`` itself, whatever the number of rows."""
    (m, k), n = xq.shape, wq.shape[0]
    y = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    ep = ops._epilogue(sx, b, u, bm, lora_scale, act)
    _lib.check(_lib.load().k2q_gemm_w4a8(ops._ptr(xq), ops._ptr(wq), ops._ptr(sw), m, n, k, C.byref(ep), ops._ptr(y), n,
                                         ops._ptr(ops.status_block(y.device)), ops._stream(y.device)), "k2q_gemm_w4a8")
    ops.check_status()
    return y


def rank_operands(m, n, rank):
    g = torch.Generator(device="cuda").manual_seed(rank)
    return dict(u=torch.randn(m, rank, generator=g, device="cuda"), bm=torch.randn(n, rank, generator=g, device="cuda") * 0.1,
                lora_scale=0.6)


@pytest.mark.parametrize("act,rank", [(None, 0), ("gelu_tanh", 0), (None, 19)])
@pytest.mark.parametrize("m,n,k", [
    (1, 36864, 1152), (9, 36864, 1152), (16, 36864, 640), (17, 36864, 1152), (32, 36864, 1152),     # 16 channels per warp
    (3, 18960, 6144), (12, 18960, 6144), (32, 18960, 6144), (25, 36864, 5248),                      # tokens staged again
    (1, 12304, 2560), (13, 12304, 2560), (32, 12304, 2560), (32, 16384, 2688), (20, 9488, 384),     # 9 to 16 warps
    (24, 6144, 6144), (32, 6144, 16384), (17, 2560, 640),                                           # up to 8 warps, one team
    (8, 6144, 16384), (16, 6144, 16384), (16, 1200, 16512), (2, 2368, 1408)])                       # warps share channels
def test_forms_against_the_large_product(m, n, k, act, rank):
    """The rows stand in a batch of 40, which only the large product takes."""
    xq, sx, wq, sw, b = make(40, n, k, 3 * m + n)
    lo = rank_operands(40, n, rank) if rank else {}
    want = ops.gemm_w4a8(xq, sx, wq, sw, b, act=act, **lo)
    ops.check_status()
    if rank:
        lo["u"] = lo["u"][:m]
    got = ops.gemv_w4a8(xq[:m].contiguous(), sx[:m].contiguous(), wq, sw, b, act=act, **lo)
    assert same_bits(got, want[:m])


@pytest.mark.parametrize("m,n,k", [(1, 16, 131072), (2, 1200, 131072), (16, 2368, 65536), (32, 1040, 131072), (32, 6144, 65536),
                                   (9, 18960, 32768), (32, 18960, 32896)])
def test_long_contractions(m, n, k):
    """The scales of a CTA's channels bound how many warps it may have; the tokens are staged many times."""
    xq, sx, wq, sw, b = make(40, n, k, m + n, bias=False)
    want = ops.gemm_w4a8(xq, sx, wq, sw)
    ops.check_status()
    got = ops.gemv_w4a8(xq[:m].contiguous(), sx[:m].contiguous(), wq, sw)
    assert same_bits(got, want[:m])
    rows = slice(0, n, max(n // 8, 1))                           # some channels against the oracle
    cpu = [t.cpu() for t in (xq[:m], sx[:m], wq[rows].contiguous(), sw[rows].contiguous())]
    assert same_bits(got[:, rows].cpu().contiguous(), R.linear_int4_exact(*cpu, None))


def test_past_the_longest_contraction():
    """131200 and more go to the large product; the few-row call itself refuses."""
    k = 131200
    xq, sx, wq, sw, _ = make(20, 32, k, 1, bias=False)
    few = (xq[:2].contiguous(), sx[:2].contiguous(), wq, sw)
    with pytest.raises(ValueError, match="131072"):
        ops.gemv_w4a8(*few)
    assert same_bits(ops.gemm_w4a8(*few), ops.gemm_w4a8(xq, sx, wq, sw)[:2])
    ops.check_status()


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 16])
@pytest.mark.parametrize("n,k,rank,act", [(16, 128, 0, None), (384, 768, 16, None), (272, 2560, 0, "gelu_tanh"), (6144, 640, 32, "gelu_tanh")])
def test_large_product_at_few_rows(m, n, k, rank, act):
    """C callers and the host-buffer call reach it with any number of rows; ``ops.gemm_w4a8`` takes the few-row kernel."""
    xq, sx, wq, sw, b = make(m, n, k, m)
    lo = rank_operands(m, n, rank) if rank else {}
    got = large(xq, sx, wq, sw, b, act=act, **lo)
    assert same_bits(got, ops.gemm_w4a8(xq, sx, wq, sw, b, act=act, **lo))
    if rank == 0 and act is None:
        assert same_bits(got.cpu(), R.linear_int4_exact(*(t.cpu() for t in (xq, sx, wq, sw, b))))
