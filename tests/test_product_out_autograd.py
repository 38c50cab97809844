"""The W4A8 products' writes into a caller's ``out`` are seen by autograd."""
import pytest
import torch

from k2q import ops


@pytest.mark.gpu
@pytest.mark.parametrize("m", [2, 40])
def test_writes_into_out_are_seen_by_autograd(m):
    """Few-row and large product: a graph that saved ``out`` must not read the new values."""
    xq = torch.ones(m, 256, dtype=torch.int8, device="cuda")
    wq = torch.full((64, 128), 0x21, dtype=torch.uint8, device="cuda")
    sx, sw = torch.ones(m, device="cuda"), torch.ones(64, 2, dtype=torch.bfloat16, device="cuda")
    out = torch.ones(m, 64, dtype=torch.bfloat16, device="cuda")
    w = torch.ones_like(out, requires_grad=True)
    loss = (w * out).sum()
    ops.gemm_w4a8(xq, sx, wq, sw, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
