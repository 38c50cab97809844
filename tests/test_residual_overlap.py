"""``residual_norm_quant(out=)`` over memory of the vectors is refused: every row of a sample reads them."""
import pytest
import torch

from k2q import ops


def test_spans():
    t = torch.zeros(40, dtype=torch.bfloat16)
    at = t.data_ptr()
    v = t[8:24].view(2, 1, 8)
    for first, n, meets in ((0, 16, False), (0, 17, True), (46, 4, True), (48, 4, False), (20, 2, True)):
        assert ops._spans_meet(at + first, n, v) == meets
    assert ops._spans_meet(at + 16, 2, t[8:9].expand(4, 8)) and not ops._spans_meet(at + 18, 2, t[8:9].expand(4, 8))
    assert not ops._spans_meet(at, 80, t[:0])


@pytest.mark.gpu
def test_out_over_a_vector_is_refused():
    buf = torch.zeros(8 * 256, dtype=torch.bfloat16, device="cuda")
    x, y = (torch.ones(1, 4, 256, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    w = torch.zeros(256, device="cuda")
    out, v = buf[:1024].view(1, 4, 256), buf[768:1024].view(1, 1, 256)
    for kw in (dict(gate=v), dict(mod_scale=v), dict(mod_shift=v), dict(norm_scale=buf[512:1024].view(torch.float32))):
        with pytest.raises(ValueError, match="overlaps"):
            ops.residual_norm_quant(x, y, kw.pop("norm_scale", w), **kw, out=out)
    assert (buf == 0).all()
    beside = buf[1024:1280].view(1, 1, 256)
    assert ops.residual_norm_quant(x, y, w, gate=beside, out=out)[0] is out and (out == 1).all()
