"""Residual norm with several rows per thread block (a sample gets as many blocks as the SMs hold): the quantising form, the
dense form and the backward with and without the vectors' gradients, against the formulas in 64 bits.

Tolerances as one rounding to bf16 (2^-8 of the value) over fp32 arithmetic of at most 64 roundings (2^-18) of the terms'
magnitudes, 2^-16 with room for the rotation's seven; a sum over R rows of a sample adds at most R roundings, 2^-24 each."""
import pytest
import torch

from k2q import fused, ops

pytestmark = pytest.mark.gpu

BF, F32 = 2.0 ** -8, 2.0 ** -16


def make(b, l, k, vectors, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")          # noqa: E731
    x = r(b, l, k)
    x[..., :: max(k // 5, 1)] *= 20.0
    t = {"x": x.bfloat16(), "y": (0.5 * r(b, l, k)).bfloat16(), "w": 0.2 * r(k)}
    for n in ("gate", "sc", "sh"):
        t[n] = (0.5 * r(b, 1, k)).bfloat16() if vectors else None
    t["ds"], t["dh"] = r(b, l, k).bfloat16(), r(b, l, k).bfloat16()
    return t


def norm64(kept, t):
    n = kept.double() * (kept.double().square().mean(-1, keepdim=True) + 1e-5) ** -0.5
    f = 1.0 + t["w"].double()
    if t["sc"] is not None:
        f = f * (1.0 + t["sc"].double())
    h = n * f
    size = h.abs()
    if t["sh"] is not None:
        h, size = h + t["sh"].double(), size + t["sh"].double().abs()
    return n, f, h, size


def check_stream(t, stream):
    gy = t["y"].double() if t["gate"] is None else t["gate"].double() * t["y"].double()
    want = t["x"].double() + gy
    assert ((stream.double() - want).abs() <= BF * want.abs() + 2.0 ** -22 * (t["x"].double().abs() + gy.abs())).all()


# rows of one sample over blocks: none of these row counts divides evenly, and every block has several rows.  One to four
# 16-byte vectors per thread; batches whose samples share the SMs.
SHAPES = [(3, 1111, 2560), (1, 5003, 520), (2, 701, 6144), (1, 1201, 8192), (1, 701, 8200), (2, 907, 12296), (1, 701, 16384), (5, 2003, 136)]


@pytest.mark.parametrize("b,l,k", SHAPES)
@pytest.mark.parametrize("modulated", [False, True])
@pytest.mark.parametrize("sums", [False, True])
def test_dense_and_gradients(b, l, k, modulated, sums):
    t = make(b, l, k, modulated, 7)
    names = ["x", "y"] + ([n for n in ("w", "gate", "sc", "sh") if t[n] is not None] if sums else [])
    leaf = {n: (None if t[n] is None else t[n].clone().requires_grad_(n in names)) for n in ("x", "y", "w", "gate", "sc", "sh")}
    stream, h = fused.residual_norm(*leaf.values(), 1e-5)
    check_stream(t, stream)
    n, f, want, size = norm64(stream.detach(), t)
    assert ((h.double() - want).abs() <= BF * want.abs() + F32 * size).all()
    got = dict(zip(names, torch.autograd.grad((stream, h), [leaf[q] for q in names], (t["ds"], t["dh"]))))
    # from the formulas, written out
    rstd = (stream.detach().double().square().mean(-1, keepdim=True) + 1e-5) ** -0.5
    dh, ds = t["dh"].double(), t["ds"].double()
    g = dh * f
    d = ds + rstd * (g - n * (g * n).mean(-1, keepdim=True))
    dsize = ds.abs() + rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    gate = torch.ones(1, dtype=torch.float64, device="cuda") if t["gate"] is None else t["gate"].double()
    assert ((got["x"].double() - d).abs() <= BF * d.abs() + F32 * dsize).all()
    assert ((got["y"].double() - gate * d).abs() <= BF * (gate * d).abs() + F32 * dsize * gate.abs()).all()
    if not sums:
        return
    u = F32 + l * 2.0 ** -24
    per, psize = (dh * n).sum(1, keepdim=True), (dh * n).abs().sum(1, keepdim=True)
    sc = 1.0 if t["sc"] is None else 1.0 + t["sc"].double()
    dw, dwsize = (per * sc).sum((0, 1)), (psize * abs(sc)).sum((0, 1))
    assert ((got["w"].double() - dw).abs() <= (u + b * 2.0 ** -24) * dwsize).all()
    if modulated:
        w = 1.0 + t["w"].double()
        y = t["y"].double()
        for name, value, terms in (("gate", (d * y).sum(1, keepdim=True), (dsize * y.abs()).sum(1, keepdim=True)),
                                   ("sc", per * w, psize * w.abs()), ("sh", dh.sum(1, keepdim=True), dh.abs().sum(1, keepdim=True))):
            assert ((got[name].double() - value).abs() <= BF * value.abs() + u * terms).all(), name


@pytest.mark.parametrize("b,l,k", [(3, 1111, 2560), (1, 701, 8192), (2, 701, 6144), (1, 701, 16384), (1, 5003, 128), (7, 301, 1024)])
@pytest.mark.parametrize("modulated", [False, True])
@pytest.mark.parametrize("inplace", [False, True])
def test_codes(b, l, k, modulated, inplace):
    t = make(b, l, k, modulated, 8)
    x = t["x"].clone()
    stream, xq, sx = ops.residual_norm_quant(x, t["y"], t["w"], t["gate"], t["sc"], t["sh"], 1e-5, out=x if inplace else None)
    check_stream(t, stream)
    _, _, h, size = norm64(stream, t)
    had = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    while had.shape[0] < 128:
        had = torch.cat((torch.cat((had, had), 1), torch.cat((had, -had), 1)), 0)
    r = (h.reshape(-1, 128) @ had / 128 ** 0.5).reshape(-1, k)
    off = (size.reshape(-1, 128).sum(1) / 128 ** 0.5 * F32).repeat_interleave(128).reshape(-1, k)
    step = r.abs().amax(1).clamp(min=1e-8) / 127
    assert ((sx.double() - step).abs() <= off.amax(1) / 127 + 2.0 ** -22 * step).all()
    assert ((xq.double() * sx.double()[:, None] - r).abs() <= 0.5 * sx.double()[:, None] * (1 + 2.0 ** -14) + off).all()
    assert int(xq.to(torch.int32).abs().max()) <= 127


@pytest.mark.parametrize("b,l,k", [(3, 1111, 2560), (2, 701, 6144), (1, 701, 16384)])
def test_one_output_unused_over_several_rows(b, l, k):
    """The norm's gradient or the stream's absent: the same as a gradient of zeros."""
    t = make(b, l, k, True, 9)
    leaf = {n: t[n].clone().requires_grad_(True) for n in ("x", "y", "w", "gate", "sc", "sh")}
    s, h = fused.residual_norm(*leaf.values(), 1e-5)
    zero = torch.zeros_like(t["ds"])
    asked = [leaf[n] for n in ("x", "y", "gate")]
    for one, both in (((s,), (t["ds"], zero)), ((h,), (zero, t["dh"]))):
        a = torch.autograd.grad(one, asked, (both[0] if one[0] is s else both[1],), retain_graph=True)
        c = torch.autograd.grad((s, h), asked, both, retain_graph=True)
        assert all(torch.equal(u, v) for u, v in zip(a, c))
