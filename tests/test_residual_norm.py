"""Residual update + RMS norm + modulation: the quantising form (``ops.residual_norm_quant``) and the
differentiable dense form (``fused.residual_norm``) against the formulas in 64 bits.

Tolerances: one rounding to bf16 is at most 2^-8 of the value; the fp32 arithmetic in front of it is bounded by
2^-16 of the terms' magnitudes.  (The norm's sum of squares runs over at most 32 products per thread, five
shuffle steps and 16 warps: 53 roundings of 2^-24; rsqrt, the products with the weights and the additions add
fewer than ten; 64 * 2^-24 = 2^-18.  The rotation adds seven.)  Sums over R rows add R * 2^-24.
"""
import pytest
import torch

from k2q import fused, ops

BF, F32U = 2.0 ** -8, 2.0 ** -16


def make(b, l, k, modulated, seed, device, zero_row=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)          # noqa: E731
    x = r(b, l, k)
    x[..., :: max(k // 5, 1)] *= 20.0
    y = 0.5 * r(b, l, k)
    if zero_row and l > 1:
        x[0, -1] = 0
        y[0, -1] = 0
    t = {"x": x.bfloat16(), "y": y.bfloat16(), "w": 0.2 * r(k), "gate": None, "sc": None, "sh": None}
    if modulated:
        t["gate"], t["sc"], t["sh"] = ((0.5 * r(b, 1, k)).bfloat16() for _ in range(3))
    t["ds"], t["dh"] = r(b, l, k).bfloat16(), r(b, l, k).bfloat16()
    return {n: None if v is None else v.to(device) for n, v in t.items()}


def norm64(kept, w, sc, sh, eps):
    v = kept.double()
    n = v * (v.square().mean(-1, keepdim=True) + eps) ** -0.5
    f = 1.0 + w.double()
    if sc is not None:
        f = f * (1.0 + sc.double())
    h = n * f
    size = h.detach().abs()
    if sh is not None:
        h = h + sh.double()
        size = size + sh.detach().double().abs()
    return h, n, f, size


def check_stream(t, stream):
    gy = t["y"].double() if t["gate"] is None else t["gate"].double() * t["y"].double()
    want = t["x"].double() + gy
    size = t["x"].double().abs() + gy.abs()
    assert ((stream.double() - want).abs() <= BF * want.abs() + 2.0 ** -22 * size).all()


def hadamard(k, device):
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < 128:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    return (h / 128 ** 0.5).to(device)


def check_codes(t, stream, xq, sx, eps):
    k = stream.shape[-1]
    h, _, _, size = norm64(stream, t["w"], t["sc"], t["sh"], eps)
    r = (h.reshape(-1, 128) @ hadamard(k, stream.device)).reshape(-1, k)
    off = (size.reshape(-1, 128).sum(1) / 128 ** 0.5 * F32U).repeat_interleave(128).reshape(-1, k)
    want = r.abs().amax(1).clamp(min=1e-8) / 127
    assert ((sx.double() - want).abs() <= off.amax(1) / 127 + 2.0 ** -22 * want).all()
    got = xq.double() * sx.double()[:, None]
    assert ((got - r).abs() <= 0.5 * sx.double()[:, None] * (1 + 2.0 ** -14) + off).all()
    assert int(xq.to(torch.int32).abs().max()) <= 127


SHAPES = [(1, 1, 128), (1, 1, 6144), (3, 5, 256), (2, 7, 2560), (1, 33, 6144), (2, 3, 16384), (2, 130, 640), (1, 700, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("b,l,k", SHAPES)
@pytest.mark.parametrize("modulated", [False, True])
def test_quant_against_64_bits(b, l, k, modulated):
    t = make(b, l, k, modulated, 11, "cuda")
    stream, xq, sx = ops.residual_norm_quant(t["x"], t["y"], t["w"], t["gate"], t["sc"], t["sh"], 1e-5)
    assert stream.shape == t["x"].shape and xq.shape == (b * l, k) and sx.shape == (b * l,)
    check_stream(t, stream)
    check_codes(t, stream, xq, sx, 1e-5)


@pytest.mark.gpu
def test_quant_each_vector_alone_strides_and_out():
    b, l, k = 2, 9, 384
    t = make(b, l, k, True, 12, "cuda")
    for only in ("gate", "sc", "sh"):
        one = dict(t, **{n: t[n] if n == only else None for n in ("gate", "sc", "sh")})
        stream, xq, sx = ops.residual_norm_quant(one["x"], one["y"], one["w"], one["gate"], one["sc"], one["sh"], 1e-3)
        check_stream(one, stream)
        check_codes(one, stream, xq, sx, 1e-3)
    want = ops.residual_norm_quant(t["x"], t["y"], t["w"], t["gate"], t["sc"], t["sh"])
    wide = torch.zeros(b, l, k + 64, dtype=torch.bfloat16, device="cuda")
    wide[..., 8:8 + k] = t["x"]
    xs = wide[..., 8:8 + k]                                      # rows inside a wider buffer
    odd = torch.zeros(b * l * k + 1, dtype=torch.bfloat16, device="cuda")
    odd[1:] = t["y"].reshape(-1)
    ys = odd[1:].view(b, l, k)                                   # a base that is not 16-byte aligned
    got = ops.residual_norm_quant(xs, ys, t["w"], t["gate"].expand(b, 1, k), t["sc"][:, 0], t["sh"])
    for u, v in zip(want, got):
        assert torch.equal(u, v)
    guard = torch.full((b, l, k + 64), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.residual_norm_quant(t["x"], t["y"], t["w"], t["gate"], t["sc"], t["sh"], out=guard[..., 8:8 + k])
    assert torch.equal(guard[..., 8:8 + k], want[0]) and (guard[..., :8] == 7).all() and (guard[..., 8 + k:] == 7).all()
    for target in ("x", "y"):                                    # in place
        c = dict(t, **{target: t[target].clone()})
        got = ops.residual_norm_quant(c["x"], c["y"], t["w"], t["gate"], t["sc"], t["sh"], out=c[target])
        assert got[0] is c[target]
        for u, v in zip(want, got):
            assert torch.equal(u, v)


@pytest.mark.gpu
def test_quant_empty_and_special_rows():
    k = 256
    w = torch.zeros(k, device="cuda")
    z = torch.empty(2, 0, k, dtype=torch.bfloat16, device="cuda")
    stream, xq, sx = ops.residual_norm_quant(z, z, w)
    assert stream.shape == z.shape and xq.shape == (0, k) and sx.numel() == 0
    x = torch.zeros(1, 4, k, dtype=torch.bfloat16, device="cuda")
    x[0, 1, 3] = float("nan")
    x[0, 2] = 3.0
    clean = x.clone()
    clean[0, 1] = 0
    a, b = ops.residual_norm_quant(x, torch.zeros_like(x), w), ops.residual_norm_quant(clean, torch.zeros_like(x), w)
    keep = [0, 2, 3]                                             # a row of NaN stays its own affair
    assert torch.equal(a[1][keep], b[1][keep]) and torch.equal(a[2][keep], b[2][keep])
    assert (b[1][0] == 0).all() and b[2][0] > 0


@pytest.mark.gpu
@pytest.mark.parametrize("b,l,k", [(1, 1, 8), (2, 3, 136), (3, 5, 2560), (2, 33, 6144), (1, 4, 8200), (2, 2, 16384), (1, 700, 512)])
@pytest.mark.parametrize("modulated", [False, True])
@pytest.mark.parametrize("vectors", [False, True])
def test_dense_and_gradients_against_64_bits(b, l, k, modulated, vectors):
    t = make(b, l, k, modulated, 21, "cuda")
    names = ["x", "y"] + ([n for n in ("w", "gate", "sc", "sh") if t[n] is not None] if vectors else [])
    leaf = {n: (v if v is None else v.clone().requires_grad_(n in names)) for n, v in t.items()}
    stream, h = fused.residual_norm(leaf["x"], leaf["y"], leaf["w"], leaf["gate"], leaf["sc"], leaf["sh"], 1e-5)
    check_stream(t, stream)
    got = dict(zip(names, torch.autograd.grad((stream, h), [leaf[n] for n in names], (t["ds"], t["dh"]))))

    v = stream.detach().double().requires_grad_(True)
    p = {n: None if t[n] is None else t[n].double().requires_grad_(True) for n in ("w", "sc", "sh")}
    want, n, f, size = norm64(v, p["w"], p["sc"], p["sh"], 1e-5)
    assert ((h.double() - want).abs() <= BF * want.abs() + F32U * size).all()
    asked = [v] + [p[q] for q in ("w", "sc", "sh") if p[q] is not None]
    dv, *rest = torch.autograd.grad(want, asked, t["dh"].double())
    ref = dict(zip([q for q in ("w", "sc", "sh") if p[q] is not None], rest))
    d = t["ds"].double() + dv
    gd = t["dh"].double() * f.detach()
    n = n.detach()
    rstd = (v.detach().square().mean(-1, keepdim=True) + 1e-5) ** -0.5
    dsize = t["ds"].double().abs() + rstd * (gd.abs() + n.abs() * (gd * n).abs().mean(-1, keepdim=True))
    gate = torch.ones(1, device="cuda").double() if t["gate"] is None else t["gate"].double()
    assert ((got["x"].double() - d).abs() <= BF * d.abs() + F32U * dsize).all()
    assert ((got["y"].double() - gate * d).abs() <= BF * (gate * d).abs() + F32U * dsize * gate.abs()).all()
    if vectors:
        u = F32U + b * l * 2.0 ** -24
        s_size = (t["dh"].double() * n).abs()
        per = 1.0 if t["sc"] is None else (1.0 + t["sc"].double()).abs()
        assert got["w"].dtype == torch.float32
        assert ((got["w"].double() - ref["w"]).abs() <= u * (s_size * per).sum((0, 1)) + 2.0 ** -22 * ref["w"].abs()).all()
        if modulated:
            dg = (d * t["y"].double()).sum(1, keepdim=True)
            size = (dsize * t["y"].double().abs()).sum(1, keepdim=True)
            assert ((got["gate"].double() - dg).abs() <= BF * dg.abs() + u * size).all()
            size = s_size.sum(1, keepdim=True) * (1.0 + t["w"].double()).abs()
            assert ((got["sc"].double() - ref["sc"]).abs() <= BF * ref["sc"].abs() + u * size).all()
            size = t["dh"].double().abs().sum(1, keepdim=True)
            assert ((got["sh"].double() - ref["sh"]).abs() <= BF * ref["sh"].abs() + u * size).all()


@pytest.mark.gpu
def test_gradients_against_differences():
    """Directional derivative of sum(ds * stream + dh * h), unrounded, by central differences in 64 bits."""
    t = make(2, 6, 136, True, 31, "cuda", zero_row=False)
    names = ["x", "y", "w", "gate", "sc", "sh"]
    leaf = {n: t[n].clone().requires_grad_(True) for n in names}
    stream, h = fused.residual_norm(leaf["x"], leaf["y"], leaf["w"], leaf["gate"], leaf["sc"], leaf["sh"], 1e-2)
    grads = torch.autograd.grad((stream, h), [leaf[n] for n in names], (t["ds"], t["dh"]))

    def loss(a):
        s = a["x"] + a["gate"] * a["y"]
        hh = norm64(s, a["w"], a["sc"], a["sh"], 1e-2)[0]
        return float((t["ds"].double() * s).sum() + (t["dh"].double() * hh).sum())

    base = {n: t[n].double() for n in names}
    gen = torch.Generator(device="cuda").manual_seed(5)
    for i, n in enumerate(names):
        dirn = torch.randn(base[n].shape, generator=gen, device="cuda", dtype=torch.float64)
        step = 1e-5
        up, down = dict(base, **{n: base[n] + step * dirn}), dict(base, **{n: base[n] - step * dirn})
        diff = (loss(up) - loss(down)) / (2 * step)
        dot = float((grads[i].double() * dirn).sum())
        # one bf16 rounding of each gradient entry, and the bf16 rounding of the stream that the kernel's norm reads
        # (it moves each term of the gradient by up to a few times 2^-8 of the terms it is made of)
        size = float((grads[i].double().abs() * dirn.abs()).sum())
        assert abs(dot - diff) <= 4 * BF * size + 1e-6 * abs(diff), n


@pytest.mark.gpu
def test_one_output_used_and_shared_inputs():
    t = make(2, 5, 256, True, 41, "cuda")
    x, y, gate = (t[n].clone().requires_grad_(True) for n in ("x", "y", "gate"))
    s, h = fused.residual_norm(x, y, t["w"], gate, t["sc"], t["sh"])
    gx, gy, gg = torch.autograd.grad(s, (x, y, gate), t["ds"], retain_graph=True)       # the norm unused
    assert torch.equal(gx, t["ds"]) and torch.equal(gy, (t["ds"].float() * t["gate"].float()).bfloat16())
    want = (t["ds"].double() * t["y"].double()).sum(1, keepdim=True)
    size = (t["ds"].double() * t["y"].double()).abs().sum(1, keepdim=True)
    assert ((gg.double() - want).abs() <= BF * want.abs() + F32U * size).all()
    (a,) = torch.autograd.grad(h, x, t["dh"], retain_graph=True)                        # the stream unused
    (b,) = torch.autograd.grad((s, h), x, (torch.zeros_like(t["ds"]), t["dh"]))
    assert torch.equal(a, b)
    # the same tensor as x and y, no gate: both gradients arrive
    x2 = t["x"].clone().requires_grad_(True)
    s, h = fused.residual_norm(x2, x2, t["w"])
    (g2,) = torch.autograd.grad(s, x2, t["ds"])
    assert torch.equal(g2, t["ds"] * 2)
    # a gate shared by the samples
    shared = t["gate"][:1].clone().requires_grad_(True)
    s, _ = fused.residual_norm(t["x"], t["y"], t["w"], shared.expand(2, 1, 256), t["sc"], t["sh"])
    (gs,) = torch.autograd.grad(s, shared, t["ds"])
    want = (t["ds"].double() * t["y"].double()).sum((0, 1))
    size = (t["ds"].double() * t["y"].double()).abs().sum((0, 1))
    assert ((gs[0, 0].double() - want).abs() <= BF * want.abs() + (F32U + 2 * BF) * size).all()


@pytest.mark.gpu
def test_repeatable_on_side_stream_and_in_a_graph():
    t = make(2, 300, 512, True, 51, "cuda")
    args = (t["x"], t["y"], t["w"], t["gate"], t["sc"], t["sh"])
    want = ops.residual_norm_quant(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.residual_norm_quant(*args)
    side.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.residual_norm_quant(*args)
    for g in got:
        g.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(want, got))
    names = ("x", "y", "w", "gate", "sc", "sh")
    leaf = [t[n].clone().requires_grad_(True) for n in names]
    runs = []
    for _ in range(2):
        out = fused.residual_norm(*leaf)
        runs.append(torch.autograd.grad(out, leaf, (t["ds"], t["dh"])))
    assert all(torch.equal(u, v) for u, v in zip(*runs))


@pytest.mark.gpu
def test_rows_past_32_bits_and_many_samples():
    """More than 2^31 elements: the last rows, alone, give the same; 70000 samples of one row, summed."""
    m, k = 350000, 6144
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.empty(1, m, k, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    y = torch.empty_like(x).normal_(generator=g)
    w = torch.randn(k, generator=g, device="cuda") * 0.1
    gate, sc, sh = ((torch.randn(1, 1, k, generator=g, device="cuda") * 0.5).bfloat16() for _ in range(3))
    stream, xq, sx = ops.residual_norm_quant(x, y, w, gate, sc, sh)
    few = ops.residual_norm_quant(x[:, -7:].contiguous(), y[:, -7:].contiguous(), w, gate, sc, sh)
    assert torch.equal(stream[:, -7:], few[0]) and torch.equal(xq[-7:], few[1]) and torch.equal(sx[-7:], few[2])
    del stream, xq, sx
    s, h = fused.residual_norm(x, y, w, gate, sc, sh)
    s7, h7 = fused.residual_norm(x[:, -7:].contiguous(), y[:, -7:].contiguous(), w, gate, sc, sh)
    assert torch.equal(s[:, -7:], s7) and torch.equal(h[:, -7:], h7)
    del x, y, s, h
    b, k = 70000, 16
    x = torch.randn(b, 1, k, generator=g, device="cuda").bfloat16()
    y = torch.randn(b, 1, k, generator=g, device="cuda").bfloat16()
    gate = torch.randn(b, 1, k, generator=g, device="cuda").bfloat16().requires_grad_(True)
    s, _ = fused.residual_norm(x, y, torch.zeros(k, device="cuda"), gate)
    (gg,) = torch.autograd.grad(s, gate, x)
    assert torch.equal(gg, (x.float() * y.float()).bfloat16())


@pytest.mark.gpu
def test_backward_captured_in_a_graph():
    t = make(2, 40, 512, True, 71, "cuda")
    names = ("x", "y", "w", "gate", "sc", "sh")

    def step(leaf):
        out = fused.residual_norm(*(leaf[n] for n in names))
        return torch.autograd.grad(out, [leaf[n] for n in names], (t["ds"], t["dh"]))

    eager = {n: t[n].clone().requires_grad_(True) for n in names}
    want = step(eager)
    leaf = {n: t[n].clone().requires_grad_(True) for n in names}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(leaf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step(leaf)
    for g in got:
        g.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for u, v in zip(got, want))


@pytest.mark.gpu
def test_in_place_write_is_seen_by_autograd():
    t = make(1, 4, 256, False, 81, "cuda")
    x = t["x"].clone().requires_grad_(True)
    stream, h = fused.residual_norm(x, t["y"], t["w"])
    kept = stream.detach()
    ops.residual_norm_quant(t["x"], t["y"], t["w"], out=kept)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(h, x, t["dh"])


# ---------------------------------------------------------------------------------------------- no GPU
@pytest.mark.parametrize("modulated", [False, True])
def test_composed_form_on_cpu(modulated):
    t = make(2, 5, 24, modulated, 61, "cpu")
    leaf = {n: None if v is None else v.clone().requires_grad_(n in ("x", "y", "w", "gate")) for n, v in t.items()}
    s, h = fused.residual_norm(leaf["x"], leaf["y"], leaf["w"], leaf["gate"], leaf["sc"], leaf["sh"], 1e-5)
    assert s.dtype == h.dtype == torch.bfloat16
    check_stream(t, s.detach())
    want, _, _, size = norm64(s.detach(), t["w"], t["sc"], t["sh"], 1e-5)
    assert ((h.double() - want).abs() <= BF * want.abs() + F32U * size).all()
    (s.float().sum() + h.float().sum()).backward()
    assert leaf["x"].grad is not None and leaf["w"].grad is not None


def test_refusals():
    x = torch.zeros(2, 3, 256, dtype=torch.bfloat16)
    w = torch.zeros(256)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.residual_norm_quant(x, x, w)
    for a, b, n in ((x.float(), x, w), (x, x[:, :2], w), (x, x, w.double()), (x, x, w[:128]), (x[0, 0], x[0, 0], w)):
        with pytest.raises(ValueError):
            ops._check_residual("t", a, b, n, 256)
    for v in (torch.zeros(2, 256), torch.zeros(1, 256, dtype=torch.bfloat16), torch.zeros(256, 2, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            ops._mod_vec("t", "gate", v, 2, 256)
    for o in (x.transpose(1, 2).contiguous().transpose(1, 2), torch.zeros(2, 3, 260, dtype=torch.bfloat16)[..., :256]):
        with pytest.raises(ValueError):
            ops._out_rows("t", o, 256)


@pytest.mark.gpu
def test_refusals_on_gpu():
    x = torch.zeros(2, 3, 256, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(256, device="cuda")
    buf = torch.zeros(2 * 3 * 256 + 256, dtype=torch.bfloat16, device="cuda")
    a, b = buf[:1536].view(2, 3, 256), buf[256:].view(2, 3, 256)
    bad = [dict(x=x[..., :200], y=x[..., :200], norm_scale=w[:200].contiguous()), dict(x=a, y=x, norm_scale=w, out=b),
           dict(x=x, y=x.cpu(), norm_scale=w), dict(x=x, y=x, norm_scale=w, out=x.float()),
           dict(x=x, y=x, norm_scale=w, gate=torch.zeros(3, 256, dtype=torch.bfloat16, device="cuda"))]
    for kw in bad:
        with pytest.raises((ValueError, RuntimeError)):
            ops.residual_norm_quant(**kw)
    s, h = fused.residual_norm(x.requires_grad_(True), x.detach(), w)
    (g,) = torch.autograd.grad(h.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()
