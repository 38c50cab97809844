"""Orthogonalised update of flat adapter buffers against the iteration in 64 bits (singular value decomposition).

Tolerances.  With u normalised to X (||X||_F <= 1), G = X X^T is formed from fp32 products, 32 of them added in
fp32: an error E with |E_ij| <= 33 * 2^-24 |x_i| |x_j|, so ||E||_F <= 33 * 2^-24, and one more rounding of each
piece's sum.  P = F(G) for the scalar function F, and ||F(G + E) - F(G)||_F <= max |F[s, t]| ||E||_F over divided
differences between eigenvalues (largest over the spectrum's range: computed in the test).  The product P u
adds S roundings of its terms, u itself at most four roundings, amplified by at most 3.4445^steps.
"""
import pytest
import torch

from k2q import ops

A, B, C = 3.4445, -4.7750, 2.0315
U = 2.0 ** -24


def poly(lam, steps):
    f = torch.ones_like(lam)
    for _ in range(steps):
        q = A + B * lam + C * lam * lam
        f, lam = f * q, lam * q * q
    return f


def reference(u, steps=5, eps=1e-7, slack=None):
    """X of one matrix in 64 bits and how far an fp32 computation may be from it, elementwise in norm."""
    u = u.double()
    wide = u if u.shape[0] <= u.shape[1] else u.t()
    norm = wide.norm()
    x = wide / (norm + eps)
    left, s, right = torch.linalg.svd(x, full_matrices=False)
    lam = s.square()
    f = poly(lam, steps)
    o = (left * (f * s)) @ right
    p = (left * f) @ left.t()
    grid = torch.linspace(float(lam.min()), max(float(lam.max()), 1e-12), 4001, dtype=torch.float64, device=u.device)
    lipschitz = float((poly(grid, steps).diff().abs() / grid.diff().clamp(min=1e-300)).max()) if lam.max() > lam.min() else \
        abs(float((poly(lam[:1] * 1.0001 + 1e-12, steps) - poly(lam[:1], steps)) / (lam[:1] * 1e-4 + 1e-12)))
    smooth = 2 * lipschitz * 34 * U                       # twice: the grid is finer than any gap, not exact
    size = (p.abs() @ x.abs()).norm()
    tol = smooth * float(s.max()) + (x.shape[0] + 4) * U * float(size) + A ** steps * 4 * U * (1.0 if slack is None else slack)
    return (o if u.shape[0] <= u.shape[1] else o.t()), float(tol)


def matrix(rows, cols, seed, fall=0.2):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")      # noqa: E731
    s, l = min(rows, cols), max(rows, cols)
    d = torch.logspace(0, torch.log10(torch.tensor(fall)).item(), s, device="cuda") if s > 1 else torch.ones(1, device="cuda")
    x = d[:, None] * r(s, l)
    return (x if rows <= cols else x.t()).contiguous() * 1e-3


SHAPES = [(1, 1), (1, 500), (500, 1), (2, 2), (4, 129), (300, 7), (16, 2560), (2560, 16), (32, 6144), (33, 1001), (1001, 33),
          (57, 2561), (64, 64), (64, 4096), (5000, 64), (63, 65)]


def close(got, want, tol):
    return float((got.double() - want).norm()) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 5])
def test_orthogonalize(steps):
    mats = [matrix(r, c, 10 + i) for i, (r, c) in enumerate(SHAPES)]
    layout = ops.MatrixLayout(SHAPES, "cuda")
    flat = torch.cat([m.reshape(-1) for m in mats])
    out = ops.orthogonalize(flat, layout, steps=steps)
    off = 0
    for m in mats:
        want, tol = reference(m, steps)
        got = out[off:off + m.numel()].view_as(m)
        assert close(got, want, tol), (tuple(m.shape), float((got.double() - want).norm()), tol)
        off += m.numel()
    # no step: u / (|u| + eps).  The kernel rounds u^2 (half of that after the root), the reciprocal and the product,
    # 2.5 U; the expression here the sum and the quotient, 2 U
    none, plain = ops.orthogonalize(flat, layout, steps=0)[0], flat[0] / (flat[0].abs() + 1e-7)
    assert abs(float(none) - float(plain)) <= 4.6 * U * abs(float(plain))
    again = ops.orthogonalize(flat, layout, steps=steps)
    assert torch.equal(again, out)
    inplace = flat.clone()
    assert ops.orthogonalize(inplace, layout, steps=steps, out=inplace) is inplace and torch.equal(inplace, out)


@pytest.mark.gpu
def test_singular_values_move_to_one():
    m = matrix(24, 3000, 3, fall=0.05)
    out = ops.orthogonalize(m.reshape(-1), ops.MatrixLayout([(24, 3000)], "cuda")).view(24, 3000)
    s = torch.linalg.svdvals(out.double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("scale", ["rms", "spectral"])
def test_step(nesterov, scale):
    shapes = [(8, 1000), (777, 8), (40, 333), (64, 200), (1, 31)]
    layout = ops.MatrixLayout(shapes, "cuda")
    g = [matrix(r, c, 40 + i) for i, (r, c) in enumerate(shapes)]
    m = [matrix(r, c, 60 + i) for i, (r, c) in enumerate(shapes)]
    p = [matrix(r, c, 80 + i) * 20 for i, (r, c) in enumerate(shapes)]
    cat = lambda ts: torch.cat([t.reshape(-1) for t in ts])        # noqa: E731
    fg, fm, fp = cat(g), cat(m), cat(p)
    keep = fg.clone()
    lr, beta, wd, max_norm = 0.03, 0.9, 0.1, 0.5 * float(fg.norm())
    normsq = fg.double().square().sum().float().reshape(1)
    ops.orthogonal_step_(fp, fg, fm, layout, lr=lr, momentum=beta, nesterov=nesterov, weight_decay=wd, scale=scale,
                         max_norm=max_norm, normsq=normsq)
    assert torch.equal(fg, keep)
    clip = min(1.0, max_norm / (float(normsq.double().sqrt()) + 1e-6))
    off = 0
    for (r, c), gi, mi, pi in zip(shapes, g, m, p):
        n = r * c
        gd, md, pd = gi.double() * clip, mi.double(), pi.double()
        m2 = beta * md + (1 - beta) * gd
        # beta and 1 - beta reach the kernel as fp32 values: one more rounding each; the clip factor adds four
        msize = beta * md.abs() + (1 - beta) * gd.abs()
        got_m, got_p = fm[off:off + n].view(r, c), fp[off:off + n].view(r, c)
        assert ((got_m.double() - m2).abs() <= 10 * U * msize).all()
        u = beta * m2 + (1 - beta) * gd if nesterov else m2
        usize = beta * msize + (1 - beta) * gd.abs() if nesterov else msize
        want, tol = reference(u, slack=4 * float(usize.norm() / u.norm()))
        s = lr * (0.2 * max(r, c) ** 0.5 if scale == "rms" else max(1.0, r / c) ** 0.5)
        want = pd * (1 - lr * wd) - s * want
        rounding = 8 * U * float((pd.abs() + s * (want - pd).abs() / max(s, 1e-9) + pd.abs()).norm())
        assert close(got_p, want, s * tol + rounding), (r, c)
        off += n


@pytest.mark.gpu
def test_zero_and_broken_matrices_keep_to_themselves():
    shapes = [(4, 600), (600, 4), (4, 600), (16, 128)]
    layout = ops.MatrixLayout(shapes, "cuda")
    mats = [matrix(r, c, 5 + i) for i, (r, c) in enumerate(shapes)]
    clean = torch.cat([t.reshape(-1) for t in mats])
    dirty = clean.clone()
    dirty[:2400] = 0                                             # the adapter whose partner is still zero: no gradient
    dirty[2400 + 77] = float("nan")
    p0 = torch.randn_like(clean)
    runs = []
    for gsrc in (clean, dirty):
        p, gr, m = p0.clone(), gsrc.clone(), torch.zeros_like(clean)
        ops.orthogonal_step_(p, gr, m, layout, lr=0.1, weight_decay=0.5, zero_grad=True)
        assert (gr == 0).all()
        runs.append(p)
    assert torch.equal(runs[1][:2400], p0[:2400] * torch.tensor(1.0 - 0.1 * 0.5))
    assert runs[1][2400:4800].isnan().all()
    assert torch.equal(runs[0][4800:], runs[1][4800:]) and torch.isfinite(runs[0]).all()


@pytest.mark.gpu
def test_streams_graph_and_shared_layout():
    shapes = [(16, 900), (700, 16)] * 3
    layout = ops.MatrixLayout(shapes, "cuda")
    flat = torch.cat([matrix(r, c, i).reshape(-1) for i, (r, c) in enumerate(shapes)])

    def buffers(k):
        return torch.ones_like(flat), flat * (1 + k), torch.zeros_like(flat)

    want = []
    for k in range(2):
        b = buffers(k)
        ops.orthogonal_step_(*b, layout, lr=0.1)
        want.append(b)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [buffers(k) for k in range(2)]
    torch.cuda.synchronize()
    for s, b in zip(streams, got):                               # two calls at once on one layout
        with torch.cuda.stream(s):
            ops.orthogonal_step_(*b, layout, lr=0.1)
    torch.cuda.synchronize()
    for w, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(w, b))
    graphs, bufs = [], []
    for k in range(2):                                           # two graphs, replayed at once
        b = buffers(k)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.orthogonal_step_(*b, layout, lr=0.1)
        graphs.append(graph)
        bufs.append(b)
    for s, graph in zip(streams, graphs):
        with torch.cuda.stream(s):
            graph.replay()
    torch.cuda.synchronize()
    for w, b in zip(want, bufs):
        assert all(torch.equal(x, y) for x, y in zip(w, b))


def test_layout_and_refusals():
    layout = ops.MatrixLayout([(4, 100), (50, 3)], "cpu")
    assert layout.numel == 550 and layout.plan.count == 2
    for bad in ([], [(65, 65)], [(0, 4)], [(4, -1)], [(3,)]):
        with pytest.raises(ValueError):
            ops.MatrixLayout(bad, "cpu")
    t = torch.zeros(550)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.orthogonal_step_(t, t.clone(), t.clone(), layout, lr=0.1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.orthogonalize(t, layout)


@pytest.mark.gpu
def test_refusals_on_gpu():
    layout = ops.MatrixLayout([(4, 100), (50, 3)], "cuda")
    t = lambda n=550, d=torch.float32: torch.zeros(n, device="cuda", dtype=d)      # noqa: E731
    a, big = t(), t(1000)
    for p, g, m, kw in ((t(549), t(), t(), {}), (t(), t(550, torch.float64), t(), {}), (a, a, t(), {}), (t(), t(), t(), {"scale": "x"}),
                        (t(), t(), t(), {"steps": 11}), (t(), t(), t(), {"normsq": t(2)}), (big[:550], big[100:650], t(), {}),
                        (t(1100)[::2], t(), t(), {})):
        with pytest.raises(ValueError):
            ops.orthogonal_step_(p, g, m, layout, lr=0.1, **kw)
    with pytest.raises(ValueError):
        ops.orthogonalize(big[:550], layout, out=big[100:650])


@pytest.mark.gpu
def test_clipping_needs_the_norm():
    layout = ops.MatrixLayout([(4, 100)], "cuda")
    p, g, m = (torch.ones(400, device="cuda") for _ in range(3))
    with pytest.raises(ValueError, match="normsq"):
        ops.orthogonal_step_(p, g, m, layout, lr=0.1, max_norm=1.0)
    assert all(torch.equal(t, torch.ones_like(t)) for t in (p, g, m))


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 19, 75])
def test_few_and_many_matrices_of_large_rank(count):
    """A matrix's result does not depend on how many stand beside it (one piece per matrix, so that its Gram sums
    are formed in one order)."""
    kinds = [(33, 50), (64, 64), (61, 57), (40, 41), (5, 64)]
    shapes = [kinds[i % 5] for i in range(count)]
    mats = [matrix(r, c, i) for i, (r, c) in enumerate(kinds)]
    flat = torch.cat([mats[i % 5].reshape(-1) for i in range(count)])
    got = ops.orthogonalize(flat, ops.MatrixLayout(shapes, "cuda")).split([r * c for r, c in shapes])
    many = torch.cat([m.reshape(-1) for m in mats]).repeat(32)                   # 160 matrices
    want = ops.orthogonalize(many, ops.MatrixLayout(kinds * 32, "cuda")).split([r * c for r, c in kinds * 32])
    for i in range(count):
        assert torch.equal(got[i], want[i % 5]), shapes[i]
