"""Orthogonalised update of layouts whose thread blocks take several sub-blocks each, of buffers at odd addresses and of
more than 2^31 elements, against the iteration in 64 bits.

Tolerances.  A thread adds its share of a piece in fp32: block / (2 * groups) terms of each sub-block, with
256 / pairs groups of threads and pairs = number of 4 x 4 tiles of the Gram matrix's upper triangle; two more additions join
the halves and up to `groups` the threads; pieces are added in 64 bits.  So |E_ij| <= c 2^-24 |x_i| |x_j| with c = terms + groups + 3
and ||E||_F <= c 2^-24 for ||X||_F <= 1.  P = F(G) moves by at most max |F'| ||E||_F over the spectrum's range; P u adds
S roundings of its terms, u itself at most four, amplified by at most 3.4445^steps."""
import pytest
import torch

from k2q import ops

pytestmark = pytest.mark.gpu

A, B, C = 3.4445, -4.7750, 2.0315
U = 2.0 ** -24


def poly(lam, steps=5):
    f = torch.ones_like(lam)
    for _ in range(steps):
        q = A + B * lam + C * lam * lam
        f, lam = f * q, lam * q * q
    return f


def roundings(s, piece):
    """c of the bound above."""
    s4 = (s + 3) // 4
    groups = 256 // (s4 * (s4 + 1) // 2)
    block = 1024 if s <= 4 else 512 if s <= 8 else 256 if s <= 16 else 128 if s <= 32 else 64
    return -(-block // (2 * groups)) * piece + groups + 3


def factor(gram, eps=1e-7):
    """P of u's Gram matrix in 64 bits (so that X = P u), and the largest |F'| over its spectrum."""
    norm = gram.diagonal().sum().sqrt() + eps
    lam, vec = torch.linalg.eigh(gram / norm ** 2)
    lam = lam.clamp(min=0.0)
    p = (vec * poly(lam)) @ vec.t() / norm
    lo, hi = float(lam.min()), max(float(lam.max()), 1e-12)
    grid = torch.linspace(lo, max(hi, lo * 1.0001), 4001, dtype=torch.float64, device=gram.device)
    steep = float((poly(grid).diff().abs() / grid.diff().clamp(min=1e-300)).max())
    return p, 2 * steep, float(lam.max().sqrt()), norm      # twice: the grid is finer than any gap, not exact


def reference(u, piece, slack=1.0):
    wide = u.double() if u.shape[0] <= u.shape[1] else u.double().t()
    p, steep, top, norm = factor(wide @ wide.t())
    o = p @ wide
    size = float(((p.abs() * norm) @ (wide.abs() / norm)).norm())
    s = wide.shape[0]
    tol = steep * roundings(s, piece) * U * top + (s + 4) * U * size + A ** 5 * 4 * U * slack
    return (o if u.shape[0] <= u.shape[1] else o.t()), tol


# short sides of every block width, wide and tall, long sides of whole and of ragged sub-blocks and 16-byte pieces
KINDS = [(3, 20483), (20480, 4), (7, 9001), (9216, 8), (13, 4099), (5001, 16), (32, 2560), (2563, 31), (57, 2561), (2052, 64), (64, 2048), (1003, 45)]


def flat_of(shapes, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    parts = []
    for r, c in shapes:
        s = min(r, c)
        fall = torch.logspace(0, -0.7, s, device="cuda") if s > 1 else torch.ones(1, device="cuda")
        x = fall[:, None] * torch.randn(s, max(r, c), generator=g, device="cuda") * 1e-3
        parts.append((x if r <= c else x.t()).reshape(-1))
    return torch.cat(parts)


def cut(flat, shapes):
    return [t.view(s) for t, s in zip(flat.split([r * c for r, c in shapes]), shapes)]


@pytest.mark.parametrize("copies", [7, 13, 40])
def test_orthogonalize_in_pieces(copies):
    shapes = KINDS * copies
    layout = ops.MatrixLayout(shapes, "cuda")
    piece = int(layout.plan.piece)
    assert piece > 1
    u = flat_of(shapes, copies)
    out = ops.orthogonalize(u, layout)
    us, outs = cut(u, shapes), cut(out, shapes)
    for i in list(range(len(KINDS))) + list(range(len(shapes) - len(KINDS), len(shapes))):
        want, tol = reference(us[i], piece)
        off = float((outs[i].double() - want).norm())
        assert off <= tol, (shapes[i], piece, off, tol)
    assert torch.equal(ops.orthogonalize(u, layout), out)


@pytest.mark.parametrize("shapes", [[(64, 6144), (10240, 64)] * 30, [(33, 4100), (4095, 35)] * 60, [(16, 20000)] * 130, [(2, 100001), (30000, 5)] * 100])
def test_step_in_pieces(shapes):
    layout = ops.MatrixLayout(shapes, "cuda")
    piece = int(layout.plan.piece)
    assert piece > 1
    g, m, p = flat_of(shapes, 1), flat_of(shapes, 2), flat_of(shapes, 3) * 20
    old = [t.clone() for t in (g, m, p)]
    lr, beta, wd = 0.03, 0.9, 0.1
    ops.orthogonal_step_(p, g, m, layout, lr=lr, momentum=beta, weight_decay=wd, zero_grad=True)
    assert (g == 0).all()
    m2 = beta * old[1].double() + (1 - beta) * old[0].double()
    # beta and 1 - beta reach the kernel as fp32 values: one more rounding each
    msize = beta * old[1].double().abs() + (1 - beta) * old[0].double().abs()
    assert ((m.double() - m2).abs() <= 6 * U * msize).all()
    u, usize = beta * m2 + (1 - beta) * old[0].double(), beta * msize + (1 - beta) * old[0].double().abs()
    for i in (0, 1, len(shapes) // 2, len(shapes) - 2, len(shapes) - 1):
        ui, zi, pi, gi = (cut(t, shapes)[i] for t in (u, usize, old[2].double(), p))
        r, c = shapes[i]
        want, tol = reference(ui, piece, slack=4 * float(zi.norm() / ui.norm()))
        s = lr * 0.2 * max(r, c) ** 0.5
        want = pi * (1 - lr * wd) - s * want
        rounding = 8 * U * float((2 * pi.abs() + (want - pi).abs()).norm())
        assert float((gi.double() - want).norm()) <= s * tol + rounding, (shapes[i], piece)


def test_longest_pieces_of_the_largest_rank():
    """30 sub-blocks per thread block: 960 terms in a thread's sum at rank 64."""
    shapes = [(64, 139259)] * 12
    layout = ops.MatrixLayout(shapes, "cuda")
    assert int(layout.plan.piece) == 30
    u = flat_of(shapes, 9)
    outs, us = cut(ops.orthogonalize(u, layout), shapes), cut(u, shapes)
    for i in (0, 1, 11):
        want, tol = reference(us[i], int(layout.plan.piece))
        assert float((outs[i].double() - want).norm()) <= tol, shapes[i]


@pytest.mark.parametrize("copies", [1, 13])
def test_buffers_at_odd_addresses(copies):
    """Any of the buffers may begin off a 16-byte boundary: the same bits."""
    shapes = KINDS * copies
    layout = ops.MatrixLayout(shapes, "cuda")
    n = layout.numel
    base = [flat_of(shapes, 1), flat_of(shapes, 2), flat_of(shapes, 3)]
    want = [t.clone() for t in base]
    ops.orthogonal_step_(*want, layout, lr=0.1, weight_decay=0.1)
    for odd in ((1, 0, 0), (0, 2, 0), (0, 0, 3), (1, 1, 1)):
        room = [torch.full((n + 8,), 7.0, device="cuda") for _ in range(3)]
        got = [r[o:o + n] for r, o in zip(room, odd)]
        for t, b in zip(got, base):
            t.copy_(b)
        ops.orthogonal_step_(*got, layout, lr=0.1, weight_decay=0.1)
        assert all(torch.equal(t, w) for t, w in zip(got, want)), odd
        assert all((r[:o] == 7).all() and (r[o + n:] == 7).all() for r, o in zip(room, odd))
    u = base[0]
    want = ops.orthogonalize(u, layout)
    room = torch.full((n + 8,), 7.0, device="cuda")
    ops.orthogonalize(u, layout, out=room[1:1 + n])
    assert torch.equal(room[1:1 + n], want) and (room[:1] == 7).all() and (room[1 + n:] == 7).all()


def test_more_than_2_31_elements():
    """One matrix of 2^31 elements and more, and small ones behind it."""
    shapes = [(64, (1 << 25) + 4100), (5, 1003), (2000, 24)]
    layout = ops.MatrixLayout(shapes, "cuda")
    assert layout.numel > 1 << 31
    piece = int(layout.plan.piece)
    g = torch.Generator(device="cuda").manual_seed(3)
    u = torch.empty(layout.numel, device="cuda").normal_(0.0, 1e-3, generator=g)
    first = cut(u, shapes)[0]
    first.mul_(torch.logspace(0, -0.7, 64, device="cuda")[:, None])
    out = ops.orthogonalize(u, layout)
    gram = torch.zeros(64, 64, dtype=torch.float64, device="cuda")
    for c in first.split(1 << 20, dim=1):
        d = c.double()
        gram += d @ d.t()
    p, steep, top, norm = factor(gram)
    # each column by itself: the error of P times the column, S + 4 roundings of its terms, the column's own
    for lo in (0, (1 << 24) - 100, (1 << 25) + 3000):
        x = first[:, lo:lo + 1100].double()
        got, want = cut(out, shapes)[0][:, lo:lo + 1100].double(), p @ x
        tol = (steep * roundings(64, piece) * U * (x / norm).norm(dim=0) + 68 * U * (p.abs() @ x.abs()).norm(dim=0)
               + A ** 5 * 4 * U * (x / norm).norm(dim=0))
        assert ((got - want).norm(dim=0) <= tol).all(), lo
    for i in (1, 2):
        want, tol = reference(cut(u, shapes)[i], piece)
        assert float((cut(out, shapes)[i].double() - want).norm()) <= tol
    m, par, last = torch.zeros_like(u), torch.zeros_like(u), u[-5000:].clone()
    ops.orthogonal_step_(par, u, m, layout, lr=1.0, momentum=0.0, nesterov=False, zero_grad=True)
    for i, s in enumerate(shapes):                               # momentum 0: u is the gradient; p = -s X
        tail, x = cut(par, shapes)[i].reshape(-1)[-4096:], cut(out, shapes)[i].reshape(-1)[-4096:]
        step = torch.tensor(0.2) * torch.tensor(float(max(s))).sqrt()
        assert ((tail.double() + float(step) * x.double()).abs() <= 4 * U * (float(step) * x.double()).abs()).all()
    assert all((c == 0).all() for c in u.split(1 << 28)) and torch.equal(m[-5000:], last)
