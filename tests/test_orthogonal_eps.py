"""The norm's epsilon at its limits: none at all, one whose reciprocal leaves fp32, and refusals."""
import pytest
import torch

from k2q import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [0.0, 1e-38, 1e-45, 1e-7])
@pytest.mark.parametrize("steps", [0, 1, 5])
def test_zero_matrix_moves_by_its_decay_alone(eps, steps):
    shapes = [(4, 300), (300, 4), (40, 70)]
    layout = ops.MatrixLayout(shapes, "cuda")
    u = torch.zeros(layout.numel, device="cuda")
    u[1200:2400] = torch.linspace(-1, 1, 1200, device="cuda")    # the one in the middle is not zero
    out = ops.orthogonalize(u, layout, steps=steps, eps=eps)
    assert (out[:1200] == 0).all() and (out[2400:] == 0).all() and torch.isfinite(out).all() and (out[1200:2400] != 0).any()
    p = torch.randn(layout.numel, device="cuda")
    want, m = p * torch.tensor(1.0 - 0.1 * 0.5), torch.zeros_like(u)
    ops.orthogonal_step_(p, u.clone(), m, layout, lr=0.1, weight_decay=0.5, steps=steps, eps=eps)
    assert torch.equal(p[:1200], want[:1200]) and torch.equal(p[2400:], want[2400:]) and torch.isfinite(p).all()


def test_epsilon_is_a_size():
    layout = ops.MatrixLayout([(4, 100)], "cuda")
    u = torch.ones(400, device="cuda")
    for eps in (-1e-7, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            ops.orthogonalize(u, layout, eps=eps)
        with pytest.raises(ValueError, match="eps"):
            ops.orthogonal_step_(u.clone(), u.clone(), u.clone(), layout, lr=0.1, eps=eps)
