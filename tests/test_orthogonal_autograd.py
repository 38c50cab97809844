"""In-place writes of the orthogonalised update are seen by autograd: a graph that saved the old values refuses."""
import pytest
import torch

from k2q import ops

pytestmark = pytest.mark.gpu


def buffers():
    return [torch.randn(300, device="cuda") for _ in range(3)], ops.MatrixLayout([(3, 100)], "cuda")


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("zero_grad", [False, True])
def test_step_is_seen(which, zero_grad):
    """Parameters and momentum are written always, gradients where they are zeroed."""
    b, layout = buffers()
    w = torch.ones(300, device="cuda", requires_grad=True)
    loss = (w * b[which]).sum()
    ops.orthogonal_step_(*b, layout, lr=0.1, zero_grad=zero_grad)
    if which == 1 and not zero_grad:
        loss.backward()
        assert torch.equal(w.grad, b[1])
    else:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


@pytest.mark.parametrize("inplace", [False, True])
def test_out_is_seen(inplace):
    (u, out, _), layout = buffers()
    w = torch.ones(300, device="cuda", requires_grad=True)
    target = u if inplace else out
    loss = (w * target).sum()
    ops.orthogonalize(u, layout, out=target)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_parameters_of_the_fused_step_are_seen():
    from k2q import parallel, trainer
    p = torch.nn.Parameter(torch.randn(4, 50, device="cuda"))
    opt = trainer.FusedOrthogonalStep(parallel.AdapterGradBuckets([[p]]))
    x = torch.ones(4, 50, device="cuda", requires_grad=True)
    loss = (x * p).sum()
    loss.backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors():
    """They have no version to advance."""
    with torch.inference_mode():
        b, layout = buffers()
        ops.orthogonal_step_(*b, layout, lr=0.1, zero_grad=True)
        ops.orthogonalize(b[0], layout, out=b[2])
    assert (b[1] == 0).all() and torch.isfinite(b[2]).all()
