"""group_norm_backward on tensors that ask for a gradient: it has no derivative of its own."""
import pytest
import torch

from flagdnn_b200 import conv_host
from test_group_norm_gpu import fd, make, params  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
def test_second_derivatives_are_refused(fd, native, monkeypatch):  # noqa: F811
    if not native:
        monkeypatch.setattr(conv_host, "_fast", False)
    x, dy, (w, b) = make((2, 24, 6, 6), torch.float32, "cl"), make((2, 24, 6, 6), torch.float32, "cl", seed=2), params(24, torch.float32)
    _, mean, rstd = fd.group_norm(x, 4, w, b, return_stats=True)
    args = [dy, x, mean, rstd, 4, w, b, "silu"]
    want = fd.group_norm_backward(*args)
    for k in (0, 1, 2, 3, 5, 6):
        asks = list(args)
        asks[k] = args[k].clone().requires_grad_()
        with pytest.raises(NotImplementedError, match="computes no gradients"):
            fd.group_norm_backward(*asks)
        with torch.no_grad():
            assert all(torch.equal(p, q) and not p.requires_grad for p, q in zip(fd.group_norm_backward(*asks), want))
    # the differentiable entry point still differentiates once, and refuses a second time
    leaf = x.clone().requires_grad_()
    grad, = torch.autograd.grad(fd.group_norm(leaf, 4, w, b, activation="silu"), leaf, dy, create_graph=True)
    assert torch.equal(grad, want[0])
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad"):
        grad.sum().backward()
