"""The convolution's other activations, and gradients of group_norm whose dy lies otherwise than x."""
import pytest
import torch

from oracle import sequence_oracle as so
from test_group_norm_gpu import DTYPES, ROUND, fd, make, params  # noqa: F401

pytestmark = pytest.mark.gpu
IDS = ["bf16", "f16", "f32"]


def near(got, want, dtype, atol, rtol=2e-5):
    got = got.double().cpu()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= (1.02 * ROUND[dtype] + rtol) * want.abs() + atol)   # (a NaN is not near)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, {int(torch.isnan(got).sum())} NaN"


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh"])
def test_activations_of_the_convolution(fd, act, dtype):  # noqa: F811
    """Tolerance: fp32 sums of four products and the activation of a value of their size, 2e-5 (1 + |y|), and one rounding."""
    g = torch.Generator().manual_seed(4)
    for c in (64, 33):
        x, w, b = (torch.randn(*s, generator=g).to(dtype).cuda() for s in ((3, 41, c), (c, 4), (c,)))
        lengths = [41, 0, 7]
        want, final = so.causal_conv1d(x, w, b, act, None, lengths)
        y, got = fd.causal_conv1d(x, w, b, act, lengths=torch.tensor(lengths, dtype=torch.int32).cuda(), return_final_state=True)
        near(y, want, dtype, 2e-5)
        assert torch.equal(got.double().cpu(), final)
        state = x[:, :3].contiguous()
        step = fd.causal_conv1d_step(x[:, 3], state, w, b, act)
        near(step, so.causal_conv1d(x[:, 3:4], w, b, act, x[:, :3])[0][:, 0], dtype, 2e-5)


LAYOUTS = [("cl", "nchw"), ("nchw", "cl"), ("cl", "crop"), ("odd", "cl"), ("crop", "nchw"), ("cl", "spread")]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("layouts", LAYOUTS, ids=["-".join(k) for k in LAYOUTS])
@pytest.mark.parametrize("shape,groups", [((2, 64, 30, 31), 8), ((3, 45, 9, 7), 3)])
def test_gradients_of_dy_in_another_layout(fd, shape, groups, layouts, dtype):  # noqa: F811
    """Tolerances: those of the gradients in one layout."""
    x = make(shape, dtype, layouts[0])
    dy = make(shape[:2] + (1, 1), dtype, "cl", seed=7).expand(shape) if layouts[1] == "spread" else make(shape, dtype, layouts[1], seed=7)
    w, b = params(shape[1], dtype)
    _, mean, rstd = fd.group_norm(x, groups, w, b, return_stats=True)
    dx, dw, db = fd.group_norm_backward(dy, x, mean, rstd, groups, w, b, activation="gelu")
    want = so.group_norm_grad(dy, x, groups, w, b, 1e-5, "gelu")
    scale, terms = float(rstd.max().clamp_min(1.0)), (x.numel() // shape[1]) ** 0.5
    near(dx, want[0], dtype, 1e-4 * scale)
    near(dw, want[1], dtype, 8e-5 * terms)
    near(db, want[2], dtype, 8e-5 * terms)
