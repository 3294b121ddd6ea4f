"""group_norm of images with one channel a group, whose slabs hold several groups: between one cluster and two launches."""
import pytest
import torch

from oracle import sequence_oracle as so
from test_group_norm_gpu import DTYPES, FP32, ROUND, fd, make, params  # noqa: F401

pytestmark = pytest.mark.gpu

# (shape, layout): few large images, channels that are no whole vectors or lie at an odd address
IMAGES = [((1, 3, 112, 112), "cl"), ((1, 3, 128, 128), "cl"), ((1, 4, 100, 100), "cl"), ((2, 12, 96, 96), "cl"), ((1, 6, 100, 100), "cl"),
          ((1, 33, 100, 100), "cl"), ((1, 8, 100, 100), "odd"), ((2, 16, 95, 101), "cl"), ((1, 5, 81, 127), "slice")]


def near(got, want, dtype, atol=FP32, rtol=FP32):
    got = got.double().cpu()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= (1.02 * ROUND[dtype] + rtol) * want.abs() + atol)   # (a NaN is not near)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, {int(torch.isnan(got).sum())} NaN"


@pytest.mark.parametrize("dtype", DTYPES, ids=["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", IMAGES, ids=["x".join(map(str, s)) + k for s, k in IMAGES])
def test_one_channel_a_group(fd, case, dtype):  # noqa: F811
    """Tolerances: as for the other sizes of group_norm."""
    shape, layout = case
    x, dy, (w, b) = make(shape, dtype, layout), make(shape, dtype, "cl", seed=7), params(shape[1], dtype)
    want, mean, rstd = so.group_norm(x, shape[1], w, b, 1e-5, "silu")
    y, got_mean, got_rstd = fd.group_norm(x, shape[1], w, b, 1e-5, activation="silu", return_stats=True)
    near(got_mean, mean, torch.float32)
    near(got_rstd, rstd, torch.float32, rtol=5e-5)
    near(y, want, dtype)
    dx, dw, db = fd.group_norm_backward(dy, x, got_mean, got_rstd, shape[1], w, b, activation="silu")
    want = so.group_norm_grad(dy, x, shape[1], w, b, 1e-5, "silu")
    scale = float(rstd.max().clamp_min(1.0))
    near(dx, want[0], dtype, atol=FP32 * scale * 5)
    terms = (x.numel() // shape[1]) ** 0.5
    near(dw, want[1], dtype, atol=FP32 * terms * 4)
    near(db, want[2], dtype, atol=FP32 * terms * 4)
