"""group_norm at values whose squares come near the ends of fp32, and over long runs of pixels behind an outlier."""
import pytest
import torch

from oracle import sequence_oracle as so
from test_group_norm_gpu import fd, make  # noqa: F401

pytestmark = pytest.mark.gpu


def near(got, want, rtol=2e-5, atol=2e-5):
    got = got.double().cpu()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= rtol * want.abs() + atol)   # (a NaN is not near)
    worst = ((got - want).abs() / want.abs().clamp_min(1e-300)).max()
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, {int(torch.isnan(got).sum())} NaN, worst {float(worst):.3g} of its size"


def test_an_outlier_whose_squares_are_near_the_largest_number(fd):  # noqa: F811
    """8e18 among small values: its square, 6.4e37, is a number, and so is the variance; the square of five values' distances
    from it, added up, is not.  All of it is fp32 arithmetic on numbers, at the tolerances of other values."""
    x = make((160, 8, 24, 24), torch.float32, "cl")
    x[:, 0, 0, 0] = 8e18
    x[:, 4, 5, 3] = -8e18
    want, mean, rstd = so.group_norm(x, 2)
    y, got_mean, got_rstd = fd.group_norm(x, 2, return_stats=True)
    near(got_rstd, rstd, rtol=5e-5, atol=0.0)
    near(got_mean, mean)
    near(y, want)


def test_a_long_run_behind_an_outlier(fd):  # noqa: F811
    """A thread of the two-launch form sums distances from a first value D away from the others.  Over 32 values each of the
    two sums is rounded 31 times, to 16 D (16 D^2) on average: 1000 and 500 times 2^-24 of D^2, which is a part of the group's
    squared deviations; 9e-5 of the variance and half of it of its root, at most.  (A run of a thousand values: a thousand times that.)"""
    x = torch.randn(1, 4096, 4096, 4, device="cuda", generator=torch.Generator("cuda").manual_seed(0)).permute(0, 3, 1, 2)
    x[:, 0, 0, 0] = 1e5
    all_of = x.double()
    mean = all_of.mean()
    rstd = ((all_of - mean).square().mean() + 1e-5).rsqrt()
    _, got_mean, got_rstd = fd.group_norm(x, 1, return_stats=True)
    near(got_mean[0, 0], mean.cpu())
    near(got_rstd[0, 0], rstd.cpu(), rtol=4.5e-5, atol=0.0)


@pytest.mark.parametrize("shape,dtype", [((10, 1, 900, 900), torch.bfloat16), ((10, 3, 590, 600), torch.float32)], ids=["bf16", "f32"])
def test_a_long_run_that_one_launch_holds(fd, shape, dtype):  # noqa: F811
    """The same for vectors of one value, of which a block holds hundreds for each of its threads."""
    n, c, h, w = shape
    x = torch.randn(n, h, w, c, device="cuda", generator=torch.Generator("cuda").manual_seed(0)).to(dtype).permute(0, 3, 1, 2)
    x[:, :, 0, 0] = 1e5
    rows = x.double().flatten(2)
    mean = rows.mean(2)
    rstd = ((rows - mean[..., None]).square().mean(2) + 1e-5).rsqrt()
    _, got_mean, got_rstd = fd.group_norm(x, c, return_stats=True)
    near(got_mean, mean.cpu())
    near(got_rstd, rstd.cpu(), rtol=4.5e-5, atol=0.0)
