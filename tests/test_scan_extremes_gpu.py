"""selective_scan where a step of no time, or a state of zeros, meets an infinity."""
import pytest
import torch

from oracle import sequence_oracle as so
from test_sequence_gpu import fd, scan_inputs  # noqa: F401

pytestmark = pytest.mark.gpu


def near(got, want, tol):
    """Within tol of itself and of one; a NaN is not."""
    got = got.double().cpu()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol * (want.abs() + 1))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, {int(torch.isnan(got).sum())} NaN"


@pytest.mark.parametrize("s", [5, 16, 64])
@pytest.mark.parametrize("l,c,lengths", [(5, 40, None), (70, 12, [70, 0]), (2500, 40, [2500, 700])])
def test_states_that_forget_at_once(fd, l, c, lengths, s):  # noqa: F811
    """A rate of minus infinity: a state is what the newest token put there, and what lies past a row's end leaves it alone.
    Tolerances: as for the other prompts."""
    g = torch.Generator().manual_seed(l)
    n = 1 if lengths is None else len(lengths)
    v = scan_inputs(g, n, l, c, s, 1, torch.float32)
    v["A"][:, 2] = float("-inf")
    v["A"][3] = float("-inf")
    before = torch.randn(n, c, s, generator=g).cuda()
    lens = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want, final = so.selective_scan(v["u"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], v["delta_bias"], True, before, lengths)
    y, got = fd.selective_scan(**v, delta_softplus=True, initial_state=before, lengths=lens, return_final_state=True)
    tol = max(2e-4, l * 2.0 ** -21)
    near(got, final, tol)
    near(y, want, tol * s ** 0.5)


def test_states_of_zeros_before_growing_ones(fd):  # noqa: F811
    """A rate above zero over a piece of a long row: e^(A sum dt) is no number, and zero states stay zero all the same."""
    l, c, s = 4000, 40, 16
    u, delta = torch.zeros(1, l, c, device="cuda"), torch.ones(1, l, c, device="cuda")
    a, bc = torch.ones(c, s, device="cuda"), torch.ones(1, l, s, device="cuda")
    u[:, -2:] = 1.0
    y, final = fd.selective_scan(u, delta, a, bc, bc, return_final_state=True)
    want, end = so.selective_scan(u, delta, a, bc[:, :, None], bc[:, :, None])
    near(final, end, 2e-5)
    near(y, want, 2e-5 * s ** 0.5)
