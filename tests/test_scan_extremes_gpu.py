"""selective_scan where a step of no time, a state of zeros or a missing skip meets an infinity."""
import pytest
import torch

from oracle import sequence_oracle as so
from test_sequence_gpu import DTYPES, IDS, fd, scan_inputs  # noqa: F401

pytestmark = pytest.mark.gpu
SEQUENCES = ("u", "delta", "z", "B", "C")


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


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("s", [4, 16, 64])
def test_an_infinite_input_without_a_skip(fd, s, dtype):  # noqa: F811
    """Without D nothing but the states meets u: an infinite one makes them, and the outputs from there on, infinite."""
    g = torch.Generator().manual_seed(s)
    v = scan_inputs(g, 2, 40, 24, s, 1, dtype)
    v["B"], v["C"], v["D"] = v["B"].abs() + 0.5, v["C"].abs() + 0.5, None
    v["A"] = v["A"] * 0.01
    v["u"][1, 7, 3] = float("inf")
    v["z"] = v["z"].abs() + 0.5
    y = fd.selective_scan(**v, delta_softplus=True)
    bad = torch.zeros(2, 40, 24, dtype=torch.bool)
    bad[1, 7:, 3] = True
    assert torch.equal(torch.isinf(y).cpu(), bad) and not torch.isnan(y).any()
    state = torch.zeros(2, 24, s, device="cuda")
    token = {k: (t[:, 7] if k in SEQUENCES else t) for k, t in v.items()}
    step = fd.selective_scan_step(**token, state=state, delta_softplus=True)
    assert torch.equal(torch.isinf(step).cpu(), bad[:, 7]) and not torch.isnan(step).any()
