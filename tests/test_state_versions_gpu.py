"""States that the single-token operators update in place count as written: autograd sees a saved tensor that has changed."""
import pytest
import torch

from flagdnn_b200 import conv_host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fd(native_lib):
    import flagdnn_b200

    assert torch.cuda.is_available()
    return flagdnn_b200


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
def test_steps_move_their_states_version(fd, native, monkeypatch):
    if not native:
        monkeypatch.setattr(conv_host, "_fast", False)
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    x, taps, a, bc = r(2, 16), r(16, 4), -r(16, 8).abs(), r(2, 8)
    conv_state, state, other = r(2, 3, 16), r(2, 16, 8), r(2, 3, 16).requires_grad_()
    saved = (other * conv_state).sum()
    versions = conv_state._version, state._version
    fd.causal_conv1d_step(x, conv_state, taps)
    fd.selective_scan_step(x, x, a, bc, bc, state)
    assert (conv_state._version, state._version) == (versions[0] + 1, versions[1] + 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    # a cache made in inference mode keeps no count; it is taken inside and outside of it
    with torch.inference_mode():
        hidden, hidden_conv = torch.zeros(2, 16, 8, device="cuda"), torch.zeros(2, 3, 16, device="cuda")
        fd.selective_scan_step(x, x, a, bc, bc, hidden)
        fd.causal_conv1d_step(x, hidden_conv, taps)
    fd.selective_scan_step(x, x, a, bc, bc, hidden)
    fd.causal_conv1d_step(x, hidden_conv, taps)
    assert hidden.any() and hidden_conv.any()
