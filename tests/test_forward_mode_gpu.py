"""Tensors with tangents (forward-mode differentiation): the operators have no such derivative and say so."""
import pytest
import torch
from torch.autograd import forward_ad

from flagdnn_b200 import conv_host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fd(native_lib):
    import flagdnn_b200

    assert torch.cuda.is_available()
    return flagdnn_b200


@pytest.mark.parametrize("native", [True, False], ids=["native", "python"])
def test_tangents_are_refused(fd, native, monkeypatch):
    if not native:
        monkeypatch.setattr(conv_host, "_fast", False)
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    x, w = r(2, 16, 4, 4), r(16)
    _, mean, rstd = fd.group_norm(x, 4, w, w, return_stats=True)
    seq, taps, a, bc = r(2, 5, 16), r(16, 4), -r(16, 8).abs(), r(2, 5, 8)
    conv_state, state = r(2, 3, 16), r(2, 16, 8)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (
            lambda: fd.group_norm(dual(x), 4),
            lambda: fd.group_norm(x, 4, dual(w), w),
            lambda: fd.group_norm(x, 4, w, dual(w), return_stats=True),
            lambda: fd.group_norm_backward(dual(x), x, mean, rstd, 4, w, w),
            lambda: fd.group_norm_backward(x, x, mean, rstd, 4, dual(w), w),
            lambda: fd.causal_conv1d(dual(seq), taps),
            lambda: fd.causal_conv1d(seq, taps, initial_state=dual(conv_state)),
            lambda: fd.causal_conv1d_step(seq[:, 0], conv_state, dual(taps)),
            lambda: fd.selective_scan(seq, dual(seq), a, bc, bc),
            lambda: fd.selective_scan(seq, seq, a, bc, bc, w, initial_state=dual(state)),
            lambda: fd.selective_scan_step(seq[:, 0], seq[:, 0], a, bc[:, 0], bc[:, 0], state, dual(w)),
        ):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        plain = fd.group_norm(x, 4, w, w)                 # tensors without one go on as ever
        primal = forward_ad.unpack_dual(dual(x)).primal
        assert torch.equal(fd.group_norm(primal, 4, w, w), plain)
    assert torch.equal(fd.group_norm(x, 4, w, w), plain)
