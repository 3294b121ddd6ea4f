"""Group norm and the state space operators through the native host path and without it: the same bits; calls that it leaves to
Python; and that it is what runs."""
import pytest
import torch

from flagdnn_b200 import conv_host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fd(native_lib):
    import flagdnn_b200

    assert torch.cuda.is_available() and conv_host.native_host()
    return flagdnn_b200


def calls(fd, dtype):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    x, tok = r(3, 32, 6, 5).contiguous(memory_format=torch.channels_last), r(7, 64)
    seq, w, b = r(2, 19, 64), r(64, 4), r(64)
    lens = torch.tensor([19, 4], dtype=torch.int32).cuda()
    A, D = -torch.rand(64, 16, generator=g).cuda(), torch.randn(64, generator=g).cuda()
    B, C = r(2, 19, 16), r(2, 19, 2, 16)
    C1 = C[:, :, 0]
    slots = torch.tensor([3, 0], dtype=torch.int32).cuda()
    stats = fd.group_norm(x, 4, return_stats=True)[1:]
    conv_state, state = r(4, 3, 64), torch.randn(4, 64, 16, generator=g).cuda()

    def steps():
        cs, st = conv_state.clone(), state.clone()
        v = fd.causal_conv1d_step(seq[:, 0], cs, w, b, "silu", slots)
        y = fd.selective_scan_step(v, seq[:, 1], A, B[:, 0], C1[:, 0], st, D, seq[:, 2], D, True, slots)
        return v, y, cs, st

    return [
        lambda: fd.group_norm(x, 4, b[:32], w[:32, 0], activation="gelu"),          # a weight that is not dense: Python makes it
        lambda: fd.group_norm(x, 4, b[:32], None, 1e-3, "silu", True),
        lambda: fd.group_norm(tok, 8, b, b),
        lambda: fd.group_norm_backward(x, x, *stats, 4, b[:32], b[:32], "silu"),
        lambda: fd.causal_conv1d(seq, w, b, "silu", seq[:, :3].contiguous(), lens, True),
        lambda: fd.causal_conv1d(seq, w, initial_state=seq[:, :3]),                 # a state that is not dense
        lambda: fd.selective_scan(seq, seq, A, B, C1, D, seq, D, True, state[:2], lens, True),
        lambda: fd.selective_scan(seq, seq.abs(), A, B[:, :, None].expand(2, 19, 2, 16), C),
        steps,
    ]


def flat(v):
    return [v] if isinstance(v, torch.Tensor) else [t for t in v if t is not None]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "f16", "f32"])
def test_both_host_paths_give_the_same(fd, dtype, monkeypatch):
    native = [flat(c()) for c in calls(fd, dtype)]
    monkeypatch.setattr(conv_host, "_fast", False)
    python = [flat(c()) for c in calls(fd, dtype)]
    for a, b in zip(native, python):
        assert len(a) == len(b)
        for p, q in zip(a, b):
            assert p.dtype == q.dtype and p.stride() == q.stride() and torch.equal(p, q)


def test_the_native_path_takes_plain_calls(fd):
    fast = conv_host.native_host()
    x = torch.randn(2, 16, 4, 4, device="cuda")
    assert isinstance(fast.group_norm(x, 4, None, None, 1e-5, 0, False), torch.Tensor)
    assert fast.group_norm(x, 5, None, None, 1e-5, 0, False) is None               # Python raises
    assert fast.group_norm(x.cpu(), 4, None, None, 1e-5, 0, False) is None
    assert fast.group_norm(x.double(), 4, None, None, 1e-5, 0, False) is None
    leaf = x.clone().requires_grad_()
    assert fast.group_norm(leaf, 4, None, None, 1e-5, 0, False) is None            # Python differentiates
    with torch.no_grad():
        assert isinstance(fast.group_norm(leaf, 4, None, None, 1e-5, 0, False), torch.Tensor)
    seq, w = torch.randn(2, 5, 16, device="cuda"), torch.randn(16, 4, device="cuda")
    assert isinstance(fast.causal_conv1d(seq, w, None, 0, None, None, False), torch.Tensor)
    assert fast.causal_conv1d(seq, w[:8], None, 0, None, None, False) is None
    assert fast.causal_conv1d_step(seq[:, 0], seq[:, :3], w, None, 0, None) is None  # a cache that is not dense
    assert fast.selective_scan(seq, seq, w, seq, seq, None, None, None, False, None, None, False) is None
    assert fast.selective_scan_step(1, seq, w, seq, seq, None, None, None, None, False, None) is None
    status = fast.group_norm(x, 4, None, None, -1.0, 0, False)
    assert isinstance(status, int) and status != 0
