"""The state space mixer: prompts against the definition in 64 bits, tokens against prompts, captured steps."""
import pytest
import torch

from oracle import sequence_oracle as so

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mixer(native_lib):
    from flagdnn_b200.state_space import StateSpaceMixer

    assert torch.cuda.is_available()
    return StateSpaceMixer(96, 192, states=16, rank=24, norm_groups=6, dtype=torch.float32, seed=3)


def oracle(m, x, lengths=None):
    """The mixer's formulas in 64 bits: outputs and the two states."""
    n, length, _ = x.shape
    d = lambda t: t.double().cpu()  # noqa: E731
    both = (d(x).reshape(n * length, -1) @ d(m.w_in)).view(n, length, -1)
    v, conv = so.causal_conv1d(both[..., :m.inner], m.w_conv, m.b_conv, "silu", None, lengths)
    steps = v @ d(m.w_steps)
    delta = steps[..., :m.rank] @ d(m.w_delta)
    B, C = steps[..., m.rank:m.rank + m.states, None].transpose(2, 3), steps[..., m.rank + m.states:, None].transpose(2, 3)
    y, scan = so.selective_scan(v, delta, m.A, B, C, m.D, both[..., m.inner:], m.delta_bias, True, None, lengths)
    z = so.group_norm(y.reshape(n * length, -1), m.norm_groups, m.w_norm, m.b_norm)[0]
    return (z @ d(m.w_out)).view(n, length, -1), conv, scan


def test_prompts(mixer):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 50, 96, generator=g).cuda()
    lengths = torch.tensor([50, 0, 23], dtype=torch.int32).cuda()
    out, state = mixer.forward(x, lengths=lengths)
    want, conv, scan = oracle(mixer, x, lengths.tolist())
    # products of 3xTF32 (relative error below 1e-5 of their terms' sizes) into a norm of 32 channels: 1e-3 holds with a margin
    torch.testing.assert_close(out[0].double().cpu(), want[0], rtol=1e-3, atol=1e-3)
    torch.testing.assert_close(out[2, :23].double().cpu(), want[2, :23], rtol=1e-3, atol=1e-3)
    torch.testing.assert_close(state.conv.double().cpu(), conv, rtol=1e-3, atol=1e-3)
    torch.testing.assert_close(state.scan.double().cpu(), scan, rtol=1e-3, atol=1e-3)


def test_tokens_continue_prompts_at_their_slots(mixer):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 20, 96, generator=g).cuda()
    whole, end = mixer.forward(x)
    _, behind = mixer.forward(x[:, :15])
    cache, slots = mixer.new_state(5), torch.tensor([4, 1], dtype=torch.int32).cuda()
    cache.put(slots, behind)
    for t in range(15, 20):
        out = mixer.step(x[:, t], cache, slots)
        torch.testing.assert_close(out, whole[:, t], rtol=1e-3, atol=1e-3)
    torch.testing.assert_close(cache.scan[slots.long()], end.scan, rtol=1e-3, atol=1e-3)
    torch.testing.assert_close(cache.conv[slots.long()], end.conv, rtol=1e-3, atol=1e-3)
    assert not cache.scan[[0, 2, 3]].any() and not cache.conv[[0, 2, 3]].any()
    second, _ = mixer.forward(x[:, 15:], state=behind)
    torch.testing.assert_close(second, whole[:, 15:], rtol=1e-3, atol=1e-3)


def test_a_captured_step(native_lib):
    from flagdnn_b200.state_space import StateSpaceMixer

    m = StateSpaceMixer(128, 256, dtype=torch.bfloat16, seed=5)
    x = torch.randn(4, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    cache = m.new_state(4)
    want = [m.step(x, cache).clone() for _ in range(3)]
    cache.conv.zero_(), cache.scan.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.step(x, cache)
    cache.conv.zero_(), cache.scan.zero_()
    for ref in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)
