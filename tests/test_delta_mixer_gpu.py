"""The delta mixer: prompts against the definition in 64 bits, tokens against prompts, captured steps.

Tolerances as for the state space mixer: products of 3 x TF32 (relative error below 1e-5 of their terms' sizes) into a norm of 24 or more
channels; 1e-3 holds with a margin."""
import pytest
import torch

from oracle import delta_oracle as do
from oracle import sequence_oracle as so

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mixer(native_lib):
    from flagdnn_b200.state_space import DeltaMixer

    assert torch.cuda.is_available()
    return DeltaMixer(96, heads=4, key_heads=2, keys=32, values=24, dtype=torch.float32, seed=3)


def oracle(m, x, lengths=None):
    """The mixer's formulas in 64 bits: outputs and the two states."""
    n, length, _ = x.shape
    d = lambda t: t.double().cpu()  # noqa: E731
    both = d(x) @ d(m.w_in)
    v, conv = so.causal_conv1d(both[..., :m.mixed], m.w_conv, m.b_conv, "silu", None, lengths)
    keys = m.key_heads * m.keys
    q, k, v = v[..., :keys].unflatten(2, (m.key_heads, -1)), v[..., keys:2 * keys].unflatten(2, (m.key_heads, -1)), v[..., 2 * keys:].unflatten(2, (m.heads, -1))
    r = do.gated_delta_rule(q, k, v, both[..., m.mixed:m.mixed + m.heads], both[..., m.mixed + m.heads:], m.A, m.delta_bias, True, True, True,
                            lengths=lengths)
    z = so.group_norm(r.y.reshape(n * length, -1), m.heads, m.w_norm, m.b_norm)[0]
    return (z @ d(m.w_out)).view(n, length, -1) + d(x), conv, r.state


def test_prompts(mixer):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 90, 96, generator=g).cuda()
    lengths = torch.tensor([90, 0, 70], dtype=torch.int32).cuda()
    out, state = mixer.forward(x, lengths=lengths)
    want, conv, scan = oracle(mixer, x, lengths.tolist())
    torch.testing.assert_close(out[0].double().cpu(), want[0], rtol=1e-3, atol=1e-3)
    torch.testing.assert_close(out[2, :70].double().cpu(), want[2, :70], rtol=1e-3, atol=1e-3)
    torch.testing.assert_close(state.conv.double().cpu(), conv, rtol=1e-3, atol=1e-3)
    torch.testing.assert_close(state.scan.double().cpu(), scan, rtol=1e-3, atol=1e-3)


def test_tokens_continue_prompts_at_their_slots(mixer):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 80, 96, generator=g).cuda()
    whole, end = mixer.forward(x)
    _, behind = mixer.forward(x[:, :75])
    cache, slots = mixer.new_state(5), torch.tensor([4, 1], dtype=torch.int32).cuda()
    cache.put(slots, behind)
    for t in range(75, 80):
        out = mixer.step(x[:, t], cache, slots)
        torch.testing.assert_close(out, whole[:, t], rtol=1e-3, atol=1e-3)
    torch.testing.assert_close(cache.scan[slots.long()], end.scan, rtol=1e-3, atol=1e-3)
    torch.testing.assert_close(cache.conv[slots.long()], end.conv, rtol=1e-3, atol=1e-3)
    assert not cache.scan[[0, 2, 3]].any() and not cache.conv[[0, 2, 3]].any()
    second, _ = mixer.forward(x[:, 75:], state=behind)
    torch.testing.assert_close(second, whole[:, 75:], rtol=1e-3, atol=1e-3)
    # prompts that continue the first slots of a larger cache
    larger = mixer.new_state(4)
    larger.put(torch.tensor([0, 1]).cuda(), behind)
    torch.testing.assert_close(mixer.forward(x[:, 75:], state=larger)[0], second, rtol=0, atol=0)


def test_captured_prompts_and_steps(native_lib):
    from flagdnn_b200.state_space import DeltaMixer

    m = DeltaMixer(128, heads=4, key_heads=2, keys=64, values=64, dtype=torch.bfloat16, seed=5)
    g = torch.Generator().manual_seed(2)
    prompt, x = torch.randn(4, 100, 128, generator=g).bfloat16().cuda(), torch.randn(4, 128, generator=g).bfloat16().cuda()
    cache = m.new_state(4)
    want = [m.step(x, cache).clone() for _ in range(3)]
    first = m.forward(prompt)[0].clone()
    cache.conv.zero_(), cache.scan.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.step(x, cache)
        whole = m.forward(prompt)[0]
    cache.conv.zero_(), cache.scan.zero_()
    for ref in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(whole, first)


def test_rows_do_not_meet(native_lib):
    """A row's outputs do not depend on its batch; idle rows leave the cache alone."""
    from flagdnn_b200.state_space import DeltaMixer

    m = DeltaMixer(64, heads=2, key_heads=2, keys=16, values=16, dtype=torch.float16, seed=6)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(5, 64, generator=g).half().cuda()
    cache, alone = m.new_state(6), m.new_state(1)
    cache.scan.normal_(generator=torch.Generator("cuda").manual_seed(1))
    alone.scan.copy_(cache.scan[3:4])
    before = cache.scan.clone()
    slots = torch.tensor([5, -1, 3, 6, 0], dtype=torch.int32).cuda()
    out = m.step(x, cache, slots)
    assert torch.equal(out[2:3], m.step(x[2:3], alone))
    assert torch.equal(cache.scan[3:4], alone.scan) and torch.equal(cache.scan[[1, 2, 4]], before[[1, 2, 4]])
