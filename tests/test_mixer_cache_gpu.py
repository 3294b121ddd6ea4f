"""StateSpaceMixer over prompts that continue a cache with more slots than prompts: row n at slot n."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_prompts_continue_the_first_slots_of_a_larger_cache(native_lib):
    from flagdnn_b200.state_space import StateSpaceMixer

    mixer = StateSpaceMixer(96, 192, states=16, rank=24, norm_groups=6, dtype=torch.float32, seed=3)
    x = torch.randn(2, 20, 96, generator=torch.Generator().manual_seed(1)).cuda()
    _, behind = mixer.forward(x[:, :15])
    want, end = mixer.forward(x[:, 15:], state=behind)
    cache = mixer.new_state(5)
    cache.put(torch.tensor([0, 1], dtype=torch.int32).cuda(), behind)
    got, after = mixer.forward(x[:, 15:], state=cache)
    assert torch.equal(got, want) and torch.equal(after.conv, end.conv) and torch.equal(after.scan, end.scan)
    with pytest.raises(RuntimeError, match="initial_state must have shape"):
        mixer.forward(x[:, 15:], state=mixer.new_state(1))
