"""gated_delta_rule where its inputs reach their ends: tokens that forget all.

Tolerances as in test_delta_rule_gpu.py."""
import pytest
import torch

from oracle import delta_oracle as do
from test_delta_rule_gpu import fd, inputs, near  # noqa: F401
from test_sequence_gpu import DTYPES, IDS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("resets", [1, 2, 8, 16, 32, 41])
@pytest.mark.parametrize("forget", [-float("inf"), -1e30, -3e4, -250.0])
def test_several_tokens_of_a_chunk_forget_all(fd, dtype, resets, forget):  # noqa: F811
    """Packed documents begin within a chunk, the last of them in its middle: what the tokens behind it write is kept as they say."""
    g = torch.Generator().manual_seed(resets)
    v, options = inputs(g, 1, 150, 1, 2, 64, 48, dtype, False, True)
    at = [40 - i * 40 // max(1, resets - 1) for i in range(resets)]
    assert len(set(at)) == resets and max(at) == 40
    for chunk in (0, 64):
        v["delta"][:, [chunk + i for i in at]] = forget
    before = torch.randn(1, 2, 48, 64, generator=g).cuda()
    for length in (64, 150):
        part = {name: t[:, :length] for name, t in v.items()}
        want = do.gated_delta_rule(**part, **options, initial_state=before)
        y, state = fd.gated_delta_rule(**part, **options, initial_state=before, return_final_state=True)
        near(state, want.state, want.state_size, torch.float32)
        near(y, want.y, want.y_size, dtype)
