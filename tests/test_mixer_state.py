"""MixerState.put: rows into their slots of a cache; a slot outside of it marks an idle row, as for the steps."""
import pytest
import torch

from flagdnn_b200.state_space import MixerState


def states(rows, seed):
    g = torch.Generator().manual_seed(seed)
    return MixerState(torch.randn(rows, 3, 8, generator=g).to(torch.bfloat16), torch.randn(rows, 8, 4, generator=g))


@pytest.mark.parametrize("slots", [[4, 1, 0], [-1, 2, 0], [2, -1, 5], [7, -3, 4], [-1, -1, 9], [3, 5, 2 ** 31 - 1]])
def test_idle_rows_write_nothing(slots):
    cache, rows = states(5, 0), states(3, 1)
    conv, scan = cache.conv.clone(), cache.scan.clone()
    for i, slot in enumerate(slots):
        if 0 <= slot < 5:
            conv[slot], scan[slot] = rows.conv[i], rows.scan[i]
    cache.put(torch.tensor(slots, dtype=torch.int32), rows)
    assert torch.equal(cache.conv, conv) and torch.equal(cache.scan, scan)


def test_nothing_to_put():
    cache, none = states(5, 0), states(0, 1)
    conv = cache.conv.clone()
    cache.put(torch.empty(0, dtype=torch.int32), none)
    assert torch.equal(cache.conv, conv)
    empty, rows = states(0, 0), states(2, 1)
    empty.put(torch.tensor([0, -1], dtype=torch.int32), rows)
    assert empty.conv.shape[0] == 0


def test_rows_that_do_not_go_with_the_slots():
    cache = states(5, 0)
    conv = cache.conv.clone()
    for slots in (torch.tensor([0, 1, 2, 3]), torch.tensor([0, 1]), torch.tensor([[0, 1, 2]])):
        with pytest.raises(RuntimeError, match="put"):
            cache.put(slots.int(), states(3, 1))
    assert torch.equal(cache.conv, conv)
    with pytest.raises(RuntimeError, match="put"):
        MixerState(cache.conv, cache.scan[:4]).put(torch.tensor([0, 1, 4]), states(3, 1))
    one = states(1, 2)                        # one row for several slots
    cache.put(torch.tensor([4, -1, 2], dtype=torch.int32), one)
    conv[[4, 2]] = one.conv
    assert torch.equal(cache.conv, conv)
