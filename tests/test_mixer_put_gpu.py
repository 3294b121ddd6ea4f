"""MixerState.put on the GPU: idle rows, and within a captured graph (it does not wait for the device)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slots", [[4, 1, 0], [-1, 2, 0], [2, -1, 7], [-1, 5, -9]])
def test_rows_into_their_slots(slots):
    from flagdnn_b200.state_space import MixerState

    g = torch.Generator().manual_seed(0)
    make = lambda n: MixerState(torch.randn(n, 3, 8, generator=g).cuda(), torch.randn(n, 8, 4, generator=g).cuda())  # noqa: E731
    cache, rows, where = make(5), make(3), torch.tensor(slots, dtype=torch.int32).cuda()
    start, conv, scan = MixerState(cache.conv.clone(), cache.scan.clone()), cache.conv.clone(), cache.scan.clone()
    for i, slot in enumerate(slots):
        if 0 <= slot < 5:
            conv[slot], scan[slot] = rows.conv[i], rows.scan[i]
    cache.put(where, rows)
    assert torch.equal(cache.conv, conv) and torch.equal(cache.scan, scan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.put(where, rows)
    cache.conv.copy_(start.conv)
    cache.scan.copy_(start.scan)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(cache.conv, conv) and torch.equal(cache.scan, scan)
