"""Page operations on lists as long as a launch's grid could not be: 2^24 requests and more."""
import pytest
import torch

import gpu_util

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(gpu_util.EMULATED, reason="size of a real GPU")]


def _range(*args):
    return torch.arange(*args, dtype=torch.int32, device="cuda:0")


def test_extend_and_fork_of_more_requests_than_a_grid_has_workgroups():
    import dfccl_amd
    n = (1 << 24) + 5
    pool = torch.zeros(n + 8, 4, dtype=torch.uint8, device="cuda:0")
    cache = dfccl_amd.PageCache.empty([pool], 2, 2 * n, 1)
    order, lengths = _range(n).flip(0).contiguous(), torch.full((n,), 2, dtype=torch.int32, device="cuda:0")
    lengths[-3:] = 1  # sequences 2, 1 and 0
    cache.extend(order, lengths)
    torch.cuda.synchronize()
    assert int(cache.report[0]) == 0
    assert torch.equal(cache.tables[order.long(), 0], _range(n)) and torch.equal(cache.lengths[order.long()], lengths)
    assert bool((cache.refcounts[:n] == 1).all()) and not bool(cache.refcounts[n:].any())
    pool[n - 3:n] = torch.tensor([[1], [2], [3]], dtype=torch.uint8, device="cuda:0")  # the pages of sequences 2, 1, 0
    parents, children = _range(n), _range(n, 2 * n)
    cache.fork(parents, children)
    torch.cuda.synchronize()
    assert int(cache.report[0]) == 0 and torch.equal(cache.lengths[:n], cache.lengths[n:])
    assert torch.equal(cache.tables[n + 3:, 0], cache.tables[3:n, 0])     # full pages are shared
    assert cache.tables[n:n + 3, 0].tolist() == [n, n + 1, n + 2]          # the three others are copied
    assert pool[n:n + 3, 0].tolist() == [3, 2, 1] and pool[n:n + 3].long().sum().item() == 24
    assert bool((cache.refcounts[:n - 3] == 2).all()) and cache.refcounts[n - 3:].tolist() == [1] * 6 + [0] * 5


def test_lists_and_sequences_up_to_the_last_that_an_integer_counts():
    import dfccl_amd
    most = (1 << 31) - 1
    pool = torch.arange(64, dtype=torch.uint8, device="cuda:0").view(64, 1)
    cache = dfccl_amd.PageCache.empty([pool], 1, most, 1)
    for seq, page in ((0, 40), (5, 41), (most - 1, 63)):
        cache.refcounts[page], cache.tables[seq, 0], cache.lengths[seq] = 1, page, 1
    cache.compact()
    torch.cuda.synchronize()
    assert cache.report[1:].tolist() == [3, 3] and pool[:3, 0].tolist() == [40, 41, 63]
    assert [int(cache.tables[seq, 0]) for seq in (0, 5, most - 1)] == [0, 1, 2]
    ended = torch.full((most,), -1, dtype=torch.int32, device="cuda:0")
    ended[0], ended[most - 1] = 5, most - 1
    cache.free(ended)
    torch.cuda.synchronize()
    assert cache.refcounts[:4].tolist() == [1, 0, 0, 0] and [int(cache.lengths[s]) for s in (0, 5, most - 1)] == [1, 0, 0]
    assert [int(cache.tables[seq, 0]) for seq in (0, 5, most - 1)] == [0, -1, -1]
