"""The row and page operators on streams of their own while the stream that is current is busy: which memory they take,
when they give it back, and what they wait for."""
import pytest
import torch

import gpu_util
import indexed_util as iu

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(gpu_util.EMULATED, reason="streams of a real GPU")]


def _busy(ms=40):
    """Work for the current stream that takes it about so long; returns the event behind it."""
    x = torch.empty(1 << 28, device="cuda:0")  # 1 GiB, written in some 0.16 ms
    for _ in range(6 * ms):
        x.fill_(1.0)
    return torch.cuda.current_stream().record_event()


def test_a_gradient_takes_no_memory_that_the_current_stream_still_uses(monkeypatch):
    import dfccl_amd
    gen = torch.Generator().manual_seed(1)
    g, ids = torch.randn(3000, 64, generator=gen).cuda(), torch.randint(0, 300, (3000,), generator=gen).cuda()
    out = torch.zeros(300, 64, device="cuda:0")
    need = dfccl_amd.embedding_grad_workspace([3000], 300, 64)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    _busy()
    freed = torch.empty(need, dtype=torch.uint8, device="cuda:0")  # as large as the workspace, written late, freed at once
    freed.fill_(0xA5)
    at = freed.data_ptr()
    del freed
    taken, empty = [], torch.empty

    def noted(*args, **kw):
        t = empty(*args, **kw)
        taken.append(t.data_ptr())
        return t
    with monkeypatch.context() as m:
        m.setattr(torch, "empty", noted)
        dfccl_amd.embedding_grad(g, ids, out, stream=s)
    assert len(taken) == 1 and not at <= taken[0] < at + need and not taken[0] <= at < taken[0] + need
    s.synchronize()
    exact, before, _ = iu.grad([g], [ids], 300, 0, 1.0, None)
    iu.check(out, exact, before)
    torch.cuda.synchronize()
