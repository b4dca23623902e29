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


def _ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda:0")


def _cache(pages=8192):
    """A cache whose even pages are live, all of one sequence."""
    import dfccl_amd
    refcounts, lengths = (torch.zeros(n, dtype=torch.int32, device="cuda:0") for n in (pages, 3))
    tables = torch.full((3, pages), -1, dtype=torch.int32, device="cuda:0")
    refcounts[::2] = 1
    tables[0, :pages // 2] = torch.arange(0, pages, 2, dtype=torch.int32, device="cuda:0")
    lengths[:1].fill_(4 * (pages // 2))
    return dfccl_amd.PageCache([torch.zeros(pages, 64, dtype=torch.uint8, device="cuda:0")], 4, refcounts, tables, lengths)


@pytest.mark.parametrize("named", [True, False])
def test_a_page_caches_first_call_on_another_stream_waits_for_its_making(named):
    s, warm = torch.cuda.Stream(), _cache()
    warm.compact(stream=s)
    torch.cuda.synchronize()
    behind = _busy()
    cache = _cache()
    if named:
        cache.compact(stream=s)
    else:
        with torch.cuda.stream(s):
            cache.compact()
    s.synchronize()
    assert behind.query()
    assert cache.report.tolist() == [0, 2048, 4096] and bool((cache.refcounts[:4096] == 1).all())
    with torch.cuda.stream(s):
        cache.extend(_ints(1), _ints(5))
    cache.fork(_ints(0), _ints(2), stream=s)
    s.synchronize()
    assert cache.tables[1, :2].tolist() == [4096, 4097] and cache.lengths.tolist() == [16384, 5, 16384]


def test_a_dropped_page_caches_memory_is_not_given_away_while_a_call_uses_it():
    s, warm = torch.cuda.Stream(), _cache()
    warm.compact(stream=s)
    kept = _cache()
    refcounts, tables, lengths = kept.refcounts, kept.tables, kept.lengths
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        behind = _busy()
    kept.compact(stream=s)
    size, own = kept._workspace.numel(), (kept._workspace.data_ptr(), kept.report.data_ptr())
    del kept
    others = [torch.empty(n, dtype=torch.uint8, device="cuda:0") for n in (size, 12) for _ in range(4)]
    if not behind.query():
        assert not set(own) & {o.data_ptr() for o in others}
    for o in others:
        o.fill_(0xA5)
    s.synchronize()
    assert bool((refcounts[:4096] == 1).all()) and not bool(refcounts[4096:].any())
    assert torch.equal(tables[0, :4096].sort().values, torch.arange(4096, dtype=torch.int32, device="cuda:0"))
    assert lengths.tolist() == [16384, 0, 0]


def test_a_page_cache_captured_first_and_used_on_other_streams_afterwards():
    cache, s = _cache(), torch.cuda.Stream()
    seqs, lengths, child = _ints(1), _ints(0), _ints(2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.extend(seqs, lengths)
        cache.compact()
    for turn in range(3):
        lengths.fill_(8 * (turn + 1))
        graph.replay()
        s.wait_stream(torch.cuda.current_stream())
        cache.fork(seqs, child, stream=s)
        cache.free(child, stream=s)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.current_stream().synchronize()
        live = 4096 + 2 * (turn + 1)
        assert cache.lengths.tolist() == [16384, 8 * (turn + 1), 0] and int(cache.report[2]) == live
        assert bool((cache.refcounts[:live] == 1).all()) and not bool(cache.refcounts[live:].any())


def test_a_dropped_cache_of_emptys_making_keeps_its_bookkeeping_while_a_call_uses_it():
    import dfccl_amd
    s, pools = torch.cuda.Stream(), [torch.zeros(3000, 64, dtype=torch.uint8, device="cuda:0")]
    warm = dfccl_amd.PageCache.empty(pools, 4, 300, 700)
    one, many = _ints(0), _ints(*range(300))
    warm.extend(one, one, stream=s)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        behind = _busy()
    cache = dfccl_amd.PageCache.empty(pools, 4, 300, 700)
    sizes = [(t.numel(), t.data_ptr()) for t in (cache.refcounts, cache.tables, cache.lengths)]
    cache.free(many, stream=s)
    del cache
    others = [torch.empty(n, dtype=torch.int32, device="cuda:0") for n, _ in sizes for _ in range(4)]
    if not behind.query():
        assert not {at for _, at in sizes} & {o.data_ptr() for o in others}
    torch.cuda.synchronize()
