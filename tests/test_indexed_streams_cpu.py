"""Streams and memory of the row and page operators' Python layer, without a GPU: streams, events and the library are
stand-ins that write down what is asked of them, buffers lie in host memory and no kernel runs."""
import ctypes

import pytest
import torch

import dfccl_amd
from dfccl_amd import api, indexed


class Stream:
    def __init__(self, handle, device="cpu"):
        self.cuda_stream, self.device, self.waited = handle, torch.device(device), []

    def wait_event(self, event):
        self.waited.append(event)


class Machine:
    """The current stream, the workspaces taken (size, stream that was current), and the library's calls (name, arguments)."""

    def __init__(self):
        self.stream, self.taken, self.calls = Stream(1), [], []

    def __getattr__(self, name):  # an entry point of the library
        def call(*args):
            self.calls.append((name, args))
            if name.endswith("Workspace"):
                args[-1]._obj.value = 4096
            return 0
        return call


@pytest.fixture
def machine(monkeypatch):
    m = Machine()

    class Current:  # torch.cuda.stream
        def __init__(self, stream):
            self.stream = stream

        def __enter__(self):
            self.before, m.stream = m.stream, self.stream

        def __exit__(self, *exc):
            m.stream = self.before
            return False
    empty = torch.empty

    def noted(*args, **kw):
        m.taken.append((args[0], m.stream))
        return empty(*args, **kw)
    monkeypatch.setattr(torch, "empty", noted)
    monkeypatch.setattr(torch.cuda, "stream", Current)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: m.stream)
    monkeypatch.setattr(api, "_dev_ptr", lambda t: ctypes.c_void_p(t.data_ptr()))
    monkeypatch.setattr(indexed._lib, "load", lambda: m)
    return m


# A block of the current stream's pool may have been freed by a tensor whose kernels are still queued there, and
# another stream does not wait for them: a workspace has to come from the pool of the stream that it is used on.
def test_the_gradients_workspace_comes_from_the_pool_of_the_stream_that_it_runs_on(machine):
    g, ids, out = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), torch.zeros(5, 8)
    other = Stream(2)
    dfccl_amd.embedding_grad(g, ids, out, stream=other)
    dfccl_amd.embedding_grad(g, ids, out)
    assert machine.taken == [(4096, other), (4096, machine.stream)]
    launched = [args for name, args in machine.calls if name == "dfcclEmbeddingGrad"]
    assert [args[-1] for args in launched] == [2, 1]
    dfccl_amd.embedding_grad(g, ids, out, workspace=torch.zeros(4096, dtype=torch.uint8), stream=other)
    assert len(machine.taken) == 2 and machine.stream.cuda_stream == 1


class Buffer:
    """A tensor on the GPU, as far as PageCache looks at one."""

    def __init__(self, machine, *shape, dtype=torch.int32):
        self.machine, self.shape, self.dtype, self.device, self.is_cuda = machine, shape, dtype, torch.device("cuda:0"), True
        self.nbytes, self.recorded = 4 * self.numel(), []

    def numel(self):
        return torch.Size(self.shape).numel()

    def dim(self):
        return len(self.shape)

    def data_ptr(self):
        return 1 << 20  # never followed

    def is_contiguous(self):
        return True

    def record_stream(self, stream):
        self.recorded.append(stream)


class Gpu(Machine):
    def __init__(self):
        super().__init__()
        self.stream, self.capturing = Stream(1, "cuda:0"), False
        self.stream.record_event = lambda: "behind what the constructor needs"


@pytest.fixture
def gpu(machine, monkeypatch):
    m = Gpu()
    monkeypatch.setattr(indexed._lib, "load", lambda: m)
    monkeypatch.setattr(torch, "empty", lambda n, **kw: Buffer(m, n))
    monkeypatch.setattr(torch, "zeros", lambda n, **kw: Buffer(m, n))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: m.stream)
    monkeypatch.setattr(indexed, "_raw_stream", lambda index: m.stream.cuda_stream)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: m.capturing)
    return m


def _cache(m):
    return dfccl_amd.PageCache([Buffer(m, 6, 8)], 4, Buffer(m, 6), Buffer(m, 3, 2), Buffer(m, 3))


def _calls(m, cache, first=0, **on):
    """The three calls that use the cache's own memory, beginning with any of them; returns the handles of their streams."""
    one, handles = Buffer(m, 1), []
    calls = [lambda: cache.extend(one, one, **on), lambda: cache.fork(one, one, **on), lambda: cache.compact(**on)]
    for k in range(3):
        del m.calls[:]
        calls[(first + k) % 3]()
        handles.append(m.calls[0][1][-1])
    return handles


# The workspace and the report come from the pool of the stream that is current in the constructor. Another stream has to
# wait for what that one still does with them, and they may not return to the pool before the other is through with them.
@pytest.mark.parametrize("first", range(3))
def test_a_page_caches_own_memory_is_shared_with_the_streams_that_it_is_used_on(gpu, first):
    cache, other = _cache(gpu), Stream(2, "cuda:0")
    assert _calls(gpu, cache, first, stream=other) == [2] * 3
    assert other.waited == ["behind what the constructor needs"]
    assert cache._workspace.recorded == [other] and cache.report.recorded == [other]
    third = Stream(3, "cuda:0")  # not named, but current
    gpu.stream, made_on = third, gpu.stream
    assert _calls(gpu, cache, first) == [3] * 3
    assert third.waited == ["behind what the constructor needs"] and cache.report.recorded == [other, third]
    gpu.stream = made_on
    assert _calls(gpu, cache, first) == [1] * 3
    assert made_on.waited == [] and cache.report.recorded == [other, third]


def test_the_bookkeeping_that_empty_makes_is_the_caches_own_memory(gpu, monkeypatch):
    monkeypatch.setattr(torch, "full", lambda shape, *a, **kw: Buffer(gpu, *shape))
    other, one = Stream(2, "cuda:0"), Buffer(gpu, 1)
    cache = dfccl_amd.PageCache.empty([Buffer(gpu, 6, 8)], 4, 3, 2)
    cache.free(one, stream=other)
    assert other.waited == ["behind what the constructor needs"]
    own = (cache.refcounts, cache.tables, cache.lengths, cache.report, cache._workspace)
    assert [b.recorded for b in own] == [[other]] * 5
    passed = _cache(gpu)  # (the caller's bookkeeping is the caller's to keep)
    passed.free(one, stream=other)
    assert [b.recorded for b in (passed.refcounts, passed.tables, passed.lengths)] == [[]] * 3


def test_a_copy_uses_none_of_it_and_waits_for_nothing(gpu):
    cache, other, one = _cache(gpu), Stream(2, "cuda:0"), Buffer(gpu, 1)
    cache.copy(one, one, stream=other)
    assert gpu.calls[-1][1][-1] == 2
    assert other.waited == [] and cache._workspace.recorded == [] and cache.report.recorded == []


def test_a_captured_call_waits_for_no_event_from_before_the_capture(gpu):
    cache, other = _cache(gpu), Stream(2, "cuda:0")
    gpu.capturing = True
    _calls(gpu, cache, stream=other)
    assert other.waited == [] and set(cache._workspace.recorded) == {other}
    gpu.capturing = False
    _calls(gpu, cache, stream=other)
    assert other.waited == ["behind what the constructor needs"]
    gpu.capturing = True
    made_in_a_capture, fourth = _cache(gpu), Stream(4, "cuda:0")  # its memory is the graph's
    gpu.capturing = False
    _calls(gpu, made_in_a_capture, stream=fourth)
    assert fourth.waited == [] and made_in_a_capture.report.recorded == [fourth]


# ctypes drops the bits of an integer that its C type does not hold: what would arrive as another number is refused
@pytest.mark.parametrize("number", [1 << 63, -(1 << 63) - 1, 1 << 64, (1 << 64) + 3])
def test_ids_that_do_not_fit_64_bits_are_refused(machine, number):
    table, ids, out = torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 8)
    with pytest.raises(ValueError, match="first_row.* 64 bits"):
        dfccl_amd.embedding_lookup(table, ids, out, first_row=number)
    with pytest.raises(ValueError, match="first_row.* 64 bits"):
        dfccl_amd.embedding_grad(out, ids, table, first_row=number)
    with pytest.raises(ValueError, match="padding_id.* 64 bits"):
        dfccl_amd.embedding_grad(out, ids, table, padding_id=number)
    with pytest.raises(ValueError, match="64 bits"):
        dfccl_amd.embedding_grad_workspace([3], number, 8)
    assert not [name for name, _ in machine.calls if not name.endswith("Workspace")]
    for fits in ((1 << 63) - 1, -(1 << 63)):
        dfccl_amd.embedding_lookup(table, ids, out, first_row=fits)
        dfccl_amd.embedding_grad(out, ids, table, first_row=fits, padding_id=fits)
    assert len([name for name, _ in machine.calls if not name.endswith("Workspace")]) == 4


@pytest.mark.parametrize("number", [1 << 31, 1 << 32, (1 << 32) + 4, -(1 << 31) - 1])
def test_sizes_of_a_page_cache_that_do_not_fit_32_bits_are_refused(gpu, number):
    def make(pages=6, page_tokens=4, sequences=3, per_seq=2):
        return dfccl_amd.PageCache([Buffer(gpu, pages, 8)], page_tokens, Buffer(gpu, pages), Buffer(gpu, sequences, per_seq),
                                   Buffer(gpu, sequences))
    with pytest.raises(ValueError, match="32 bits"):
        make(page_tokens=number)
    if number > 0:
        for size in ("pages", "sequences", "per_seq"):
            with pytest.raises(ValueError, match="32 bits"):
                make(**{size: number})
        cache, many = make(), Buffer(gpu, number)
        del gpu.calls[:]
        for call in (lambda: cache.free(many), lambda: cache.copy(many, many), lambda: cache.extend(many, many),
                     lambda: cache.fork(many, many)):
            with pytest.raises(ValueError, match="32 bits"):
                call()
        assert not gpu.calls


def test_a_stream_of_another_device_is_refused(gpu):
    elsewhere, one = Stream(2, "cuda:1"), Buffer(gpu, 1)
    cache = _cache(gpu)
    del gpu.calls[:]
    for call in (lambda: cache.copy(one, one, stream=elsewhere), lambda: cache.extend(one, one, stream=elsewhere),
                 lambda: cache.fork(one, one, stream=elsewhere), lambda: cache.free(one, stream=elsewhere),
                 lambda: cache.compact(stream=elsewhere)):
        with pytest.raises(ValueError, match="stream on cuda:1"):
            call()
    assert not gpu.calls and not elsewhere.waited and not cache._workspace.recorded


def test_a_lookup_and_a_gradient_on_a_stream_of_another_device_are_refused(machine):
    table, ids, out = torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 8)
    for call in (lambda s: dfccl_amd.embedding_lookup(table, ids, out, stream=s),
                 lambda s: dfccl_amd.embedding_grad(out, ids, table, stream=s)):
        with pytest.raises(ValueError, match="stream on cuda:1"):
            call(Stream(2, "cuda:1"))
    assert not machine.taken and not [name for name, _ in machine.calls if not name.endswith("Workspace")]
