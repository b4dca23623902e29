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
