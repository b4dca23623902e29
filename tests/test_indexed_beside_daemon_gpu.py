"""The row and page operators while the daemon is resident: all-reduces are in flight on every rank when lookups,
gradients and page operations are launched on the current stream, and both sides come out as they do alone."""
import numpy as np
import pytest
import torch

import datagen
import dfccl_oracle as orc
import gpu_util
import indexed_util as iu
from gpu_util import geom_of, to_gpu, to_np

pytestmark = pytest.mark.gpu
SMALL = gpu_util.EMULATED


def test_rows_and_pages_while_collectives_are_in_flight(monkeypatch):
    import dfccl_amd
    from dfccl_amd.ring import VirtualRing
    monkeypatch.setenv("DFCCL_DAEMON_MAX_MS", "20000")
    ranks, colls, count, rounds = 4, 3, 5003 if SMALL else 4_000_037, 1 if SMALL else 3
    tokens, vocab, width = (90, 40, 24) if SMALL else (3500, 900, 264)  # (one workgroup sorts so many, with 57 KiB of LDS)
    dev = gpu_util.DEVICE
    gen = torch.Generator().manual_seed(7)
    table, grad = (torch.randn(n, width, generator=gen).bfloat16().to(dev) for n in (vocab, tokens))
    ids = [torch.randint(0, vocab, (tokens,), generator=gen).to(dev) for _ in range(rounds)]
    outs = [torch.zeros(tokens, width, dtype=torch.bfloat16, device=dev) for _ in range(rounds)]
    sums = [torch.zeros(vocab, width, device=dev) for _ in range(rounds)]
    contents = np.random.RandomState(1).randint(0, 256, (60, 48)).astype(np.uint8)
    cache = dfccl_amd.PageCache.empty([torch.from_numpy(contents.copy()).to(dev)], 4, 12, 8)
    books = iu.Books([contents], 4, 12, 8)
    lists = [torch.tensor(x, dtype=torch.int32, device=dev) for x in ([0, 1, 2, 3], [9, 32, 2, 17], [0, 1, 3], [4, 5, 6], [1, 2])]
    workspace = torch.zeros(dfccl_amd.embedding_grad_workspace([tokens], vocab, width), dtype=torch.uint8, device=dev)
    with VirtualRing(ranks) as ring:
        for c in range(colls):
            ring.prepare(c, "all_reduce", count, dfccl_amd.ncclFloat32, dfccl_amd.ncclSum)
        ring.finalize()
        sends_np = [datagen.make(orc.F32, 50 + r, count) for r in range(ranks)]
        sends = [to_gpu(orc.F32, s) for s in sends_np]
        recvs = [[torch.zeros_like(s) for s in sends] for _ in range(colls)]
        torch.cuda.current_stream().synchronize()
        for k in range(rounds):
            for r in range(ranks):
                for c in range(colls):
                    ring.submit(r, c, sends[r], recvs[c][r])
            dfccl_amd.embedding_lookup(table, ids[k], outs[k], scale=2.0)
            dfccl_amd.embedding_grad(grad, ids[k], sums[k], scale=0.5, workspace=workspace)
            if k == 0:
                cache.extend(lists[0], lists[1])
                cache.fork(lists[2], lists[3])
                cache.free(lists[4])
                cache.compact()
            ring.wait([(r, c) for r in range(ranks) for c in range(colls)], timeout=40)
        torch.cuda.current_stream().synchronize()
        want = orc.all_reduce(orc.F32, orc.SUM, geom_of(ring, 0), sends_np)
        for c in range(colls):
            for r in range(ranks):
                assert np.array_equal(to_np(orc.F32, recvs[c][r]), want[r]), (c, r)
    for k in range(rounds):
        iu.check(outs[k], *iu.lookup(table, ids[k], 0, 2.0))
        exact, before, _ = iu.grad([grad], [ids[k]], vocab, 0, 0.5, None)
        iu.check(sums[k], exact, before)
    books.extend([0, 1, 2, 3], [9, 32, 2, 17])
    books.fork([0, 1, 3], [4, 5, 6])
    books.free([1, 2])
    books.compact()
    assert np.array_equal(cache.refcounts.cpu().numpy(), books.refs) and np.array_equal(cache.tables.cpu().numpy(), books.tables)
    assert np.array_equal(cache.lengths.cpu().numpy(), books.lengths)
    assert np.array_equal(cache.pools[0].cpu().numpy(), books.contents[0])
