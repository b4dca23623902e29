"""The row and page operators as a program uses them, next to the collectives and to each other: a vocabulary split over
ranks, whose lookups an all-reduce puts together and whose gradients need none; a cache that forks, ends, grows and is
handed from rank to rank while the tokens' rows are looked up and written into its pages."""
import numpy as np
import pytest
import torch

import gpu_util
import indexed_util as iu

pytestmark = pytest.mark.gpu


def _sync():
    torch.cuda.current_stream().synchronize()


def _dev(t):
    return t.to(gpu_util.DEVICE)


@pytest.mark.parametrize("ranks", [2, 4])
def test_vocabulary_split_over_ranks(ranks):
    """Every rank looks all tokens up in its own piece, an all-reduce sums the ranks' rows: exactly one of them is not
    zero, so the sum is the lookup in the whole table bit for bit. Backwards, every rank sums the gradients of all
    ranks' tokens into its piece: side by side the pieces are the gradient of the whole table."""
    import dfccl_amd
    from dfccl_amd.ring import VirtualRing
    g = torch.Generator().manual_seed(ranks)
    rows, width, tokens = 37, 40, 60
    vocab = rows * ranks - 3  # the last piece is shorter
    table = _dev(torch.randn(vocab, width, generator=g).bfloat16())
    ids = _dev(torch.randint(0, vocab, (tokens,), generator=g))
    pieces = [table[r * rows:(r + 1) * rows] for r in range(ranks)]
    parts = [torch.full((tokens, width), 9.0, dtype=torch.bfloat16, device=gpu_util.DEVICE) for _ in range(ranks)]
    sums = [torch.zeros_like(p) for p in parts]
    for r in range(ranks):
        dfccl_amd.embedding_lookup(pieces[r], ids, parts[r], scale=6.0, first_row=r * rows)
    whole = torch.empty_like(parts[0])
    dfccl_amd.embedding_lookup(table, ids, whole, scale=6.0)
    _sync()
    with VirtualRing(ranks) as ring:
        ring.prepare(0, "all_reduce", tokens * width, dfccl_amd.ncclBfloat16, dfccl_amd.ncclSum)
        ring.finalize()
        ring.run(0, parts, sums, timeout=60)
    for r in range(ranks):
        assert torch.equal(sums[r], whole)  # (x + 0 is x, also for the zeros: none of the parts holds -0)
    iu.check(whole, *iu.lookup(table, ids, 0, 6.0))

    grads = [_dev(torch.randn(tokens - 7 * r, width, generator=g)) for r in range(ranks)]
    batches = [_dev(torch.randint(0, vocab, (tokens - 7 * r,), generator=g)) for r in range(ranks)]
    got = torch.empty(vocab, width, device=gpu_util.DEVICE)
    for r in range(ranks):
        dfccl_amd.embedding_grad(grads, batches, got[r * rows:(r + 1) * rows], scale=0.5, first_row=r * rows)
    one = torch.empty_like(got)
    dfccl_amd.embedding_grad(grads, batches, one, scale=0.5)
    _sync()
    assert torch.equal(got, one)
    exact, before, _ = iu.grad(grads, batches, vocab, 0, 0.5, None)
    iu.check(got, exact, before)


def test_gradients_of_ranks_by_all_reduce_and_at_once():
    """Dense gradients per rank put together by an all-reduce, against all ranks' tokens in one call."""
    import dfccl_amd
    from dfccl_amd.ring import VirtualRing
    g = torch.Generator().manual_seed(8)
    ranks, vocab, width = 3, 50, 24
    grads = [_dev(torch.randn(40 + r, width, generator=g)) for r in range(ranks)]
    ids = [_dev(torch.randint(0, vocab, (40 + r,), generator=g)) for r in range(ranks)]
    own = [torch.empty(vocab, width, device=gpu_util.DEVICE) for _ in range(ranks)]
    sums = [torch.empty(vocab, width, device=gpu_util.DEVICE) for _ in range(ranks)]
    for r in range(ranks):
        dfccl_amd.embedding_grad(grads[r], ids[r], own[r])
    at_once = torch.empty(vocab, width, device=gpu_util.DEVICE)
    dfccl_amd.embedding_grad(grads, ids, at_once)
    _sync()
    with VirtualRing(ranks) as ring:
        ring.prepare(0, "all_reduce", vocab * width, dfccl_amd.ncclFloat32, dfccl_amd.ncclSum)
        ring.finalize()
        ring.run(0, own, sums, timeout=60)
    exact, before, count = iu.grad(grads, ids, vocab, 0, 1.0, None)
    iu.check(at_once, exact, before)
    for s in sums:  # the ranks' sums add up to `ranks` roundings more of what the bound counts once per token
        iu.check(s, exact, before + ranks * iu.U32 * (exact.abs() + before))


def test_a_cache_that_serves():
    """Sequences grow by looked-up rows written into their pages, branch, end, are compacted and handed to another
    rank's cache; at every step each sequence's pages hold exactly the rows of its own tokens."""
    import dfccl_amd
    rs = np.random.RandomState(4)
    width, page_tokens, pages, seqs, per_seq = 20, 4, 64, 12, 6
    table = _dev(torch.randn(100, width, generator=torch.Generator().manual_seed(1)).half())
    pools = [torch.zeros(pages, page_tokens, width, dtype=torch.float16, device=gpu_util.DEVICE) for _ in range(2)]
    cache = dfccl_amd.PageCache.empty(pools, page_tokens, seqs, per_seq)
    history = {q: [] for q in range(seqs)}

    def ints(values):
        return _dev(torch.tensor(list(values), dtype=torch.int32))

    def append(running):
        """One token for each running sequence: its page is taken, its row looked up, scaled by pool, written."""
        tokens = rs.randint(0, 100, len(running))
        cache.extend(ints(running), ints(len(history[q]) + 1 for q in running))
        rows = torch.empty(len(running), width, dtype=torch.float16, device=gpu_util.DEVICE)
        where = torch.tensor([len(history[q]) for q in running], device=gpu_util.DEVICE)
        for k, pool in enumerate(pools):
            dfccl_amd.embedding_lookup(table, _dev(torch.from_numpy(tokens)), rows, scale=float(k + 1))
            _sync()
            page = cache.tables[torch.tensor(running, device=gpu_util.DEVICE), where // page_tokens].long()
            pool[page, where % page_tokens] = rows
        for q, t in zip(running, tokens):
            history[q].append(int(t))

    def holds(c):
        _sync()
        for q, tokens in history.items():
            assert int(c.lengths[q]) == len(tokens)
            for k, pool in enumerate(c.pools):
                got = pool[c.tables[q, :-(-len(tokens) // page_tokens)].long()].reshape(-1, width)[:len(tokens)]
                assert torch.equal(got, (table[tokens].float() * (k + 1)).half()), (q, k)
        assert int(c.report[0]) == 0

    for _ in range(6):
        append([0, 1, 2])
    holds(cache)
    cache.fork(ints([0, 0, 1]), ints([5, 6, 7]))
    for p, c in ((0, 5), (0, 6), (1, 7)):
        history[c] = list(history[p])
    holds(cache)
    for _ in range(5):
        append([0, 5, 6, 7, 2])
    holds(cache)
    cache.free(ints([0, 1, 6]))
    for q in (0, 1, 6):
        history[q] = []
    cache.compact()
    holds(cache)
    live = int((cache.refcounts > 0).sum())
    assert not bool(cache.refcounts[live:].any())
    append([5, 7, 2, 9])
    # another rank's cache takes all of it over: contents page by page, bookkeeping as it is
    others = [torch.full_like(p, float("nan")) for p in pools]
    other = dfccl_amd.PageCache(others, page_tokens, cache.refcounts.clone(), cache.tables.clone(), cache.lengths.clone())
    _sync()
    used = torch.nonzero(cache.refcounts > 0)[:, 0].int()
    other.copy(used, used, source=cache)
    holds(other)
    cache.free(ints(range(seqs)))
    _sync()
    assert not bool(cache.refcounts.any()) and bool((cache.tables == -1).all())
