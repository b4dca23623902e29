"""The page operations of a cache (dfcclPages* through the C ABI) against their definition, one request after another on
the host (indexed_util.Books): contents and bookkeeping have to be equal bit for bit after every call."""
import numpy as np
import pytest
import torch

import gpu_util
import indexed_util as iu

pytestmark = pytest.mark.gpu
big_only = pytest.mark.skipif(gpu_util.EMULATED, reason="size or feature of a real GPU")


def _sync():
    torch.cuda.current_stream().synchronize()


def _ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device=gpu_util.DEVICE)


class Both:
    """A cache on the GPU and its definition on the host, driven together and compared after every call."""

    def __init__(self, pages, page_tokens, sequences, per_seq, page_bytes=(24,), seed=0):
        import dfccl_amd
        rs = np.random.RandomState(seed)
        contents = [rs.randint(0, 256, (pages, page_bytes[0])).astype(np.uint8) for _ in page_bytes]
        pools = [torch.from_numpy(c.copy()).to(gpu_util.DEVICE) for c in contents]
        self.cache = dfccl_amd.PageCache.empty(pools, page_tokens, sequences, per_seq)
        self.books = iu.Books(contents, page_tokens, sequences, per_seq)

    def same(self, what):
        _sync()
        c, b = self.cache, self.books
        assert np.array_equal(c.refcounts.cpu().numpy(), b.refs), what
        assert np.array_equal(c.tables.cpu().numpy(), b.tables), what
        assert np.array_equal(c.lengths.cpu().numpy(), b.lengths), what
        for k, (got, want) in enumerate(zip(c.pools, b.contents)):
            assert np.array_equal(got.cpu().numpy(), want), f"{what}: pool {k}"

    def extend(self, seqs, lengths):
        self.cache.extend(_ints(seqs), _ints(lengths))
        self.books.extend(seqs, lengths)
        self.same(f"extend {seqs} {lengths}")
        assert int(self.cache.report[0]) == self.books.refused

    def fork(self, parents, children):
        self.cache.fork(_ints(parents), _ints(children))
        self.books.fork(parents, children)
        self.same(f"fork {parents} {children}")
        assert int(self.cache.report[0]) == self.books.refused

    def free(self, seqs):
        self.cache.free(_ints(seqs))
        self.books.free(seqs)
        self.same(f"free {seqs}")

    def compact(self):
        self.cache.compact()
        self.books.compact()
        self.same("compact")
        assert self.cache.report[1:].tolist() == [self.books.moved, self.books.live]


@pytest.mark.parametrize("page_tokens", [1, 3, 16])
@pytest.mark.parametrize("seed", range(4))
def test_random_calls_one_after_another(page_tokens, seed):
    # few pages, so that they run out; sequences out of range, listed twice, in use, empty and too long among the requests
    rs = np.random.RandomState(1000 + 10 * seed + page_tokens)
    both = Both(pages=int(rs.randint(5, 60)), page_tokens=page_tokens, sequences=9, per_seq=7, page_bytes=(40, 40), seed=seed)
    for _ in range(6 if gpu_util.EMULATED else 60):
        n = int(rs.randint(0, 10))
        seqs = rs.randint(-1, 10, n).tolist()
        op = rs.choice(["extend", "extend", "fork", "free", "compact"])
        if op == "extend":
            now = [int(both.books.lengths[q]) if 0 <= q < 9 else 0 for q in seqs]
            both.extend(seqs, [int(x + rs.randint(-1, 3 * page_tokens + 1)) for x in now])
        elif op == "fork":
            both.fork(seqs, rs.randint(-1, 10, n).tolist())
        elif op == "free":
            both.free(seqs[:3])
        else:
            both.compact()


def test_extend_at_the_edges_of_pages_and_of_the_cache():
    both = Both(pages=8, page_tokens=4, sequences=5, per_seq=4)
    both.extend([0, 1, 2, 3, 4], [0, 1, 4, 5, 16])   # 0 + 1 + 1 + 2 + 4 pages: all of them
    both.extend([0, 1, 2], [1, 4, 4])                 # no page left; grows within its page; stays as it is
    both.extend([1], [3])                             # shorter than it is
    both.extend([4], [17])                            # longer than its table row
    both.extend([2, 2], [4, 8])                       # listed twice
    both.extend([-1, 5, 1 << 30], [1, 1, 1])
    both.extend([], [])
    both.free([3])
    both.extend([0, 1, 2], [1, 8, 9])                 # two pages left: the first two requests take them
    both.extend([3], [-1])


def test_requests_behind_one_that_found_no_pages_need_none_or_are_refused():
    both = Both(pages=4, page_tokens=2, sequences=6, per_seq=8)
    both.extend([0, 1], [1, 0])
    both.extend([2, 3, 0, 4], [9, 2, 2, 1])           # 5 pages of 3; then 1; then none; then 1
    both.free([0])
    both.extend([1, 3], [8, 0])


def test_fork_shares_full_pages_and_copies_the_last():
    both = Both(pages=20, page_tokens=4, sequences=10, per_seq=4, page_bytes=(33, 33, 33))
    both.extend([0, 1, 2], [4, 7, 1])
    both.fork([0, 1, 2, 5], [3, 4, 6, 7])             # full last page, one not full, a single token, an empty parent
    both.extend([1, 4], [9, 8])                       # parent and child go on by themselves
    both.fork([1, 1, 1], [8, 9, 5])                   # three children of one parent
    both.free([1])
    both.free([8, 4, 3, 0])


def test_fork_refusals():
    both = Both(pages=6, page_tokens=4, sequences=8, per_seq=4)
    both.extend([0, 1], [6, 4])
    both.fork([0, 0, 0], [1, 0, 2])                   # a child in use, itself, an empty one
    both.fork([0, 1, 1], [3, 3, 9])                   # a child listed twice, one out of range
    both.fork([-1, 8], [4, 5])
    both.fork([0, 0, 1], [4, 5, 6])                   # one page left for two; the third needs none
    both.fork([4], [7])
    both.fork([3, 7], [7, 2])                         # a parent that is a child of the same call is forked as it was


def test_free_of_the_same_sequence_twice_and_of_none():
    both = Both(pages=12, page_tokens=2, sequences=6, per_seq=5)
    both.extend([0, 1, 2], [9, 4, 3])
    both.fork([0, 0], [4, 5])
    both.free([0, 0, 0, 3, -1, 6])
    both.free([])
    both.free([4, 5, 1, 2, 1, 2])
    assert not both.cache.refcounts.any()


def test_compact_full_empty_and_already_compact():
    both = Both(pages=9, page_tokens=1, sequences=4, per_seq=9, page_bytes=(17,))
    both.compact()
    both.extend([0, 1, 2], [3, 3, 3])
    both.compact()
    both.free([0])
    both.compact()
    both.compact()
    both.fork([1], [3])
    both.free([1])
    both.compact()
    both.free([2, 3])
    both.compact()


@pytest.mark.parametrize("pages", [127, 512, 513, 2047, 2100, 5000, 16384, 16385, 40000])
def test_compact_and_extend_over_several_rounds_of_the_scan(pages):
    if gpu_util.EMULATED and pages > 2100:
        pytest.skip("too many emulated threads")
    rs = np.random.RandomState(pages)
    both = Both(pages=pages, page_tokens=1, sequences=40, per_seq=pages // 30, page_bytes=(4,), seed=1)
    every = list(range(40))
    both.extend(every, [pages // 40] * 40)
    both.free(rs.permutation(40)[:20].tolist())
    both.extend(every, rs.randint(0, pages // 30 + 1, 40).tolist())
    both.free(rs.permutation(40)[:15].tolist())
    both.compact()


# page sizes around a wave's 1024, 2048 and 4096 bytes and the 16 bytes of a load; pools around the 64 of a launch
@pytest.mark.parametrize("page_bytes,npools", [(1, 1), (15, 3), (16, 2), (17, 2), (1023, 1), (1024, 1), (1025, 1), (2047, 1),
                                               (2048, 1), (2049, 1), (4095, 1), (4096, 2), (4097, 2), (8195, 1),
                                               (8, 64), (6, 65), (32, 131)])
def test_contents_of_odd_pages_and_many_pools(page_bytes, npools):
    import dfccl_amd
    both = Both(pages=7, page_tokens=4, sequences=4, per_seq=3, page_bytes=(page_bytes,) * npools, seed=page_bytes)
    both.extend([0, 1], [6, 2])
    both.fork([0], [2])
    both.free([0])
    both.compact()
    # copy: from another cache, within one, and pairs out of range left out
    rs = np.random.RandomState(3)
    others = [torch.from_numpy(rs.randint(0, 256, (5, page_bytes)).astype(np.uint8)).to(gpu_util.DEVICE) for _ in range(npools)]
    other = dfccl_amd.PageCache.empty(others, 4, 1, 1)
    src, dst = [4, 0, 0, 5, -1, 2, 3], [6, 0, 5, 1, 2, 7, -1]
    both.cache.copy(_ints(src), _ints(dst), source=other)
    for k, pool in enumerate(both.books.contents):
        for s, d in ((4, 6), (0, 0), (0, 5)):
            pool[d] = others[k][s].cpu().numpy()
    both.same("copy from another cache")
    both.cache.copy(_ints([6, 5]), _ints([2, 3]))
    for pool in both.books.contents:
        pool[2], pool[3] = pool[6], pool[5]
    both.same("copy within")
    both.cache.copy(_ints([]), _ints([]))
    both.same("copy of nothing")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.int8])
def test_pools_of_any_type_keep_every_bit(dtype):
    import dfccl_amd
    bits = torch.from_numpy(np.random.RandomState(9).randint(0, 256, (6, 5, 3, 8)).astype(np.uint8)).to(gpu_util.DEVICE)
    pool = bits.view(dtype)
    cache = dfccl_amd.PageCache.empty([pool], 5, 2, 2)
    cache.copy(_ints([0, 1]), _ints([4, 5]))
    _sync()
    assert torch.equal(bits[4], bits[0]) and torch.equal(bits[5], bits[1])


def test_entries_out_of_range_in_the_tables_are_not_followed():
    both = Both(pages=6, page_tokens=2, sequences=4, per_seq=3)
    both.extend([0, 1], [5, 4])
    c = both.cache
    c.tables[0] = _ints([-7, 6, 1 << 30])
    c.fork(_ints([0]), _ints([2]))
    c.free(_ints([0, 2]))
    c.compact()
    _sync()
    assert c.lengths.tolist() == [0, 4, 0, 0]
    # lengths that no table row can hold
    c.lengths[1] = 100
    c.fork(_ints([1]), _ints([3]))
    c.extend(_ints([1]), _ints([101]))
    _sync()
    assert int(c.report[0]) == 1 and c.lengths.tolist() == [0, 100, 0, 0]
    c.lengths[0] = -3
    c.free(_ints([0]))
    c.fork(_ints([0]), _ints([3]))
    _sync()
    assert int(c.lengths[3]) == 0
    c.compact()
    c.free(_ints([1]))
    _sync()
    assert int(c.lengths[1]) == 0


@big_only
def test_a_large_cache_over_several_rounds_and_workgroups():
    rs = np.random.RandomState(5)
    both = Both(pages=150_000, page_tokens=2, sequences=1500, per_seq=150, page_bytes=(16,), seed=2)
    every = list(range(1500))
    both.extend(every, rs.randint(0, 200, 1500).tolist())
    gone = rs.permutation(1500)[:700].tolist()
    both.free(gone)
    both.fork(sorted(set(every) - set(gone))[:600], gone[:600])
    both.extend(gone[600:], rs.randint(0, 300, 100).tolist())
    both.free(rs.permutation(1500)[:600].tolist())
    both.compact()


@big_only
def test_offsets_that_pass_32_bits():
    import dfccl_amd
    page = 1 << 20
    pools = [torch.zeros(5000, page, dtype=torch.uint8, device="cuda:0") for _ in range(2)]  # 5.2 GB each
    for k, p in enumerate(pools):
        p[4999], p[4096], p[1] = 10 + k, 20 + k, 30 + k
    cache = dfccl_amd.PageCache.empty(pools, 1, 3, 2500)
    cache.copy(_ints([4999, 4096, 1]), _ints([0, 4097, 4998]))
    _sync()
    for k, p in enumerate(pools):
        assert bool((p[0] == 10 + k).all()) and bool((p[4097] == 20 + k).all()) and bool((p[4998] == 30 + k).all())
        assert not bool(p[2:4096].any()) and not bool(p[4098:4998].any())
    cache.extend(_ints([0, 1]), _ints([2500, 2500]))
    cache.free(_ints([0]))
    cache.compact()  # pages 2500 .. 4999 move to 0 .. 2499
    _sync()
    assert cache.report[1:].tolist() == [2500, 2500]
    for k, p in enumerate(pools):
        assert bool((p[2499] == 10 + k).all()) and bool((p[1596] == 20 + k).all()) and bool((p[2498] == 30 + k).all())


@big_only
def test_captured_and_replayed():
    both = Both(pages=400, page_tokens=4, sequences=40, per_seq=20, page_bytes=(1024, 1024))
    seqs, lengths = torch.arange(20, dtype=torch.int32, device="cuda:0"), torch.zeros(20, dtype=torch.int32, device="cuda:0")
    parents, children = _ints([0, 1, 2]), _ints([30, 31, 32])
    ended = _ints([30, 31, 5])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both.cache.extend(seqs, lengths)
        both.cache.fork(parents, children)
        both.cache.free(ended)
        both.cache.compact()
    both.same("captured, not run")
    rs = np.random.RandomState(11)
    for k in range(5):
        now = [int(both.books.lengths[q]) + int(rs.randint(0, 6)) for q in range(20)]
        lengths.copy_(_ints(now))
        children.copy_(_ints([30, 31, 32 + k]))
        graph.replay()
        both.books.extend(list(range(20)), now)
        both.books.fork([0, 1, 2], [30, 31, 32 + k])
        both.books.free([30, 31, 5])
        both.books.compact()
        both.same(f"replay {k}")
        both.extend([33 + k], [3])  # the program's own calls between the replays
        both.free([33 + k])


@big_only
def test_on_a_stream_of_its_own():
    both = Both(pages=300, page_tokens=4, sequences=30, per_seq=20, page_bytes=(64,))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    lists = [_ints(range(20)), _ints([9 + k for k in range(20)]), _ints([3, 4]), _ints([25, 26]), _ints([3, 7])]
    s.wait_stream(torch.cuda.current_stream())
    both.cache.extend(lists[0], lists[1], stream=s)
    both.cache.fork(lists[2], lists[3], stream=s)
    both.cache.free(lists[4], stream=s)
    both.cache.compact(stream=s)
    s.synchronize()
    both.books.extend(list(range(20)), [9 + k for k in range(20)])
    both.books.fork([3, 4], [25, 26])
    both.books.free([3, 7])
    both.books.compact()
    both.same("own stream")


def test_workspace_of_exactly_the_size_asked_for():
    both = Both(pages=90, page_tokens=2, sequences=11, per_seq=9)
    c = both.cache
    n = c._workspace.numel()
    buf = torch.full((n + 512,), 0xA5, dtype=torch.uint8, device=gpu_util.DEVICE)
    c._workspace, c._struct.workspace = buf, buf.data_ptr() + 256
    both.extend(list(range(11)), [2 * k for k in range(11)])
    both.free([4, 5])
    both.fork([1, 2], [4, 5])
    both.free([10, 9])
    both.compact()
    assert bool((buf[:256] == 0xA5).all()) and bool((buf[256 + n:] == 0xA5).all())


def test_refusals():
    import dfccl_amd
    d = gpu_util.DEVICE
    pools = [torch.zeros(6, 8, device=d) for _ in range(2)]
    cache = dfccl_amd.PageCache.empty(pools, 4, 3, 2)
    with pytest.raises(ValueError, match="agree in pages"):
        dfccl_amd.PageCache.empty([pools[0], torch.zeros(6, 9, device=d)], 4, 3, 2)
    with pytest.raises(TypeError, match="int32"):
        dfccl_amd.PageCache(pools, 4, cache.refcounts.long(), cache.tables, cache.lengths)
    with pytest.raises(ValueError, match="refcounts is"):
        dfccl_amd.PageCache(pools, 4, cache.refcounts[:5], cache.tables, cache.lengths)
    with pytest.raises(TypeError, match="int32"):
        cache.extend(torch.zeros(1, dtype=torch.int64, device=d), torch.zeros(1, dtype=torch.int64, device=d))
    with pytest.raises(ValueError, match="agree in length"):
        cache.fork(_ints([0]), _ints([1, 2]))
    with pytest.raises(ValueError, match="agree in length"):
        cache.copy(_ints([0]), _ints([1, 2]))
    with pytest.raises(dfccl_amd.NcclError):
        cache.extend(_ints([0, 1, 2, 0]), _ints([1, 1, 1, 1]))  # more requests than sequences
    other = dfccl_amd.PageCache.empty([torch.zeros(6, 9, device=d) for _ in range(2)], 4, 3, 2)
    with pytest.raises(dfccl_amd.NcclError):
        cache.copy(_ints([0]), _ints([1]), source=other)
    with pytest.raises(dfccl_amd.NcclError):
        dfccl_amd.PageCache.empty(pools, 0, 3, 2).compact()
    _sync()
    assert not bool(cache.refcounts.any()) and cache.lengths.tolist() == [0, 0, 0]


@big_only
def test_two_graphs_of_one_cache_replayed_in_turn():
    both = Both(pages=300, page_tokens=4, sequences=30, per_seq=30, page_bytes=(256,))
    seqs, lengths, ended, parents, children = _ints(range(10)), _ints([0] * 10), _ints([0, 1]), _ints([4, 5]), _ints([20, 21])
    torch.cuda.synchronize()
    grow, shrink = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(grow):
        both.cache.extend(seqs, lengths)
        both.cache.fork(parents, children)
    with torch.cuda.graph(shrink):
        both.cache.free(ended)
        both.cache.compact()
    rs = np.random.RandomState(21)
    for turn in range(6):
        now = [int(both.books.lengths[q]) + int(rs.randint(0, 9)) for q in range(10)]
        gone = rs.permutation(10)[:2].tolist() + []
        lengths.copy_(_ints(now))
        children.copy_(_ints([20 + turn, 26]))
        ended.copy_(_ints(gone))
        grow.replay()
        both.books.extend(list(range(10)), now)
        both.books.fork([4, 5], [20 + turn, 26])
        both.same(f"grow {turn}")
        shrink.replay()
        both.books.free(gone)
        both.books.compact()
        both.same(f"shrink {turn}")


@big_only
def test_pages_of_more_than_4_gigabytes():
    import dfccl_amd
    size = (1 << 32) + 1025  # one page: its parts are counted behind 32 bits, and the last one is odd
    pool = torch.zeros(3, size, dtype=torch.uint8, device="cuda:0")
    marks = torch.tensor([0, 1, (1 << 31) + 5, (1 << 32) - 1, 1 << 32, size - 2, size - 1], device="cuda:0")
    pool[2, marks] = torch.arange(1, 8, dtype=torch.uint8, device="cuda:0")
    cache = dfccl_amd.PageCache.empty([pool], 4, 2, 2)
    cache.copy(_ints([2]), _ints([0]))
    _sync()
    assert torch.equal(pool[0, marks], pool[2, marks]) and int(pool[0].count_nonzero()) == 7
    assert int(pool[1].count_nonzero()) == 0
