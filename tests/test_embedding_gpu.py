"""The embedding lookup and its gradient (dfcclEmbeddingLookup, dfcclEmbeddingGrad through the C ABI) against their
definitions in 64 bits, within bounds that follow from the arithmetic (indexed_util): types, odd sizes and strides,
pieces of the vocabulary, padding, runs around the block sizes, several sources, graphs and streams."""
import numpy as np
import pytest
import torch

import gpu_util
import indexed_util as iu

pytestmark = pytest.mark.gpu
big_only = pytest.mark.skipif(gpu_util.EMULATED, reason="size or feature of a real GPU")


def _sync():
    torch.cuda.current_stream().synchronize()


def _randn(seed, *shape, dtype=torch.float32, pad=0):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn(*shape[:-1], shape[-1] + pad, generator=g).to(dtype).to(gpu_util.DEVICE)
    return t[..., :shape[-1]]


def _ids(seed, n, low, high, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(low, high, (n,), generator=g).to(dtype).to(gpu_util.DEVICE)


def _lookup(table, ids, out_dtype, scale=1.0, first=0, pad=0):
    """Runs the lookup into a marked buffer and checks that nothing but the output was written."""
    import dfccl_amd
    n, w = ids.numel(), table.shape[1]
    buf = torch.full((n + 1, w + pad), 7.0, dtype=out_dtype, device=gpu_util.DEVICE)
    out = buf[:n, :w]
    dfccl_amd.embedding_lookup(table, ids, out, scale=scale, first_row=first)
    _sync()
    assert bool((buf[:, w:] == 7).all()) and bool((buf[n] == 7).all())
    return out


# ---- lookup ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("out", iu.FLOATS)
@pytest.mark.parametrize("table", iu.FLOATS)
def test_lookup_types(table, out):
    t, ids = _randn(1, 40, 75, dtype=table), _ids(2, 33, 0, 40)
    iu.check(_lookup(t, ids, out, scale=8.66), *iu.lookup(t, ids, 0, 8.66))


@pytest.mark.parametrize("width", [1, 7, 8, 9, 511, 512, 513, 1000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_lookup_widths_and_strides(width, dtype):
    for pad_table, pad_out in ((0, 0), (3, 0), (8, 5)):
        t, ids = _randn(3, 21, width, dtype=dtype, pad=pad_table), _ids(4, 13, 0, 21, torch.int32)
        iu.check(_lookup(t, ids, dtype, scale=0.3, pad=pad_out), *iu.lookup(t, ids, 0, 0.3))


@pytest.mark.parametrize("tokens", [0, 1, 2, 3, 64, 65])
def test_lookup_token_counts(tokens):
    t, ids = _randn(5, 10, 40, dtype=torch.float16), _ids(6, tokens, 0, 10)
    iu.check(_lookup(t, ids, torch.float16, scale=2.0), *iu.lookup(t, ids, 0, 2.0))


@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
def test_lookup_of_a_piece_gives_zeros_for_ids_outside(id_type):
    t = _randn(7, 20, 33, dtype=torch.bfloat16)
    t[3] = float("nan")  # a row that no id names, and rows that ids outside may not be mistaken for
    info = torch.iinfo(id_type)
    named = [info.min, info.min + 1, -1, 0, 99, 100, 102, 104, 119, 120, 121, info.max, info.max - 1, 100]
    ids = torch.tensor(named, dtype=id_type, device=gpu_util.DEVICE)
    got = _lookup(t, ids, torch.float32, scale=1.5, first=100)
    iu.check(got, *iu.lookup(t, ids, 100, 1.5))
    inside = torch.tensor([100 <= i < 120 for i in named])
    assert bool((got.cpu()[~inside] == 0).all()) and bool((got.cpu()[inside] != 0).any(1).all())


def test_lookup_at_the_end_of_the_id_range():
    first = (1 << 63) - 20
    t = _randn(8, 19, 16)
    ids = torch.tensor([first, first + 18, -(1 << 63), -(1 << 63) + 3, 0, first - 1], device=gpu_util.DEVICE)
    got = _lookup(t, ids, torch.float32, first=first)
    assert torch.equal(got[0], t[0]) and torch.equal(got[1], t[18]) and not bool(got[2:].any())


def test_lookup_passes_infinities_and_nan_through_and_only_there():
    t = _randn(9, 6, 24)
    t[1, 3], t[1, 4], t[2, 20] = float("inf"), float("-inf"), float("nan")
    ids = torch.tensor([0, 1, 2, 5, 9], device=gpu_util.DEVICE)
    got = _lookup(t, ids, torch.float16, scale=2.0).cpu()
    assert got[1, 3] == float("inf") and got[1, 4] == float("-inf") and torch.isnan(got[2, 20])
    assert int((~torch.isfinite(got)).sum()) == 3 and not bool(got[4].any())


def test_lookup_of_an_empty_piece_and_of_rows_of_no_width():
    import dfccl_amd
    ids = torch.tensor([0, 5], device=gpu_util.DEVICE)
    out = torch.ones(2, 8, device=gpu_util.DEVICE)
    dfccl_amd.embedding_lookup(torch.empty(0, 8, device=gpu_util.DEVICE), ids, out)
    _sync()
    assert not bool(out.any())
    dfccl_amd.embedding_lookup(torch.empty(4, 0, device=gpu_util.DEVICE), ids, torch.empty(2, 0, device=gpu_util.DEVICE))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_lookup_from_and_to_addresses_aligned_to_an_element_only(dtype):
    import dfccl_amd
    flat = _randn(10, 1 + 15 * 72, dtype=dtype)
    t = flat[1:].view(15, 72)
    ids = _ids(11, 17, 0, 15)
    buf = torch.full((3 + 17 * 72,), 7.0, dtype=dtype, device=gpu_util.DEVICE)
    out = buf[3:].view(17, 72)
    dfccl_amd.embedding_lookup(t, ids, out, scale=-1.25)
    _sync()
    assert bool((buf[:3] == 7).all())
    iu.check(out, *iu.lookup(t, ids, 0, -1.25))


def test_lookup_with_several_rows_a_wave():
    # from 16384 pieces of 512 elements on a wave takes two tokens' rows; 4099 tokens leave the last one a single one
    t, ids = _randn(12, 9, 4100, dtype=torch.bfloat16), _ids(13, 4099, -1, 10)
    iu.check(_lookup(t, ids, torch.bfloat16, scale=0.7), *iu.lookup(t, ids, 0, 0.7))


@big_only
def test_lookup_where_offsets_pass_32_bits():
    rows, width = 600_000, 4096  # 4.9 GB
    t = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda:0")
    ids = torch.tensor([0, 262_143, 262_144, 524_288, 524_287, 599_999], device="cuda:0")
    t[ids] = torch.arange(1, 7, device="cuda:0", dtype=torch.bfloat16)[:, None]
    got = _lookup(t, ids, torch.bfloat16)
    assert torch.equal(got, t[ids])
    out = torch.zeros(600_000, 4096, dtype=torch.bfloat16, device="cuda:0")
    many = torch.arange(600_000, device="cuda:0")
    import dfccl_amd
    dfccl_amd.embedding_lookup(t, many, out)
    _sync()
    assert torch.equal(out, t)


# ---- gradient -------------------------------------------------------------------------------------------------

def _grad(grads, ids, rows, dtype, scale=1.0, first=0, padding=None, accumulate=False, pad=0):
    """Runs the gradient into a marked buffer and compares it with the definition."""
    import dfccl_amd
    width = grads[0].shape[1]
    buf = torch.full((rows + 1, width + pad), 7.0, dtype=dtype, device=gpu_util.DEVICE)
    if accumulate:
        buf[:rows, :width] = _randn(99, rows, width, dtype=dtype)
    old = buf[:rows, :width].clone()
    out = buf[:rows, :width]
    dfccl_amd.embedding_grad(list(grads), list(ids), out, scale=scale, first_row=first, padding_id=padding,
                             accumulate=accumulate)
    _sync()
    exact, before, count = iu.grad(grads, ids, rows, first, scale, padding, old if accumulate else None)
    iu.check(out, exact, before)
    unnamed = (count == 0).to(gpu_util.DEVICE)
    if accumulate:
        assert torch.equal(out[unnamed], old[unnamed])  # not a bit of the other rows changes
    else:
        assert not bool(out[unnamed].any())
    assert bool((buf[:, width:] == 7).all()) and bool((buf[rows] == 7).all())
    return out


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("table", iu.FLOATS)
@pytest.mark.parametrize("g", iu.FLOATS)
def test_grad_types(g, table, accumulate):
    _grad([_randn(20, 50, 41, dtype=g)], [_ids(21, 50, 0, 12)], 12, table, scale=0.5, accumulate=accumulate)


@pytest.mark.parametrize("width", [1, 7, 8, 511, 513, 1030])
@pytest.mark.parametrize("accumulate", [False, True])
def test_grad_widths_and_strides(width, accumulate):
    for pad_grad, pad in ((0, 0), (1, 3)):
        _grad([_randn(22, 70, width, dtype=torch.bfloat16, pad=pad_grad)], [_ids(23, 70, 0, 4, torch.int32)], 6,
              torch.float32, accumulate=accumulate, pad=pad)


# runs around the block of 16 tokens, the 64 that a wave sees, and the block of 16 blocks
@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 31, 32, 33, 62, 63, 64, 65, 66, 100, 255, 256, 257, 1023, 1024, 1300, 3100])
@pytest.mark.parametrize("accumulate", [False, True])
def test_grad_of_one_token_many_times(tokens, accumulate):
    _grad([_randn(24, tokens, 24)], [torch.full((tokens,), 3, device=gpu_util.DEVICE)], 5, torch.float32,
          accumulate=accumulate)


@big_only
@pytest.mark.parametrize("tokens", [8191, 8192, 8193, 20000, 33000])
def test_grad_of_one_token_thousands_of_times(tokens):
    for ahead in (0, 45):
        ids = torch.full((tokens + ahead,), 3, device="cuda:0")
        ids[:ahead] = 1
        _grad([_randn(24, tokens + ahead, 24)], [ids], 5, torch.float32)


@pytest.mark.parametrize("ahead", [0, 1, 2, 3, 4, 13, 15, 16, 17, 31, 250])
def test_grad_of_long_runs_that_begin_anywhere(ahead):
    ids = torch.cat([torch.full((n,), v) for v, n in ((0, ahead), (2, 600), (3, 1), (4, 64), (5, 31), (6, 600))])
    ids = ids[torch.randperm(ids.numel(), generator=torch.Generator().manual_seed(ahead))].to(gpu_util.DEVICE)
    _grad([_randn(25, ids.numel(), 16, dtype=torch.float16)], [ids], 8, torch.float32, scale=-0.1)


@pytest.mark.parametrize("accumulate", [False, True])
def test_grad_of_a_piece_with_padding_and_ids_outside(accumulate):
    info = torch.iinfo(torch.int64)
    ids = torch.cat([_ids(26, 200, 90, 130), torch.tensor([info.min, info.max, -1, 0], device=gpu_util.DEVICE)])
    ids[5:90] = 105
    _grad([_randn(27, 204, 30)], [ids], 20, torch.float32, first=100, padding=105, accumulate=accumulate)


def test_grad_of_padding_alone_of_no_tokens_and_of_ids_all_outside():
    import dfccl_amd
    for ids in (torch.full((40,), 2), torch.empty(0, dtype=torch.int64), torch.full((40,), 50)):
        ids = ids.to(gpu_util.DEVICE)
        _grad([_randn(28, ids.numel(), 12)], [ids], 9, torch.bfloat16, padding=2)
        _grad([_randn(28, ids.numel(), 12)], [ids], 9, torch.float32, padding=2, accumulate=True)
    # NaN in the gradients of tokens that do not count stays out
    g = _randn(29, 6, 8)
    g[2:4] = float("nan")
    ids = torch.tensor([0, 1, 7, 7, 1, 20], device=gpu_util.DEVICE)
    out = torch.full((9, 8), 5.0, device=gpu_util.DEVICE)
    dfccl_amd.embedding_grad(g, ids, out, padding_id=7)
    _sync()
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("counts", [(50, 50), (1, 0, 33), (0, 0), (7,) * 8, (300, 2, 0, 1200)])
def test_grad_of_several_sources(counts, accumulate):
    grads = [_randn(30 + r, n, 20, dtype=torch.bfloat16) for r, n in enumerate(counts)]
    ids = [_ids(40 + r, n, 0, 7, torch.int32) for r, n in enumerate(counts)]
    _grad(grads, ids, 7, torch.float32, scale=0.125, padding=6, accumulate=accumulate)


def test_grad_sums_in_the_order_of_sources_and_tokens():
    # (a + b) + c differs from a + (b + c) here; the sum goes source by source, token by token
    big = 2.0 ** 25
    a = [torch.tensor([[big], [1.0]], device=gpu_util.DEVICE), torch.tensor([[1.0], [-big]], device=gpu_util.DEVICE)]
    ids = [torch.tensor([1, 1], device=gpu_util.DEVICE)] * 2
    out = torch.zeros(2, 1, device=gpu_util.DEVICE)
    import dfccl_amd
    dfccl_amd.embedding_grad(a, ids, out)
    _sync()
    assert out[1, 0].item() == 0.0  # ((big + 1) + 1) - big, each 1 lost
    dfccl_amd.embedding_grad([a[0].flip(0), a[1].flip(0)], ids, out)
    _sync()
    assert out[1, 0].item() == 1.0  # ((1 + big) - big) + 1


def test_grad_gives_the_same_bits_again():
    import dfccl_amd
    n = 2500 if gpu_util.EMULATED else 20000
    g, ids = _randn(50, n, 40, dtype=torch.bfloat16), _ids(51, n, 0, 30)
    outs = []
    for _ in range(2 if gpu_util.EMULATED else 5):
        out = torch.empty(30, 40, device=gpu_util.DEVICE)
        dfccl_amd.embedding_grad(g, ids, out, scale=1 / 3)
        _sync()
        outs.append(out)
    assert all(torch.equal(outs[0], o) for o in outs)


@pytest.mark.parametrize("rows", [1, 2, 255, 256, 1023, 1024, 1025, 3000])
def test_grad_row_counts_around_the_digits_of_the_sort(rows):
    ids = _ids(52, 400, -2, rows + 2)
    ids[:3] = torch.tensor([0, rows - 1, rows])
    _grad([_randn(53, 400, 9)], [ids], rows, torch.float32)


@pytest.mark.parametrize("tokens", [1500, 1501] + ([] if gpu_util.EMULATED else [4096, 4097, 16384, 16385, 65536, 65537]))
def test_grad_sorts_by_one_workgroup_and_over_several_tiles(tokens):
    # one workgroup sorts up to 4096 tokens (up to 1500 in the host build); tiles are of 512, 1024 and 4096
    ids = _ids(54, tokens, 0, 1500)
    _grad([_randn(55, tokens, 8)], [ids], 1500, torch.float32, accumulate=tokens % 2 == 0)


@big_only
@pytest.mark.parametrize("tokens,rows,width", [(70_001, 50_257, 24), (65_536, 1_100_003, 8), (65_537, 3, 16),
                                               (300_000, 200, 40)])
def test_grad_of_many_tokens_and_of_three_digit_ids(tokens, rows, width):
    _grad([_randn(56, tokens, width, dtype=torch.bfloat16)], [_ids(57, tokens, 0, rows)], rows, torch.float32, scale=0.01)
    _grad([_randn(56, tokens, width, dtype=torch.bfloat16)], [_ids(57, tokens, 0, rows)], rows, torch.float32, scale=0.01,
          accumulate=True)


@big_only
def test_grad_where_offsets_pass_32_bits():
    import dfccl_amd
    tokens, rows, width = 600_000, 600_000, 4096
    g = torch.zeros(tokens, width, dtype=torch.bfloat16, device="cuda:0")
    at = torch.tensor([0, 262_144, 524_288, 524_289, 599_999], device="cuda:0")
    g[at] = torch.arange(1, 6, device="cuda:0", dtype=torch.bfloat16)[:, None]
    ids = torch.arange(tokens, device="cuda:0").flip(0).contiguous()
    out = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda:0")
    dfccl_amd.embedding_grad(g, ids, out)
    _sync()
    assert torch.equal(out, g.flip(0))


@pytest.mark.parametrize("first,padding", [(0, None), (4, 6)])
def test_grad_is_the_adjoint_of_the_lookup(first, padding):
    # <lookup(T + h E) - lookup(T), W> / h = <E, grad(W)>: with h a power of two and everything a multiple of 1/64
    # below 2^8, fp32 holds each lookup exactly and the two sides differ only by the sums taken here in 64 bits
    import dfccl_amd
    g = torch.Generator().manual_seed(60)
    def grid(*shape):
        return torch.randint(-64, 65, shape, generator=g).float().div_(64).to(gpu_util.DEVICE)
    table, direction, w = grid(10, 17), grid(10, 17), grid(40, 17)
    ids = _ids(61, 40, 0, 16)
    out = torch.empty(40, 17, device=gpu_util.DEVICE)
    sides = []
    for h in (0.0, 0.5):
        dfccl_amd.embedding_lookup(table + h * direction, ids, out, scale=0.25, first_row=first)
        _sync()
        counted = torch.ones(40, 1, device=gpu_util.DEVICE) if padding is None else (ids != padding)[:, None].float()
        sides.append((out * counted).double().cpu())
    left = ((sides[1] - sides[0]) * w.double().cpu()).sum().item() / 0.5
    got = torch.empty(10, 17, device=gpu_util.DEVICE)
    dfccl_amd.embedding_grad(w, ids, got, scale=0.25, first_row=first, padding_id=padding)
    _sync()
    right = (got.double().cpu() * direction.double().cpu()).sum().item()
    assert left == right


# ---- graphs, streams, workspaces --------------------------------------------------------------------------------

@big_only
def test_captured_and_replayed_with_new_ids():
    import dfccl_amd
    t, g = _randn(70, 500, 130, dtype=torch.bfloat16), _randn(71, 3000, 130, dtype=torch.bfloat16)
    ids = _ids(72, 3000, 0, 500)
    out, dt = torch.empty(3000, 130, device="cuda:0"), torch.empty(500, 130, device="cuda:0")
    added = torch.zeros(500, 130, device="cuda:0")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dfccl_amd.embedding_lookup(t, ids, out, scale=3.0)
        dfccl_amd.embedding_grad(g, ids, dt)
        dfccl_amd.embedding_grad(g, ids, added, accumulate=True)
    for k in range(4):
        ids.copy_(_ids(80 + k, 3000, 0, 500 if k % 2 else 5))
        added.zero_()
        graph.replay()
        torch.cuda.synchronize()
        iu.check(out, *iu.lookup(t, ids, 0, 3.0))
        eager, again = torch.empty_like(dt), torch.zeros_like(dt)
        dfccl_amd.embedding_grad(g, ids, eager)
        dfccl_amd.embedding_grad(g, ids, again, accumulate=True)
        torch.cuda.synchronize()
        assert torch.equal(dt, eager) and torch.equal(added, again)


@big_only
def test_on_a_stream_of_its_own():
    import dfccl_amd
    s = torch.cuda.Stream()
    t, ids = _randn(73, 300, 64), _ids(74, 900, 0, 300)
    g = _randn(75, 900, 64)
    out, dt = torch.zeros(900, 64, device="cuda:0"), torch.zeros(300, 64, device="cuda:0")
    s.wait_stream(torch.cuda.current_stream())
    dfccl_amd.embedding_lookup(t, ids, out, stream=s)
    dfccl_amd.embedding_grad(g, ids, dt, stream=s)
    torch.empty(1 << 22, device="cuda:0").fill_(float("nan"))  # (takes the workspace's memory if it came back too early)
    s.synchronize()
    iu.check(out, *iu.lookup(t, ids, 0, 1.0))
    exact, before, _ = iu.grad([g], [ids], 300, 0, 1.0, None)
    iu.check(dt, exact, before)


def test_grad_in_a_workspace_of_exactly_the_size_asked_for():
    import dfccl_amd
    n = dfccl_amd.embedding_grad_workspace([1100, 40], 70, 33)
    buf = torch.full((n + 512,), 0xA5, dtype=torch.uint8, device=gpu_util.DEVICE)
    g, ids = [_randn(76, 1100, 33), _randn(77, 40, 33)], [torch.full((1100,), 7, device=gpu_util.DEVICE), _ids(78, 40, 0, 70)]
    out = torch.empty(70, 33, device=gpu_util.DEVICE)
    dfccl_amd.embedding_grad(g, ids, out, workspace=buf[256:256 + n])
    _sync()
    assert bool((buf[:256] == 0xA5).all()) and bool((buf[256 + n:] == 0xA5).all())
    exact, before, _ = iu.grad(g, ids, 70, 0, 1.0, None)
    iu.check(out, exact, before)


# ---- refusals -----------------------------------------------------------------------------------------------------

def test_refusals_of_the_python_layer():
    import dfccl_amd
    d = gpu_util.DEVICE
    t, ids, out = torch.zeros(5, 8, device=d), torch.zeros(3, dtype=torch.int64, device=d), torch.zeros(3, 8, device=d)
    with pytest.raises(ValueError, match="out has shape"):
        dfccl_amd.embedding_lookup(t, ids, out[:2])
    with pytest.raises(TypeError, match="ids"):
        dfccl_amd.embedding_lookup(t, ids.to(torch.int16), out)
    with pytest.raises(TypeError, match="table"):
        dfccl_amd.embedding_lookup(t.double(), ids, out)
    with pytest.raises(ValueError, match="contiguous"):
        dfccl_amd.embedding_lookup(torch.zeros(8, 5, device=d).t(), ids, out)
    with pytest.raises(ValueError, match="overlap"):
        dfccl_amd.embedding_lookup(t, ids, torch.zeros(8, device=d).expand(3, 8))
    with pytest.raises(dfccl_amd.NcclError):
        dfccl_amd.embedding_lookup(t, ids, out, first_row=-1)
    with pytest.raises(ValueError, match="grads"):
        dfccl_amd.embedding_grad(out, ids[:2], t)
    with pytest.raises(ValueError, match="as many ids"):
        dfccl_amd.embedding_grad([out], [], t)
    with pytest.raises(ValueError, match="dtype"):
        dfccl_amd.embedding_grad([out, out.half()], [ids, ids], t)
    with pytest.raises(ValueError, match="stride"):
        dfccl_amd.embedding_grad([out, torch.zeros(3, 9, device=d)[:, :8]], [ids, ids], t)
    with pytest.raises(dfccl_amd.NcclError):
        dfccl_amd.embedding_grad([out] * 9, [ids] * 9, t)
    with pytest.raises(dfccl_amd.NcclError):
        dfccl_amd.embedding_grad(out, ids, t, workspace=torch.empty(16, dtype=torch.uint8, device=d))
    _sync()
    assert not bool(out.any()) and not bool(t.any())


@big_only
def test_gradients_on_two_streams_at_once():
    import dfccl_amd
    s = [torch.cuda.Stream() for _ in range(2)]
    g = [_randn(90 + k, 9000, 256, dtype=torch.bfloat16) for k in range(2)]
    ids = [_ids(92 + k, 9000, 0, 700) for k in range(2)]
    outs = [[torch.empty(700, 256, device="cuda:0") for _ in range(8)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(8):
        for k in range(2):
            dfccl_amd.embedding_grad(g[k], ids[k], outs[k][i], stream=s[k])
    torch.cuda.synchronize()
    for k in range(2):
        exact, before, _ = iu.grad([g[k]], [ids[k]], 700, 0, 1.0, None)
        iu.check(outs[k][0], exact, before)
        assert all(torch.equal(outs[k][0], o) for o in outs[k])


@big_only
def test_two_graphs_that_share_a_workspace_replayed_in_turn():
    import dfccl_amd
    n = dfccl_amd.embedding_grad_workspace([5000], 400, 96)
    assert n >= dfccl_amd.embedding_grad_workspace([300], 400, 96)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda:0")
    g = [_randn(94, 5000, 96), _randn(95, 300, 96)]
    ids = [_ids(96, 5000, 0, 400), _ids(97, 300, 0, 400)]
    outs, graphs = [torch.empty(400, 96, device="cuda:0") for _ in range(2)], []
    torch.cuda.synchronize()
    for k in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[k]):
            dfccl_amd.embedding_grad(g[k], ids[k], outs[k], workspace=ws)
    for turn in range(4):
        for k in (turn % 2, 1 - turn % 2):
            ids[k].copy_(_ids(100 + 2 * turn + k, ids[k].numel(), 0, 400))
            outs[k].fill_(float("nan"))
            graphs[k].replay()
        torch.cuda.synchronize()
        for k in range(2):
            exact, before, _ = iu.grad([g[k]], [ids[k]], 400, 0, 1.0, None)
            iu.check(outs[k], exact, before)
