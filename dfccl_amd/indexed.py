"""Rows of a table and pages of a cache that are named by an index on the GPU: the embedding lookup and its gradient,
and the page operations of a cache, over the C ABI (dfcclEmbedding*, dfcclPages* in include/ofccl.h).  As everywhere
in this layer, buffers are torch tensors on the GPU, calls are asynchronous on `stream` (default: torch's current
stream) and the entry points check sizes; what is checked here is what a pointer no longer tells.

A call on a few rows or pages takes the GPU some three microseconds, so the checks avoid what costs as much on the
host: no tensor is made, and torch is asked for nothing twice."""
import ctypes

import torch

from . import _lib, api

_FLOATS = frozenset((torch.float32, torch.float16, torch.bfloat16))
_INT32, _INT64 = (1 << 31) - 1, -(1 << 63)  # the largest, the smallest of the C types
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the current stream's handle without an object


def _stream_of(device, stream):
    if stream is not None:
        if stream.device != device:
            raise ValueError(f"tensors on {device}, stream on {stream.device}: one call works on one device")
        return stream.cuda_stream
    if device.type == "cuda" and _raw_stream is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _capturing(stream):
    with torch.cuda.stream(stream):
        return torch.cuda.is_current_stream_capturing()


def _call(device, fn, what, *args):
    """Runs an entry point with `device` as the current one, as a launch on that device's streams needs it."""
    if device.type == "cuda" and device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            code = fn(*args)
    else:
        code = fn(*args)
    if code != 0:
        api.check(code, what)


def _ptr(t):
    return t.data_ptr() if t.is_cuda else api._dev_ptr(t)


def _row_stride(t, what):
    """Row stride (in elements) of a 2-d tensor whose rows are contiguous and do not overlap."""
    if t.dim() != 2:
        raise ValueError(f"{what} must have two dimensions")
    rows, width = t.shape
    stride, inner = t.stride()
    if rows > 1 and stride < width or width > 1 and inner != 1:
        if not t.is_contiguous():  # (strides of a tensor without elements mean nothing)
            raise ValueError(f"{what}: the elements of a row must be contiguous, and rows must not overlap")
    return stride if rows > 1 and stride > width else width


def _rows_ptr(t, what):
    """Address and row stride of a table, an output or a gradient."""
    if t.dtype not in _FLOATS:
        raise TypeError(f"{what}: dtype {t.dtype} is not one of float32, float16, bfloat16")
    return _ptr(t), _row_stride(t, what)


def _ids_ptr(ids, device):
    if ids.dtype is not torch.int64 and ids.dtype is not torch.int32:
        raise TypeError(f"ids: dtype {ids.dtype} is not int32 or int64")
    if ids.device != device:
        _on(device, ids)
    if not ids.is_contiguous():
        raise ValueError("ids must be contiguous")
    return _ptr(ids)


def _on(device, *tensors):
    for t in tensors:
        if t.device != device:
            raise ValueError(f"tensors on {device} and {t.device}: one call works on one device")


def _fits(bits, what, *numbers):
    """Refuses what ctypes would pass on as another number: it drops the bits that the C type does not hold."""
    for n in numbers:
        if not -1 << bits - 1 <= n < 1 << bits - 1:
            raise ValueError(f"{what}: {n} does not fit {bits} bits")


def embedding_lookup(table, ids, out, scale=1.0, first_row=0, stream=None):
    """out[t, :] = scale * table[ids[t] - first_row, :] (dfcclEmbeddingLookup), zeros for ids outside the table, which
    may be one rank's piece of the vocabulary.  ids may have any shape, out is [ids.numel(), width]; rows of `table`
    and `out` may be further apart than their width."""
    table_ptr, table_stride = _rows_ptr(table, "table")
    out_ptr, out_stride = _rows_ptr(out, "out")
    rows, width = table.shape
    tokens, device = ids.numel(), table.device
    if tuple(out.shape) != (tokens, width):
        raise ValueError(f"out has shape {tuple(out.shape)}, not {(tokens, width)}")
    _on(device, out)
    if not _INT64 <= first_row < -_INT64:
        _fits(64, "first_row", first_row)
    _call(device, _lib.load().dfcclEmbeddingLookup, "dfcclEmbeddingLookup", table_ptr, api.DTYPE_OF[table.dtype], rows,
          table_stride, first_row, _ids_ptr(ids, device), api.DTYPE_OF[ids.dtype], tokens, width, scale, out_ptr,
          api.DTYPE_OF[out.dtype], out_stride, _stream_of(device, stream))


def embedding_grad_workspace(tokens, rows, width):
    """Bytes of workspace that embedding_grad needs for sources of so many tokens (a list)."""
    n = ctypes.c_size_t()
    _fits(64, "sizes", *tokens, rows, width)
    api.check(_lib.load().dfcclEmbeddingGradWorkspace(len(tokens), (ctypes.c_size_t * len(tokens))(*tokens), rows, width,
                                                      ctypes.byref(n)), "dfcclEmbeddingGradWorkspace")
    return n.value


def embedding_grad(grads, ids, table_grad, scale=1.0, first_row=0, padding_id=None, accumulate=False, workspace=None,
                   stream=None):
    """table_grad[v, :] = scale * sum of the gradients of all tokens whose id is first_row + v (dfcclEmbeddingGrad),
    over one source or a list of them (the ranks' batches): grads[r] is [ids[r].numel(), width].  Tokens whose id is
    padding_id are left out.  accumulate: add to the rows that tokens name instead of writing all rows.  workspace: a
    tensor of at least embedding_grad_workspace() bytes (default: one is allocated)."""
    if isinstance(grads, torch.Tensor):
        grads, ids = (grads,), (ids,)
    n = len(grads)
    if n != len(ids) or n == 0:
        raise ValueError("as many ids as gradients, and at least one of each")
    table_ptr, table_stride = _rows_ptr(table_grad, "table_grad")
    rows, width = table_grad.shape
    device, dtype, id_type = table_grad.device, grads[0].dtype, ids[0].dtype
    if dtype not in _FLOATS:
        raise TypeError(f"grads: dtype {dtype} is not one of float32, float16, bfloat16")
    _fits(64, "first_row", first_row)
    padding_id = -1 if padding_id is None else padding_id
    _fits(64, "padding_id", padding_id)
    grad_ptrs, id_ptrs, sizes = (ctypes.c_void_p * n)(), (ctypes.c_void_p * n)(), (ctypes.c_size_t * n)()
    grad_stride = None
    for r in range(n):
        g, i = grads[r], ids[r]
        if g.dtype is not dtype or i.dtype is not id_type:
            raise ValueError("the sources must agree in dtype")
        tokens = i.numel()
        stride = _row_stride(g, "grads")
        if g.shape[0] != tokens or g.shape[1] != width:
            raise ValueError(f"grads[{r}] has shape {tuple(g.shape)}, not {(tokens, width)}")
        if g.device != device:
            _on(device, g)
        grad_ptrs[r], id_ptrs[r], sizes[r] = _ptr(g), _ids_ptr(i, device), tokens
        if tokens > 1:
            if grad_stride is not None and grad_stride != stride:
                raise ValueError("the sources must agree in their row stride")
            grad_stride = stride
    lib, handle = _lib.load(), _stream_of(device, stream)
    if workspace is None:
        need = ctypes.c_size_t()
        api.check(lib.dfcclEmbeddingGradWorkspace(n, sizes, rows, width, ctypes.byref(need)), "dfcclEmbeddingGradWorkspace")
        # From the pool of the stream that the call runs on: a block of another stream's pool may have been freed by a
        # tensor whose kernels are still queued there, and this stream does not wait for those.
        if stream is None:
            workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
        else:
            with torch.cuda.stream(stream):
                workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
    else:
        _on(device, workspace)
    _call(device, lib.dfcclEmbeddingGrad, "dfcclEmbeddingGrad", grad_ptrs, id_ptrs, sizes, n, api.DTYPE_OF[dtype],
          width if grad_stride is None else grad_stride, api.DTYPE_OF[id_type], first_row, rows, width,
          padding_id, scale, int(accumulate), table_ptr, api.DTYPE_OF[table_grad.dtype],
          table_stride, api._dev_ptr(workspace), workspace.numel() * workspace.element_size(), handle)


class PageCache:
    """A rank's cache of pages (dfcclPageCache): `pools` is a list of contiguous tensors [pages, ...] whose pages hold
    `page_tokens` tokens, and refcounts [pages], tables [sequences, pages per sequence] and lengths [sequences] are its
    bookkeeping, int32 tensors that the caller owns (PageCache.empty makes those of an empty cache).  report[0]:
    requests refused by the last extend or fork; report[1], report[2]: pages moved, pages live at the last compact.

    The report and a workspace (and what empty() makes) are the cache's own memory, taken on the stream that is current in
    the constructor; the first call on another stream waits for what the constructor needs of that one.  A graph with captured calls uses
    them too: keep the cache as long as the graph, and capture once the constructor's stream has got that far
    (torch.cuda.graph waits for the device)."""

    def __init__(self, pools, page_tokens, refcounts, tables, lengths):
        pages, size, device = pools[0].shape[0], pools[0].nbytes, refcounts.device
        pointers = (ctypes.c_void_p * len(pools))()
        for k, p in enumerate(pools):
            if p.nbytes != size or p.shape[0] != pages:
                raise ValueError("the pools must agree in pages and bytes per page")
            if p.device != device:
                _on(device, p)
            pointers[k] = p.data_ptr() if p.is_cuda and p.is_contiguous() else api._dev_ptr(p)
        for t in (refcounts, tables, lengths):
            if t.dtype != torch.int32:
                raise TypeError("the bookkeeping is held in int32 tensors")
        if refcounts.shape != (pages,) or tables.dim() != 2 or lengths.shape != (tables.shape[0],):
            raise ValueError("refcounts is [pages], tables [sequences, pages per sequence], lengths [sequences]")
        _on(device, tables, lengths)
        _fits(32, "a cache's sizes", len(pools), pages, page_tokens, *tables.shape)
        lib = _lib.load()
        need = ctypes.c_size_t()
        api.check(lib.dfcclPageCacheWorkspace(pages, tables.shape[0], ctypes.byref(need)), "dfcclPageCacheWorkspace")
        self.pools, self.page_tokens = pools, page_tokens
        self.refcounts, self.tables, self.lengths = refcounts, tables, lengths
        self.report = torch.zeros(3, dtype=torch.int32, device=device)
        self._device, self._lib, self._pointers = device, lib, pointers
        self._workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
        self._struct = _lib.PageCacheStruct(
            ctypes.sizeof(_lib.PageCacheStruct), pointers, size // max(1, pages), len(pools), pages, page_tokens,
            tables.shape[0], tables.shape[1], api._dev_ptr(refcounts), api._dev_ptr(tables), api._dev_ptr(lengths),
            api._dev_ptr(self.report), api._dev_ptr(self._workspace), need.value)
        self._ref = ctypes.byref(self._struct)
        self._own = [self._workspace, self.report]
        # What comes before this place on the constructor's stream may still use the memory, and clears the report.
        self._made_on, self._joined, self._made = _stream_of(device, None), {}, None
        if device.type == "cuda":
            here = torch.cuda.current_stream(device)
            if not _capturing(here):
                self._made = here.record_event()

    @classmethod
    def empty(cls, pools, page_tokens, sequences, pages_per_sequence):
        """A cache whose pages are all free."""
        def ints(value, *shape):
            return torch.full(shape, value, dtype=torch.int32, device=pools[0].device)
        cache = cls(pools, page_tokens, ints(0, pools[0].shape[0]), ints(-1, sequences, pages_per_sequence),
                    ints(0, sequences))
        cache._own += [cache.refcounts, cache.tables, cache.lengths]
        return cache

    def _stream(self, stream):
        """The stream's handle, for calls that use the cache's own memory. Another stream than the constructor's waits for
        that one once, and the memory does not return to its pool before that other stream is through with it."""
        handle = _stream_of(self._device, stream)
        if handle != self._made_on and handle not in self._joined:
            if stream is None:
                stream = torch.cuda.current_stream(self._device)
            for t in self._own:
                t.record_stream(stream)
            if not _capturing(stream):  # (a capture may not wait for an event from before it)
                if self._made is not None:
                    stream.wait_event(self._made)
                self._joined[handle] = stream
        return handle

    def _lists(self, *lists):
        """Addresses of the lists, and their common length."""
        n = lists[0].numel()
        if n > _INT32:
            _fits(32, "a list's length", n)
        for t in lists:
            if t.dtype is not torch.int32:
                raise TypeError("lists of sequences, pages and lengths are int32 tensors")
            if t.numel() != n:
                raise ValueError("the lists must agree in length")
        _on(self._device, *lists)
        return [api._dev_ptr(t) for t in lists] + [n]

    def copy(self, src_pages, dst_pages, source=None, stream=None):
        """Contents of the pages src_pages of `source` (default: this cache) into this cache's dst_pages, all pools."""
        lists = self._lists(src_pages, dst_pages)
        if source is None:
            source = self
        elif source._device != self._device:
            raise ValueError("the two caches must be on one device")
        _call(self._device, self._lib.dfcclPagesCopy, "dfcclPagesCopy", self._ref, source._ref, *lists,
              _stream_of(self._device, stream))

    def extend(self, sequences, lengths, stream=None):
        """The sequences grow to these lengths; new entries get the lowest free pages."""
        _call(self._device, self._lib.dfcclPagesExtend, "dfcclPagesExtend", self._ref, *self._lists(sequences, lengths),
              self._stream(stream))

    def fork(self, parents, children, stream=None):
        """The children (empty) become copies of the parents: full pages shared, a last page that is not full copied."""
        _call(self._device, self._lib.dfcclPagesFork, "dfcclPagesFork", self._ref, *self._lists(parents, children),
              self._stream(stream))

    def free(self, sequences, stream=None):
        """The sequences become empty and give up their pages."""
        _call(self._device, self._lib.dfcclPagesFree, "dfcclPagesFree", self._ref, *self._lists(sequences),
              self._stream(stream))

    def compact(self, stream=None):
        """Moves pages until the live ones have the lowest numbers; counts and tables follow."""
        _call(self._device, self._lib.dfcclPagesCompact, "dfcclPagesCompact", self._ref, self._stream(stream))
