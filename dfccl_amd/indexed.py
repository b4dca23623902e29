"""Rows of a table and pages of a cache that are named by an index on the GPU: the embedding lookup and its gradient,
and the page operations of a cache, over the C ABI (dfcclEmbedding*, dfcclPages* in include/ofccl.h).  As everywhere
in this layer, buffers are torch tensors on the GPU, calls are asynchronous on `stream` (default: torch's current
stream) and the entry points check sizes; what is checked here is what a pointer no longer tells."""
import ctypes
import functools

import torch

from . import _lib, api

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _stream_of(t, stream):
    return ctypes.c_void_p((torch.cuda.current_stream(t.device) if stream is None else stream).cuda_stream)


def _on_device_of(fn):
    """Runs fn with the current device that of its `where` tensor, as a launch on that device's streams needs it."""
    @functools.wraps(fn)
    def wrapped(where, *args):
        if where.is_cuda and where.device.index != torch.cuda.current_device():
            with torch.cuda.device(where.device):
                return fn(where, *args)
        return fn(where, *args)
    return wrapped


def _rows_ptr(t, what):
    """Address and row stride (in elements) of a 2-d tensor whose rows are contiguous."""
    if t.dim() != 2:
        raise ValueError(f"{what} must have two dimensions")
    if t.dtype not in _FLOATS:
        raise TypeError(f"{what}: dtype {t.dtype} is not one of float32, float16, bfloat16")
    if t.is_contiguous():
        return api._dev_ptr(t), t.shape[1]
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError(f"{what}: the elements of a row must be contiguous, and rows must not overlap")
    return api._dev_ptr(t[0]), t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _ids_ptr(ids):
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids: dtype {ids.dtype} is not int32 or int64")
    return api._dev_ptr(ids)


def _same_device(first, *others):
    for t in others:
        if t.device != first.device:
            raise ValueError(f"tensors on {first.device} and {t.device}: one call works on one device")


@_on_device_of
def _call(where, fn, what, *args):
    api.check(fn(*args), what)


def embedding_lookup(table, ids, out, scale=1.0, first_row=0, stream=None):
    """out[t, :] = scale * table[ids[t] - first_row, :] (dfcclEmbeddingLookup), zeros for ids outside the table, which
    may be one rank's piece of the vocabulary.  ids may have any shape, out is [ids.numel(), width]; rows of `table`
    and `out` may be further apart than their width."""
    _same_device(table, ids, out)
    table_ptr, table_stride = _rows_ptr(table, "table")
    out_ptr, out_stride = _rows_ptr(out, "out")
    if out.shape[0] != ids.numel() or out.shape[1] != table.shape[1]:
        raise ValueError(f"out has shape {tuple(out.shape)}, not {(ids.numel(), table.shape[1])}")
    _call(table, _lib.load().dfcclEmbeddingLookup, "dfcclEmbeddingLookup", table_ptr, api.nccl_dtype(table),
          table.shape[0], table_stride, first_row, _ids_ptr(ids), api.nccl_dtype(ids), ids.numel(), table.shape[1], scale,
          out_ptr, api.nccl_dtype(out), out_stride, _stream_of(table, stream))


def embedding_grad_workspace(tokens, rows, width):
    """Bytes of workspace that embedding_grad needs for sources of so many tokens (a list)."""
    n = ctypes.c_size_t()
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
        grads, ids = [grads], [ids]
    if len(grads) != len(ids) or not grads:
        raise ValueError("as many ids as gradients, and at least one of each")
    _same_device(table_grad, *grads, *ids)
    table_ptr, table_stride = _rows_ptr(table_grad, "table_grad")
    rows, width = table_grad.shape
    n = len(grads)
    grad_ptrs, id_ptrs, tokens, strides = (ctypes.c_void_p * n)(), (ctypes.c_void_p * n)(), [], set()
    for r, (g, i) in enumerate(zip(grads, ids)):
        grad_ptrs[r], stride = _rows_ptr(g, "grads")
        id_ptrs[r] = _ids_ptr(i)
        if g.dtype != grads[0].dtype or i.dtype != ids[0].dtype:
            raise ValueError("the sources must agree in dtype")
        if g.shape[0] != i.numel() or g.shape[1] != width:
            raise ValueError(f"grads[{r}] has shape {tuple(g.shape)}, not {(i.numel(), width)}")
        tokens.append(g.shape[0])
        if g.shape[0] > 1:
            strides.add(stride)
    if len(strides) > 1:
        raise ValueError("the sources must agree in their row stride")
    lib = _lib.load()
    sizes = (ctypes.c_size_t * n)(*tokens)
    need = ctypes.c_size_t()
    api.check(lib.dfcclEmbeddingGradWorkspace(n, sizes, rows, width, ctypes.byref(need)), "dfcclEmbeddingGradWorkspace")
    if workspace is None:
        workspace = torch.empty(need.value, dtype=torch.uint8, device=table_grad.device)
        if stream is not None and table_grad.is_cuda:
            workspace.record_stream(stream)
    _same_device(table_grad, workspace)
    _call(table_grad, lib.dfcclEmbeddingGrad, "dfcclEmbeddingGrad", grad_ptrs, id_ptrs, sizes, n, api.nccl_dtype(grads[0]),
          strides.pop() if strides else width, api.nccl_dtype(ids[0]), first_row, rows, width,
          -1 if padding_id is None else padding_id, scale, int(accumulate), table_ptr, api.nccl_dtype(table_grad),
          table_stride, api._dev_ptr(workspace), workspace.numel() * workspace.element_size(), _stream_of(table_grad, stream))


class PageCache:
    """A rank's cache of pages (dfcclPageCache): `pools` is a list of contiguous tensors [pages, ...] whose pages hold
    `page_tokens` tokens, and refcounts [pages], tables [sequences, pages per sequence] and lengths [sequences] are its
    bookkeeping, int32 tensors that the caller owns (PageCache.empty makes those of an empty cache).  report[0]:
    requests refused by the last extend or fork; report[1], report[2]: pages moved, pages live at the last compact."""

    def __init__(self, pools, page_tokens, refcounts, tables, lengths):
        pages = pools[0].shape[0]
        page_bytes = pools[0].numel() // max(1, pages) * pools[0].element_size()
        for p in pools:
            if p.shape[0] != pages or p.numel() * p.element_size() != pages * page_bytes:
                raise ValueError("the pools must agree in pages and bytes per page")
        for t in (refcounts, tables, lengths):
            if t.dtype != torch.int32:
                raise TypeError("the bookkeeping is held in int32 tensors")
        if refcounts.shape != (pages,) or tables.dim() != 2 or lengths.shape != (tables.shape[0],):
            raise ValueError("refcounts is [pages], tables [sequences, pages per sequence], lengths [sequences]")
        _same_device(refcounts, tables, lengths, *pools)
        self.lib = _lib.load()
        need = ctypes.c_size_t()
        api.check(self.lib.dfcclPageCacheWorkspace(pages, tables.shape[0], ctypes.byref(need)), "dfcclPageCacheWorkspace")
        self.pools, self.page_tokens = pools, page_tokens
        self.refcounts, self.tables, self.lengths = refcounts, tables, lengths
        self.report = torch.zeros(3, dtype=torch.int32, device=refcounts.device)
        self._workspace = torch.empty(need.value, dtype=torch.uint8, device=refcounts.device)
        self._pointers = (ctypes.c_void_p * len(pools))(*[api._dev_ptr(p).value for p in pools])
        self._struct = _lib.PageCacheStruct(
            ctypes.sizeof(_lib.PageCacheStruct), self._pointers, page_bytes, len(pools), pages, page_tokens, tables.shape[0],
            tables.shape[1], api._dev_ptr(refcounts), api._dev_ptr(tables), api._dev_ptr(lengths), api._dev_ptr(self.report),
            api._dev_ptr(self._workspace), need.value)
        self._ref = ctypes.byref(self._struct)

    @classmethod
    def empty(cls, pools, page_tokens, sequences, pages_per_sequence):
        """A cache whose pages are all free."""
        def ints(value, *shape):
            return torch.full(shape, value, dtype=torch.int32, device=pools[0].device)
        return cls(pools, page_tokens, ints(0, pools[0].shape[0]), ints(-1, sequences, pages_per_sequence),
                   ints(0, sequences))

    def _run(self, name, stream, *lists):
        for t in lists:
            if t.dtype != torch.int32:
                raise TypeError("lists of sequences, pages and lengths are int32 tensors")
            if t.numel() != lists[0].numel():
                raise ValueError("the lists must agree in length")
        _same_device(self.refcounts, *lists)
        args = [api._dev_ptr(t) for t in lists] + ([lists[0].numel()] if lists else [])
        _call(self.refcounts, getattr(self.lib, name), name, self._ref, *args, _stream_of(self.refcounts, stream))

    def copy(self, src_pages, dst_pages, source=None, stream=None):
        """Contents of the pages src_pages of `source` (default: this cache) into this cache's dst_pages, all pools."""
        if src_pages.dtype != torch.int32 or dst_pages.dtype != torch.int32:
            raise TypeError("lists of pages are int32 tensors")
        if src_pages.numel() != dst_pages.numel():
            raise ValueError("the lists must agree in length")
        source = self if source is None else source
        _same_device(self.refcounts, source.refcounts, src_pages, dst_pages)
        _call(self.refcounts, self.lib.dfcclPagesCopy, "dfcclPagesCopy", self._ref, source._ref, api._dev_ptr(src_pages),
              api._dev_ptr(dst_pages), src_pages.numel(), _stream_of(self.refcounts, stream))

    def extend(self, sequences, lengths, stream=None):
        """The sequences grow to these lengths; new entries get the lowest free pages."""
        self._run("dfcclPagesExtend", stream, sequences, lengths)

    def fork(self, parents, children, stream=None):
        """The children (empty) become copies of the parents: full pages shared, a last page that is not full copied."""
        self._run("dfcclPagesFork", stream, parents, children)

    def free(self, sequences, stream=None):
        """The sequences become empty and give up their pages."""
        self._run("dfcclPagesFree", stream, sequences)

    def compact(self, stream=None):
        """Moves pages until the live ones have the lowest numbers; counts and tables follow."""
        self._run("dfcclPagesCompact", stream)
