"""Pages of a cache that several sequences share: beside ``cache_append`` and ``cache_attention``, for a
program that continues one prompt several times (samples, beams) and lets sequences come and go.

They have no counterpart in the reference, which has no cache.  Beside the page table and the lengths
a program keeps ``holders``, how many entries of the table name each page; a page with 0 is free.

    cache_fork(pages, lengths, holders, parents, page)        # rows continue others, or end
    lengths += counts
    copies = cache_reserve(pages, lengths, holders, page, counts)   # pages for the new tokens
    cache_copy(k_cache, v_cache, k_scale, v_scale, copies)    # what shared pages held, for every layer
    cache_append(k, v, k_cache, v_cache, k_scale, v_scale, pages, lengths, counts)
    o = cache_attention(q, k_cache, v_cache, k_scale, v_scale, pages, lengths, None, scale, counts, shared)

No call waits for the GPU, so a step can be captured into a graph; what they write depends on their
arguments alone.  An entry of the table outside the cache's pages is no page (these calls write -1, but a
row that continues another has its entries as they are), and all of a row counts, also behind its last
token: a table starts filled with -1.  At most 2^30 pages.

Like the others they run through the native torch binding where it is built (operators
``enatten::cache_fork``, ...), else through ctypes.
"""
from __future__ import annotations

import torch

from . import _lib
from .ops import NATIVE_BINDING, _check, _require_gpu, _stream_of
from .sequence import _CACHE_DTYPES, _no_gradient, _share_memory, _tensors

_OPS = {name: getattr(torch.ops.enatten, name).default
        for name in ("cache_fork", "cache_reserve", "cache_copy", "cache_compact")} if NATIVE_BINDING else None


def _numbers(name, t, n, pages) -> None:
    if t.dim() != 1 or t.dtype != torch.int32 or (t.shape[0] < 1 if n is None else t.shape[0] != n):
        raise ValueError("%s must be int32 %s, got %s %s"
                         % (name, "[pages of the cache]" if n is None else "[B]", t.dtype, list(t.shape)))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    if t.device != pages.device:
        raise ValueError("all tensors must be on the same device")


def _validate_table(pages, holders, page) -> None:
    if pages.dim() != 2 or pages.dtype != torch.int32 or pages.numel() == 0:
        raise ValueError("pages must be int32 [B, columns], got %s %s" % (pages.dtype, list(pages.shape)))
    if pages.shape[1] > 1 and pages.stride(1) != 1:
        raise ValueError("pages needs unit stride on the columns")
    if pages.shape[0] > 1 and pages.stride(0) < pages.shape[1]:
        raise ValueError("the rows of pages must not overlap")
    if page < 16 or page > 1024 or page % 16:
        raise ValueError("pages must hold a multiple of 16 tokens up to 1024, got %d" % page)
    _numbers("holders", holders, None, pages)
    if max(pages.shape) > 0x7fffffff or holders.shape[0] > 1 << 30:
        raise ValueError("tensor too large")


def _page(page) -> int:
    if not isinstance(page, int) or isinstance(page, bool):
        raise TypeError("page must be an int")
    return page


def _written(*tensors) -> None:
    for t in tensors:
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)


def _fork_impl(pages, lengths, holders, parents, page) -> None:
    _validate_table(pages, holders, page)
    parents = parents.contiguous()
    _numbers("lengths", lengths, pages.shape[0], pages)
    _numbers("parents", parents, pages.shape[0], pages)
    _require_gpu(pages, "cache_fork")
    lib = _lib.load()
    with torch.cuda.device(pages.device):
        _check(lib.enatten_cache_fork(pages.data_ptr(), lengths.data_ptr(), holders.data_ptr(), parents.data_ptr(),
                                      *pages.shape, holders.shape[0], page, pages.stride(0), _stream_of(pages)))
    _written(pages, lengths, holders)


def _reserve_impl(pages, lengths, holders, page, counts, count):
    _validate_table(pages, holders, page)
    lengths, counts = lengths.contiguous(), None if counts is None else counts.contiguous()
    _numbers("lengths", lengths, pages.shape[0], pages)
    if counts is not None:
        _numbers("counts", counts, pages.shape[0], pages)
    if not 0 <= count <= 0x7fffffff:
        raise ValueError("counts must not be negative, got %d" % count)
    _require_gpu(pages, "cache_reserve")
    lib = _lib.load()
    copies = pages.new_empty((pages.shape[0], 3))
    with torch.cuda.device(pages.device):
        ws = torch.empty(lib.enatten_cache_reserve_workspace_bytes(*pages.shape, holders.shape[0]), dtype=torch.uint8,
                         device=pages.device)
        _check(lib.enatten_cache_reserve(
            pages.data_ptr(), lengths.data_ptr(), None if counts is None else counts.data_ptr(), count, holders.data_ptr(),
            copies.data_ptr(), ws.data_ptr(), *pages.shape, holders.shape[0], page, pages.stride(0), _stream_of(pages)))
    _written(pages, holders)
    return copies


def _compact_impl(pages, holders, page):
    _validate_table(pages, holders, page)
    _require_gpu(pages, "cache_compact")
    lib = _lib.load()
    copies = pages.new_empty((max(holders.shape[0] // 2, 1), 3))
    with torch.cuda.device(pages.device):
        ws = torch.empty(lib.enatten_cache_compact_workspace_bytes(holders.shape[0]), dtype=torch.uint8,
                         device=pages.device)
        _check(lib.enatten_cache_compact(pages.data_ptr(), holders.data_ptr(), copies.data_ptr(), ws.data_ptr(),
                                         *pages.shape, holders.shape[0], page, pages.stride(0), _stream_of(pages)))
    _written(pages, holders)
    return copies


def _copy_impl(k_cache, v_cache, k_scale, v_scale, copies) -> None:
    if k_cache.dim() not in (4, 5) or k_cache.shape != v_cache.shape or k_cache.numel() == 0:
        raise ValueError("k_cache and v_cache must be [pages, heads, tokens, head_dim], or that for some layers, got "
                         "%s, %s" % (tuple(k_cache.shape), tuple(v_cache.shape)))
    if k_cache.dtype not in _CACHE_DTYPES or v_cache.dtype != k_cache.dtype:
        raise ValueError("k_cache and v_cache must both be int8 or float8_e4m3fn, got %s, %s"
                         % (k_cache.dtype, v_cache.dtype))
    if k_cache.stride(-1) != 1 or v_cache.stride(-1) != 1:
        raise ValueError("the cache needs unit stride on the channels")
    for t in (k_scale, v_scale):
        if t.shape != k_cache.shape[:-2]:
            raise ValueError("k_scale and v_scale must be [pages, heads] = %s, got %s"
                             % (list(k_cache.shape[:-2]), list(t.shape)))
        if t.dtype != torch.float32:
            raise ValueError("k_scale and v_scale must be float32")
    if copies.dim() != 2 or copies.shape[1] != 3 or copies.dtype != torch.int32:
        raise ValueError("copies must be int32 [n, 3], got %s %s" % (copies.dtype, list(copies.shape)))
    written = (k_cache, v_cache, k_scale, v_scale)
    if any(t.device != k_cache.device for t in (*written, copies)):
        raise ValueError("all tensors must be on the same device")
    for t in written:
        if any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride())):
            raise RuntimeError("the cache must not share memory between its elements")
    if _share_memory(k_cache, v_cache) or _share_memory(k_scale, v_scale):
        raise ValueError("keys and values must not share a cache")
    lead = k_cache.dim() - 4
    layers = k_cache.shape[0] if lead else 1
    num, heads, page, D = k_cache.shape[lead:]
    if num > 0x7fffffff or max(heads, layers) > 1 << 20 or copies.shape[0] > 0x7fffffff or page > 1024 or D > 256:
        raise ValueError("tensor too large, more than 1024 tokens in a page, or a head_dim above 256")
    _require_gpu(k_cache, "cache_copy")
    _no_gradient("cache_copy", *written)
    lib = _lib.load()
    copies = copies.contiguous()
    one = [t if lead else t.unsqueeze(0) for t in written]
    with torch.cuda.device(k_cache.device):
        _check(lib.enatten_cache_copy(*(t.data_ptr() for t in written), copies.data_ptr(), copies.shape[0], layers, heads,
                                      D, num, page, _lib.strides(one[0], 4), _lib.strides(one[1], 4),
                                      _lib.strides(one[2], 3), _lib.strides(one[3], 3), _stream_of(k_cache)))
    _written(*written)


def cache_fork(pages, lengths, holders, parents, page) -> None:
    """Rows of the page table become continuations of other rows, in place.

    ``pages``  int32 ``[B, columns]``; ``lengths``  int32 ``[B]``, tokens of each row; ``holders``  int32, one
        for each page of the cache: how many entries of the table name it; ``page``, tokens of a page.
    ``parents``  int32 ``[B]``: row b becomes what row ``parents[b]`` was before the call, its length and the
        pages of its tokens, which both hold then; -1 leaves the row empty.  Its own number, and any
        outside -1 .. B - 1, leaves the row as it is, pages behind its last token included.

    Pages that no entry names any more are free.  At most 4096 rows.  Values at the front that several rows
    share may be read by all of them; before a row writes into one, :func:`cache_reserve` gives it its own.
    """
    _tensors(pages=pages, lengths=lengths, holders=holders, parents=parents)
    call = _OPS["cache_fork"] if NATIVE_BINDING else _fork_impl
    call(pages, lengths, holders, parents, _page(page))


def cache_reserve(pages, lengths, holders, page, counts=1):
    """Pages for the new tokens of every row, in place: ``copies``, int32 ``[B, 3]``, for :func:`cache_copy`.

    ``pages, holders, page``  those of :func:`cache_fork`; ``lengths``  int32 ``[B]``, the new tokens
        included, as :func:`cache_append` takes them; ``counts``  int32 ``[B]``, how many of these are new,
        or one int for all rows.

    An entry that new tokens go to and that is no page gets the lowest free page, rows and columns in
    their order.  Where the first of them holds older tokens and other rows hold its page, the row gets a
    free page instead, and its line of ``copies`` is (page left, page got, older tokens), else (-1, -1, 0);
    if all that hold a page leave it in one call, the last row keeps it.
    A page without older tokens that others hold even then, as where a row's length went back behind tokens
    that it shares, is replaced without a copy; if nobody holds it any more it is free after the call.

    Where no page is free the entry becomes -1: :func:`cache_append` leaves its tokens out and
    :func:`cache_attention` gives NaN.  An entry that older tokens belong to and that is no page stays none.
    Rows whose numbers do not fit together are left out.  At most 4096 rows.
    """
    _tensors(pages=pages, lengths=lengths, holders=holders)
    count = 0
    if isinstance(counts, int) and not isinstance(counts, bool):
        counts, count = None, counts
    else:
        _tensors(counts=counts)
    call = _OPS["cache_reserve"] if NATIVE_BINDING else _reserve_impl
    return call(pages, lengths, holders, _page(page), counts, count)


def cache_copy(k_cache, v_cache, k_scale, v_scale, copies) -> None:
    """Copy pages of a cache, in place: for each (source, target, tokens) of ``copies``, int32 ``[n, 3]``,
    the codes of the first tokens of every head, and its scales.

    The cache is that of :func:`cache_append`, or a pool of several layers that have one page table:
    ``k_cache, v_cache [layers, pages, heads, page, d]``, ``k_scale, v_scale [layers, pages, heads]``.
    Lines with a page outside the cache, or with the same page twice, are passed over; more tokens than a
    page holds are all of it.  A page may be the target of one line only, and not also a source.  No gradient.
    """
    _tensors(k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, copies=copies)
    call = _OPS["cache_copy"] if NATIVE_BINDING else _copy_impl
    call(k_cache, v_cache, k_scale, v_scale, copies)


def cache_compact(pages, holders, page):
    """Move the held pages to the low end of the cache, table and holders in place: ``copies``, int32
    ``[max(pages of the cache // 2, 1), 3]``, for :func:`cache_copy`.

    With n held pages, those from n on move to the free ones below n, both in their order, after which
    the pages from n on are free.  ``copies`` has (source, target, page) for each move, then (-1, -1, 0).  A page
    that a program holds by ``holders`` alone moves too: it finds it in ``copies``.  At most 4096 rows.
    """
    _tensors(pages=pages, holders=holders)
    call = _OPS["cache_compact"] if NATIVE_BINDING else _compact_impl
    return call(pages, holders, _page(page))
