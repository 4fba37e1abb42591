"""The pages of a key/value cache: who holds them, and their copies.

``tables`` int32 [seqs][width] names each sequence's pages (-1: none), ``lengths``
int32 [seqs] counts its tokens and ``refs`` int32 [pages] the table entries that name
a page (0: free).  All three are on the GPU and change in place; new pages are the
free ones of the lowest index, in the order of the call's list.  A pool is a
contiguous tensor [...planes][pages][kv_heads][page_size][dim], one plane per layer
and keys or values.

The lists (int32 on the GPU, each sequence at most once) are checked there: a call
that is refused changes nothing and leaves a code in ``status`` (int32 [1], if given,
while it is 0), which :func:`page_check` turns into an error.  Streams are as in
:mod:`praghip.attention`.
"""
from __future__ import annotations

import math
import struct

from . import attention
from ._lib import E_STATE, PraghipError, check, lib, shape_error
from .attention import _stream, _type_error, _work

_REFUSED = {1: "E_PAGES_SEQUENCE", 2: "E_PAGES_CAPACITY", 3: "E_PAGES_EXHAUSTED"}
_TABLE = struct.Struct("Pq2Q2P2QP").pack  # praghip_page_table
_POOL = struct.Struct("Pq3Q").pack        # praghip_page_pool


def _table(tables, lengths, refs, page_size: int, status, index: int) -> bytes:
    if attention._int32 is None:
        attention._load()
    int32 = attention._int32
    if not tables.dtype is refs.dtype is int32 or not tables.get_device() == refs.get_device() == index >= 0:
        raise _type_error("E_PAGES_INTS")
    shape, ts, pages = tables.shape, tables.stride(), refs.shape
    if len(shape) != 2 or (ts[1] != 1 and shape[1] > 1) or len(pages) != 1 or \
            (pages[0] > 1 and refs.stride(0) != 1) or page_size < 0:
        raise shape_error("E_PAGES_SHAPE")
    # (a compaction has no use for lengths: any address stands for them)
    held = refs.data_ptr() if lengths is None else _list(lengths, shape[0], index)
    return _TABLE(tables.data_ptr(), ts[0], shape[1], shape[0], held, refs.data_ptr(), pages[0], page_size,
                  0 if status is None else _list(status, 1, index))


def _pool(pool, index: int) -> bytes:
    shape = pool.shape
    if len(shape) < 4 or not pool.is_contiguous():
        raise shape_error("E_PAGES_POOL")
    if pool.get_device() != index or index < 0:
        raise _type_error("E_PAGES_DEVICE")
    page = math.prod(shape[-3:]) * pool.element_size()
    return _POOL(pool.data_ptr(), shape[-4] * page, page, math.prod(shape[:-4]), shape[-4])


def _list(t, n: int, index: int) -> int:
    if attention._int32 is None:
        attention._load()
    if t.dtype is not attention._int32 or t.get_device() != index or index < 0:
        raise _type_error("E_PAGES_INTS")
    if t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        raise shape_error("E_PAGES_SHAPE")
    return t.data_ptr()


def _length(t) -> int:
    """Entries of a call's list."""
    if len(t.shape) != 1:
        raise shape_error("E_PAGES_SHAPE")
    return t.shape[0]


def page_reserve(tables, lengths, refs, page_size: int, sequences, counts, status=None, stream=None) -> None:
    """counts[i] more tokens for sequences[i]: its new pages, and its length."""
    index = tables.get_device()
    t = _table(tables, lengths, refs, page_size, status, index)
    n = _length(sequences)
    check(lib().praghip_page_reserve(index, t, _list(sequences, n, index), _list(counts, n, index), n,
                                     _stream(index, stream)))


def page_free(tables, lengths, refs, sequences, status=None, stream=None) -> None:
    """Empties sequences: their pages lose a reference, their rows become -1, their lengths 0."""
    index = tables.get_device()
    t = _table(tables, lengths, refs, 1, status, index)
    n = _length(sequences)
    check(lib().praghip_page_free(index, t, _list(sequences, n, index), n, _stream(index, stream)))


def page_trim(tables, lengths, refs, page_size: int, sequences, window: int, sinks: int = 0, status=None,
              stream=None) -> None:
    """Gives back the pages that no token after a sequence's last one sees through this window and these sinks."""
    index = tables.get_device()
    t = _table(tables, lengths, refs, page_size, status, index)
    if window < 0 or sinks < 0:
        raise shape_error("E_PAGES_WINDOW")
    n = _length(sequences)
    check(lib().praghip_page_trim(index, t, _list(sequences, n, index), n, window, sinks, _stream(index, stream)))


def page_fork(pool, tables, lengths, refs, parents, children, status=None, stream=None) -> None:
    """children[i], an empty sequence, becomes a copy of parents[i] (which may have several).

    Full pages are shared; a last page that is not full is copied in every plane of
    the pool to a new page.
    """
    index = tables.get_device()
    p = _pool(pool, index)
    t = _table(tables, lengths, refs, pool.shape[-2], status, index)
    n = _length(parents)
    of, to = _list(parents, n, index), _list(children, n, index)
    if n:
        L = lib()
        size = L.praghip_page_fork_workspace(n)
        work = _work(size, tables, stream)
        check(L.praghip_page_fork(index, t, p, of, to, n, work.data_ptr(), size,
                                  _stream(index, stream)))


def page_compact(pool, tables, refs, stream=None) -> None:
    """Moves pages so that the held ones are 0 .. count - 1: held pages above move into
    the holes below, both in rising order, and the tables follow."""
    index = tables.get_device()
    p = _pool(pool, index)
    t, pages = _table(tables, None, refs, pool.shape[-2], None, index), refs.shape[0]
    L = lib()
    size = L.praghip_page_compact_workspace(pages)
    work = _work(size, tables, stream)
    check(L.praghip_page_compact(index, t, p, work.data_ptr(), size,
                                 _stream(index, stream)))


def page_copy(pool, sources, targets, stream=None) -> None:
    """Page sources[i] of every plane over page targets[i]; indexes that are no pages are
    skipped.  No page may be both a source and a target, or a target twice."""
    index = pool.get_device()
    p = _pool(pool, index)
    n = _length(sources)
    check(lib().praghip_page_copy(index, p, _list(sources, n, index), _list(targets, n, index), n,
                                  _stream(index, stream)))


def page_check(status) -> None:
    """Waits for the GPU; raises where a call was refused since `status` was 0, and clears it."""
    code = int(status.item())
    if code:
        status.zero_()
        raise PraghipError(E_STATE, _REFUSED.get(code, f"E_PAGES_{code}"))
