"""Attention over a paged key/value cache: one new token per sequence
(:func:`paged_decode`) or many (:func:`paged_prompt`).

The reference's attention is a two-party protocol; these serve a model in the
clear beside it, and have no counterpart there.  Tensors are on one GPU; calls
are asynchronous on ``stream`` (the tensors' device's current stream by default).
"""
from __future__ import annotations

import ctypes
import functools

from ._lib import E_ARGUMENT, Cache, PraghipError, check, lib, shape_error


@functools.lru_cache(maxsize=None)
def _types():
    import torch
    return {torch.bfloat16: 0, torch.float16: 1}


@functools.lru_cache(maxsize=None)
def _torch():
    import torch
    return torch


@functools.lru_cache(maxsize=None)
def _raw_stream():
    torch = _torch()
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
    return raw or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _stream(index: int, stream):
    """hipStream_t of a call on device `index`: the given stream, or the device's current one."""
    return (_raw_stream()(index) if stream is None else stream.cuda_stream) or None


def _type_error(text: str) -> PraghipError:
    return PraghipError(E_ARGUMENT, text)


def _ints(t, shape, index: int):
    """Address of an int32 tensor of this shape (None: any size) with contiguous rows."""
    if t.dtype is not _torch().int32 or t.get_device() != index:
        raise _type_error("E_ATTENTION_INTS")
    if t.dim() != len(shape) or any(n is not None and n != m for n, m in zip(shape, t.shape)) or \
            (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise shape_error("E_ATTENTION_SHAPE")
    return t.data_ptr()


def _cache(k, v, tables, lengths, type_of, index: int) -> Cache:
    if k.get_device() != index or v.get_device() != index or index < 0:
        raise _type_error("E_ATTENTION_DEVICE")
    if k.dtype is not type_of or v.dtype is not type_of:
        raise _type_error("E_ATTENTION_TYPE")
    pages, kv, size, dim = k.shape
    ks, vs = k.stride(), v.stride()
    if v.shape != k.shape or ks[3] != 1 or vs[3] != 1:
        raise shape_error("E_ATTENTION_SHAPE")
    seqs = lengths.shape[0]
    at = _ints(tables, (seqs, None), index)
    held = _ints(lengths, (seqs,), index)
    return Cache(k.data_ptr(), v.data_ptr(), ks[:3], vs[:3], pages, kv, size, dim, _types()[type_of], at,
                 tables.stride(0), tables.shape[1], held, seqs)


def _outputs(q, out, lse):
    torch = _torch()
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype is not q.dtype or out.get_device() != q.get_device() or \
            (out.shape[2] > 1 and out.stride(2) != 1):
        raise shape_error("E_ATTENTION_OUT")
    return out, torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if lse else None


def _queries(q):
    if q.dtype not in _types():
        raise _type_error("E_ATTENTION_TYPE")
    if q.dim() != 3 or (q.shape[2] > 1 and q.stride(2) != 1):
        raise shape_error("E_ATTENTION_SHAPE")


_Two = ctypes.c_int64 * 2


def _work(size: int, q, stream):
    """Workspace of one call; torch's allocator keeps it until `stream` is done with it."""
    work = _torch().empty(size, dtype=_torch().uint8, device=q.device)
    if stream is not None:
        work.record_stream(stream)
    return work


def paged_decode(q, k_pages, v_pages, tables, lengths, *, scale: float | None = None, window: int = 0, sinks: int = 0,
                 max_length: int = 0, lse: bool = False, out=None, stream=None):
    """Attention of the newest token of every sequence over its cached keys.

    q [seqs][heads][dim] bfloat16 or float16; k_pages, v_pages [pages][kv_heads]
    [page_size][dim] of the same type, any strides that are multiples of 8 with the
    last dim contiguous; tables int32 [seqs][width] names each sequence's pages (an
    entry outside 0 .. pages - 1 is no page), lengths int32 [seqs] counts its tokens,
    the newest among them.  heads is a multiple of kv_heads; dim a multiple of 8 up
    to 256; page_size a power of two of 16 or more.

    scale: of q.k, 1 / sqrt(dim) by default.  window > 0: only the last `window`
    tokens and the first `sinks` are seen.  max_length: a bound of the lengths, which
    sizes the launch and no result.  Returns out [seqs][heads][dim], and with lse the
    logarithm of each softmax's sum, float32 [seqs][heads]; a sequence that sees
    nothing gets zeros and -inf.
    """
    _queries(q)
    index = q.get_device()
    cache = _cache(k_pages, v_pages, tables, lengths, q.dtype, index)
    seqs, heads, dim = q.shape
    if cache.seqs != seqs or cache.head_dim != dim or not cache.kv_heads or heads % cache.kv_heads or window < 0 or \
            sinks < 0 or max_length < 0:
        raise shape_error("E_ATTENTION_SHAPE")
    out, sums = _outputs(q, out, lse)
    if seqs:
        L, c = lib(), ctypes.byref(cache)
        size = L.praghip_paged_decode_workspace(c, heads, max_length)
        work = _work(size, q, stream)
        check(L.praghip_paged_decode(index, c, q.data_ptr(), _Two(q.stride(0), q.stride(1)), heads, out.data_ptr(),
                                     _Two(out.stride(0), out.stride(1)), sums.data_ptr() if lse else None,
                                     dim ** -0.5 if scale is None else scale, window, sinks, max_length,
                                     work.data_ptr(), size, _stream(index, stream)))
    return (out, sums) if lse else out


def paged_prompt(q, k_pages, v_pages, tables, lengths, starts, max_rows: int, *, scale: float | None = None,
                 window: int = 0, sinks: int = 0, max_length: int = 0, lse: bool = False, out=None, stream=None):
    """Causal attention of each sequence's newest tokens over its cached keys.

    q [tokens][heads][dim]: rows starts[s] .. starts[s + 1] - 1 (starts int32
    [seqs + 1]) are the newest tokens of sequence s, the last at position
    lengths[s] - 1; the cache holds their keys and values already.  max_rows is at
    least the longest of these stretches (rows beyond it are not computed).  Token p
    sees key j where j <= p and, with a window, j > p - window or j < sinks.  The rest
    is as in :func:`paged_decode`.
    """
    _queries(q)
    index = q.get_device()
    cache = _cache(k_pages, v_pages, tables, lengths, q.dtype, index)
    tokens, heads, dim = q.shape
    if cache.head_dim != dim or not cache.kv_heads or heads % cache.kv_heads or window < 0 or sinks < 0 or \
            max_length < 0 or max_rows < 0:
        raise shape_error("E_ATTENTION_SHAPE")
    first = _ints(starts, (cache.seqs + 1,), index)
    out, sums = _outputs(q, out, lse)
    if tokens and cache.seqs:
        L, c = lib(), ctypes.byref(cache)
        max_rows = min(max_rows, tokens)
        size = L.praghip_paged_prompt_workspace(c, heads, max_rows, window, sinks, max_length)
        work = _work(size, q, stream) if size else None
        check(L.praghip_paged_prompt(index, c, q.data_ptr(), _Two(q.stride(0), q.stride(1)), heads, first, tokens,
                                     max_rows, out.data_ptr(), _Two(out.stride(0), out.stride(1)),
                                     sums.data_ptr() if lse else None, dim ** -0.5 if scale is None else scale, window,
                                     sinks, max_length, work.data_ptr() if size else None, size,
                                     _stream(index, stream)))
    return (out, sums) if lse else out


def page_write(k, v, k_pages, v_pages, tables, lengths, starts, stream=None) -> None:
    """Writes new tokens' keys and values into the cache.

    k, v [tokens][kv_heads][dim]: rows starts[s] .. starts[s + 1] - 1 are the newest
    tokens of sequence s, the last at position lengths[s] - 1 (so the lengths, and the
    pages, are those after :func:`page_reserve`).  Tokens without a page are dropped.
    """
    if k.dtype not in _types():
        raise _type_error("E_ATTENTION_TYPE")
    index = k.get_device()
    cache = _cache(k_pages, v_pages, tables, lengths, k.dtype, index)
    if k.dim() != 3 or v.shape != k.shape or k.shape[1] != cache.kv_heads or k.shape[2] != cache.head_dim or \
            k.stride(2) != 1 or v.stride(2) != 1:
        raise shape_error("E_ATTENTION_SHAPE")
    if v.dtype is not k.dtype or v.get_device() != index:
        raise _type_error("E_ATTENTION_TYPE")
    first = _ints(starts, (cache.seqs + 1,), index)
    check(lib().praghip_page_write(index, ctypes.byref(cache), k.data_ptr(), _Two(k.stride(0), k.stride(1)),
                                   v.data_ptr(), _Two(v.stride(0), v.stride(1)), first, k.shape[0],
                                   _stream(index, stream)))
