"""Attention over a paged key/value cache: one new token per sequence
(:func:`paged_decode`, and :func:`paged_shared` where sequences share prefixes) or many
(:func:`paged_prompt`).

The reference's attention is a two-party protocol, and its float Qwen3 a transformers
model; these serve such a model in the clear beside the protocol.  Tensors are on one GPU; calls
are asynchronous on ``stream`` (the tensors' device's current stream by default).

On another stream than the current one a call's workspace and the tensors that it
returns come from that stream's memory, so they wait for nothing.  The caller orders
the rest: ``stream`` behind the work that makes the call's inputs, the current stream
behind ``stream`` before it reads the result, and inputs kept until the call is done.

The calls have no backward pass: one whose inputs require gradients is refused, unless
gradients are off (``torch.no_grad``).
"""
from __future__ import annotations

import struct

from ._lib import E_ARGUMENT, PraghipError, check, lib, shape_error

# A call's checks and packing are a few microseconds, as long as a small kernel: they
# read each attribute of a tensor once, and structures go to the library as packed bytes.
_torch = _int32 = _uint8 = _float32 = _current = None
_kinds: dict = {}                     # torch dtype -> type code
_CACHE = struct.Struct("2P6q4Qi4xPqQPQ")  # praghip_cache
_two = struct.Struct("2q").pack


def _load():
    global _torch, _int32, _uint8, _float32, _current
    import torch
    _torch, _int32, _uint8, _float32 = torch, torch.int32, torch.uint8, torch.float32
    _kinds.update({torch.bfloat16: 0, torch.float16: 1})
    _current = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
        (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _stream(index: int, stream):
    """hipStream_t of a call on device `index`: the given stream, or the device's current one."""
    if _current is None:
        _load()
    return (_current(index) if stream is None else stream.cuda_stream) or None


def _type_error(text: str) -> PraghipError:
    return PraghipError(E_ARGUMENT, text)


def _no_gradients(text: str) -> None:
    """A call of inputs that require gradients: its output would pass for a constant."""
    if _torch.is_grad_enabled():
        raise _type_error(text)


def _kind(t, text: str) -> int:
    code = _kinds.get(t.dtype)
    if code is None:
        _load()
        code = _kinds.get(t.dtype)
        if code is None:
            raise _type_error(text)
    return code


def _cache(k, v, tables, lengths, like, kind: int, index: int):
    """(praghip_cache as bytes, pages' shape, sequences) of one layer's pages, tables and lengths."""
    if not k.get_device() == v.get_device() == index >= 0:
        raise _type_error("E_ATTENTION_DEVICE")
    if not k.dtype is v.dtype is like.dtype:
        raise _type_error("E_ATTENTION_TYPE")
    if not tables.dtype is lengths.dtype is _int32 or not tables.get_device() == lengths.get_device() == index:
        raise _type_error("E_ATTENTION_INTS")
    shape, held, named = k.shape, lengths.shape, tables.shape
    ks, vs, ts = k.stride(), v.stride(), tables.stride()
    if len(shape) != 4 or v.shape != shape or ks[3] != 1 or vs[3] != 1 or len(held) != 1 or len(named) != 2 or \
            named[0] != held[0] or (ts[1] != 1 and named[1] > 1) or (held[0] > 1 and lengths.stride(0) != 1):
        raise shape_error("E_ATTENTION_SHAPE")
    return _CACHE.pack(k.data_ptr(), v.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], *shape, kind,
                       tables.data_ptr(), ts[0], named[1], lengths.data_ptr(), held[0]), shape, held[0]


def _starts(t, seqs: int, index: int) -> int:
    if t.dtype is not _int32 or t.get_device() != index:
        raise _type_error("E_ATTENTION_INTS")
    if t.shape != (seqs + 1,) or (seqs and t.stride(0) != 1):
        raise shape_error("E_ATTENTION_SHAPE")
    return t.data_ptr()


def _there(stream, make, *args, **kw):
    """make(...), a tensor that a call on another stream writes, from the memory of that stream:
    a block of the current one's may have been freed there with work under way that uses it."""
    with _torch.cuda.stream(stream):
        return make(*args, **kw)


def _result(stream, index: int, make, *args, **kw):
    """The same for what a call returns: its block goes back once the current stream, where it
    is read, is done with it too."""
    t = _there(stream, make, *args, **kw)
    t.record_stream(_torch.cuda.current_stream(index))
    return t


def _lse(q, shape, index: int, stream):
    shape, kind = shape[:2], dict(dtype=_torch.float32, device=q.device)
    return _torch.empty(shape, **kind) if stream is None else _result(stream, index, _torch.empty, shape, **kind)


def _output(q, shape, out, index: int, stream):
    if out is None:
        return _torch.empty_like(q) if stream is None else _result(stream, index, _torch.empty_like, q)
    if out.shape != shape or out.dtype is not q.dtype or out.get_device() != index or \
            (shape[2] > 1 and out.stride(2) != 1):
        raise shape_error("E_ATTENTION_OUT")
    return out


def _work(size: int, like, stream):
    """Workspace of one call, which `stream` alone uses."""
    if stream is None:
        return _torch.empty(size, dtype=_uint8, device=like.device)
    return _there(stream, _torch.empty, size, dtype=_uint8, device=like.device)


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
    kind, index, shape, qs = _kind(q, "E_ATTENTION_TYPE"), q.get_device(), q.shape, q.stride()
    cache, pages, seqs = _cache(k_pages, v_pages, tables, lengths, q, kind, index)
    if len(shape) != 3 or shape[0] != seqs or shape[2] != pages[3] or (qs[2] != 1 and shape[2] > 1) or not pages[1] or \
            shape[1] % pages[1] or window < 0 or sinks < 0 or max_length < 0:
        raise shape_error("E_ATTENTION_SHAPE")
    if q.requires_grad or k_pages.requires_grad or v_pages.requires_grad:
        _no_gradients("E_ATTENTION_GRADIENT")
    out = _output(q, shape, out, index, stream)
    sums = _lse(q, shape, index, stream) if lse else None
    if seqs:
        L, heads, to = lib(), shape[1], out.stride()
        size = L.praghip_paged_decode_workspace(cache, heads, max_length)
        work = _work(size, q, stream)
        check(L.praghip_paged_decode(index, cache, q.data_ptr(), _two(qs[0], qs[1]), heads, out.data_ptr(),
                                     _two(to[0], to[1]), sums.data_ptr() if lse else None,
                                     shape[2] ** -0.5 if scale is None else scale, window, sinks, max_length,
                                     work.data_ptr(), size, _stream(index, stream)))
    return (out, sums) if lse else out


def paged_shared(q, k_pages, v_pages, tables, lengths, groups, shared, *, scale: float | None = None, max_length: int = 0,
                 lse: bool = False, out=None, stream=None):
    """:func:`paged_decode` of sequences that share prefixes, each read once for its group.

    groups int32 [count + 1], not falling: sequences groups[g] .. groups[g + 1] - 1 have their
    first shared[g] positions (int32 [count]) in common, as :func:`page_fork` leaves a parent
    and its children.  Those are read from the pages of the group's first sequence, as far as
    that one is long; a sequence that is shorter, or in no group, reads its own.  There is no
    window: one that moves on leaves the prefix.  The rest is as in :func:`paged_decode`.
    """
    kind, index, shape, qs = _kind(q, "E_ATTENTION_TYPE"), q.get_device(), q.shape, q.stride()
    cache, pages, seqs = _cache(k_pages, v_pages, tables, lengths, q, kind, index)
    if len(shape) != 3 or shape[0] != seqs or shape[2] != pages[3] or (qs[2] != 1 and shape[2] > 1) or not pages[1] or \
            shape[1] % pages[1] or max_length < 0 or len(shared.shape) != 1:
        raise shape_error("E_ATTENTION_SHAPE")
    count = shared.shape[0]
    first = _starts(groups, count, index)
    if shared.dtype is not _int32 or shared.get_device() != index:
        raise _type_error("E_ATTENTION_INTS")
    if count > 1 and shared.stride(0) != 1:
        raise shape_error("E_ATTENTION_SHAPE")
    if q.requires_grad or k_pages.requires_grad or v_pages.requires_grad:
        _no_gradients("E_ATTENTION_GRADIENT")
    out = _output(q, shape, out, index, stream)
    sums = _lse(q, shape, index, stream) if lse else None
    if seqs:
        L, heads, to = lib(), shape[1], out.stride()
        size = L.praghip_paged_shared_workspace(cache, heads, count, max_length)
        work = _work(size, q, stream)
        check(L.praghip_paged_shared(index, cache, q.data_ptr(), _two(qs[0], qs[1]), heads, first, shared.data_ptr(), count,
                                     out.data_ptr(), _two(to[0], to[1]), sums.data_ptr() if lse else None,
                                     shape[2] ** -0.5 if scale is None else scale, max_length, work.data_ptr(), size,
                                     _stream(index, stream)))
    return (out, sums) if lse else out


def paged_prompt(q, k_pages, v_pages, tables, lengths, starts, max_rows: int, *, scale: float | None = None,
                 window: int = 0, sinks: int = 0, max_length: int = 0, lse: bool = False, out=None, stream=None):
    """Causal attention of each sequence's newest tokens over its cached keys.

    q [tokens][heads][dim]: rows starts[s] .. starts[s + 1] - 1 (starts int32
    [seqs + 1]) are the newest tokens of sequence s, the last at position
    lengths[s] - 1; the cache holds their keys and values already.  max_rows is at
    least the longest of these stretches (rows beyond it may be left unwritten, as rows
    of no stretch are).  Token p
    sees key j where j <= p and, with a window, j > p - window or j < sinks.  The rest
    is as in :func:`paged_decode`.
    """
    kind, index, shape, qs = _kind(q, "E_ATTENTION_TYPE"), q.get_device(), q.shape, q.stride()
    cache, pages, seqs = _cache(k_pages, v_pages, tables, lengths, q, kind, index)
    if len(shape) != 3 or shape[2] != pages[3] or (qs[2] != 1 and shape[2] > 1) or not pages[1] or \
            shape[1] % pages[1] or window < 0 or sinks < 0 or max_length < 0 or max_rows < 0:
        raise shape_error("E_ATTENTION_SHAPE")
    first = _starts(starts, seqs, index)
    if q.requires_grad or k_pages.requires_grad or v_pages.requires_grad:
        _no_gradients("E_ATTENTION_GRADIENT")
    out = _output(q, shape, out, index, stream)
    sums = _lse(q, shape, index, stream) if lse else None
    tokens, heads = shape[0], shape[1]
    if tokens and seqs:
        L, to = lib(), out.stride()
        max_rows = min(max_rows, tokens)
        size = L.praghip_paged_prompt_workspace(cache, heads, max_rows, window, sinks, max_length)
        work = _work(size, q, stream) if size else None
        check(L.praghip_paged_prompt(index, cache, q.data_ptr(), _two(qs[0], qs[1]), heads, first, tokens, max_rows,
                                     out.data_ptr(), _two(to[0], to[1]), sums.data_ptr() if lse else None,
                                     shape[2] ** -0.5 if scale is None else scale, window, sinks, max_length,
                                     work.data_ptr() if size else None, size, _stream(index, stream)))
    return (out, sums) if lse else out


def page_write(k, v, k_pages, v_pages, tables, lengths, starts, stream=None) -> None:
    """Writes new tokens' keys and values into the cache.

    k, v [tokens][kv_heads][dim]: rows starts[s] .. starts[s + 1] - 1 are the newest
    tokens of sequence s, the last at position lengths[s] - 1 (so the lengths, and the
    pages, are those after :func:`page_reserve`).  Tokens without a page are dropped.
    """
    kind, index, shape = _kind(k, "E_ATTENTION_TYPE"), k.get_device(), k.shape
    cache, pages, seqs = _cache(k_pages, v_pages, tables, lengths, k, kind, index)
    if v.dtype is not k.dtype or v.get_device() != index:
        raise _type_error("E_ATTENTION_TYPE")
    ks, vs = k.stride(), v.stride()
    if len(shape) != 3 or v.shape != shape or shape[1] != pages[1] or shape[2] != pages[3] or ks[2] != 1 or vs[2] != 1:
        raise shape_error("E_ATTENTION_SHAPE")
    if k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad:
        _no_gradients("E_ATTENTION_GRADIENT")
    check(lib().praghip_page_write(index, cache, k.data_ptr(), _two(ks[0], ks[1]), v.data_ptr(), _two(vs[0], vs[1]),
                                   _starts(starts, seqs, index), shape[0], _stream(index, stream)))
