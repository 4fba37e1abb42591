"""New tokens of a step into a paged cache, with the norms and rotations that stand between
the projection and the attention (streams and gradients as in :mod:`praghip.attention`)."""
from __future__ import annotations

import math
import struct

from . import attention
from ._lib import check, lib, shape_error
from .attention import _cache, _kind, _no_gradients, _output, _starts, _stream, _type_error

_APPEND = struct.Struct("3P6qP2q4P2q4Qfi").pack  # praghip_append


def rotary_table(positions: int, dim: int, *, theta: float = 1e6, factor: float = 1.0, original: int = 0,
                 fast: float = 32.0, slow: float = 1.0, magnitude: float = 1.0, device="cuda"):
    """(cos, sin), float32 [positions][dim // 2], of the angles p theta^(-2 i / dim), times `magnitude`.

    For contexts `factor` times as long as those a model was trained on: with original 0 every
    frequency is divided by the factor; with the number of tokens that the model was trained on,
    the frequencies that turn `fast` times or more within them stay, those that turn `slow`
    times or less are divided, and the share between falls linearly with the number of turns'
    logarithm (YaRN's interpolation by parts, arXiv 2309.00071, whose scores are also scaled:
    magnitude 0.1 ln(factor) + 1).  Angles are 64-bit, so that far positions are exact.
    """
    import torch
    if positions < 0 or dim < 0 or dim % 2 or original < 0 or not theta > 0 or not factor > 0 or \
            (original and not (0 < slow < fast and theta > 1)):
        raise shape_error("E_ROTARY_SHAPE")
    half = dim // 2
    i = torch.arange(half, dtype=torch.float64, device=device)
    frequency = theta ** (-i / max(half, 1))
    if original:
        # the pair that turns n times within `original` tokens
        def pair(n):
            return half * math.log(original / (2 * math.pi * n)) / math.log(theta)
        low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
        divided = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        frequency = frequency * (1 - divided) + frequency / factor * divided
    else:
        frequency = frequency / factor
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * frequency
    return (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()


def page_append(q, k, v, k_pages, v_pages, tables, lengths, starts, cos, sin, *, q_norm=None, k_norm=None,
                eps: float = 1e-6, interleaved: bool = False, out=None, stream=None):
    """Norms and rotates new tokens' queries and keys, and writes the keys and values into the cache.

    q [tokens][heads][dim], k and v [tokens][kv_heads][dim] of one type, any strides that are
    multiples of 8 with the last dim contiguous (views of a joint projection, say); the cache,
    lengths and starts as in :func:`page_write`.  q_norm, k_norm [dim] of the same type: the
    weights of a root-mean-square norm of each head, or None.  cos, sin float32
    [positions][half] (:func:`rotary_table`): the rotation of the first 2 half values of a head
    by its token's position, of pairs half apart, or of neighbours where `interleaved`; they
    hold every position that the tables have room for.  Returns the queries (in ``out``, which
    may be q).  Sums and products are 32-bit, rounded once.
    """
    kind, index, shape = _kind(q, "E_ATTENTION_TYPE"), q.get_device(), q.shape
    cache, pages, seqs = _cache(k_pages, v_pages, tables, lengths, q, kind, index)
    type = q.dtype
    if not k.dtype is v.dtype is type:
        raise _type_error("E_ATTENTION_TYPE")
    if not k.get_device() == v.get_device() == index:
        raise _type_error("E_ATTENTION_DEVICE")
    new, qs, ks, vs = k.shape, q.stride(), k.stride(), v.stride()
    if len(shape) != 3 or len(new) != 3 or v.shape != new or new[0] != shape[0] or new[1] != pages[1] or \
            not shape[2] == new[2] == pages[3] or qs[2] != 1 or ks[2] != 1 or vs[2] != 1 or not shape[1]:
        raise shape_error("E_ATTENTION_SHAPE")
    wide, far = attention._float32, cos.shape
    if not cos.dtype is sin.dtype is wide:
        raise _type_error("E_ROTARY_TYPE")
    if not cos.get_device() == sin.get_device() == index:
        raise _type_error("E_ROTARY_DEVICE")
    if len(far) != 2 or sin.shape != far or (far[1] > 1 and not cos.stride(1) == sin.stride(1) == 1):
        raise shape_error("E_ROTARY_SHAPE")
    grad = q.requires_grad or k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad or \
        cos.requires_grad or sin.requires_grad
    norms = []
    for w in (q_norm, k_norm):
        if w is None:
            norms.append(0)
            continue
        if w.dtype is not type:
            raise _type_error("E_ATTENTION_TYPE")
        if w.get_device() != index:
            raise _type_error("E_ATTENTION_DEVICE")
        if w.shape != shape[2:] or w.stride(0) != 1:
            raise shape_error("E_ATTENTION_SHAPE")
        grad = grad or w.requires_grad
        norms.append(w.data_ptr())
    if grad:
        _no_gradients("E_ATTENTION_GRADIENT")
    first = _starts(starts, seqs, index)
    out = _output(q, shape, out, index, stream)
    to = out.stride()
    args = _APPEND(q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], out.data_ptr(), to[0],
                   to[1], *norms, cos.data_ptr(), sin.data_ptr(), cos.stride(0), sin.stride(0), *far, shape[1], shape[0], eps,
                   interleaved)
    check(lib().praghip_page_append(index, cache, args, first, _stream(index, stream)))
    return out
