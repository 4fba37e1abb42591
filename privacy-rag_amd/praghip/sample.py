"""Tokens drawn from logits with given random numbers (streams and gradients as in
:mod:`praghip.attention`)."""
from __future__ import annotations

import math
import operator
import struct

from . import attention
from ._lib import check, lib, shape_error
from .attention import _no_gradients, _result, _stream, _type_error, _work

_SAMPLE = struct.Struct("Pq2Q5P3fiPi4x").pack  # praghip_sample
_types: dict = {}


def _load():
    attention._load()
    torch = attention._torch
    _types.update({torch.bfloat16: 0, torch.float16: 1, torch.float32: 2})


def _each(value, rows: int, index: int, dtype, least, most):
    """(address or 0, value of all rows) of one of the filters."""
    if hasattr(value, "data_ptr"):
        if value.dtype is not dtype:
            raise _type_error("E_SAMPLE_TYPE")
        if value.get_device() != index:
            raise _type_error("E_SAMPLE_DEVICE")
        if value.shape != (rows,) or (rows > 1 and value.stride(0) != 1):
            raise shape_error("E_SAMPLE_SHAPE")
        if value.requires_grad:
            _no_gradients("E_SAMPLE_GRADIENT")
        return value.data_ptr(), 0
    if dtype is attention._int32:
        try:
            value = operator.index(value)
        except TypeError:
            raise shape_error("E_SAMPLE_FILTER") from None
    if not least <= value <= most:
        raise shape_error("E_SAMPLE_FILTER")
    return 0, value


def sample_tokens(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, out=None, stream=None):
    """One token of each row of logits, drawn with the row's number of ``uniform``.

    logits [rows][vocab] bfloat16, float16 or float32, rows of any stride; uniform float32
    [rows] of [0, 1).  temperature, top_p and min_p are numbers or float32 [rows], top_k a
    whole number or int32 [rows]; numbers below 0, and a min_p above 1, are refused, in a list
    (which is on the GPU) they count as the nearest that is not.  With w = exp((x - max x) / temperature): of the tokens by falling
    logit (of equal ones the lower index first) the first top_k stay (0: all); of those the
    shortest run whose sum of w reaches top_p times theirs; of those the ones with w >= min_p.
    The token is the first, by index, up to which the sum of w is above uniform times the sum
    of all that stay.  Temperature 0 takes the largest logit's lowest index.  NaN counts as
    -infinity, which is never drawn: a row of nothing else gets -1.  Returns int64 [rows].
    """
    kind, index, shape = _types.get(logits.dtype), logits.get_device(), logits.shape
    if kind is None:
        _load()
        kind = _types.get(logits.dtype)
        if kind is None:
            raise _type_error("E_SAMPLE_TYPE")
    torch = attention._torch
    wide = attention._float32
    if uniform.dtype is not wide:
        raise _type_error("E_SAMPLE_TYPE")
    if not uniform.get_device() == index >= 0:
        raise _type_error("E_SAMPLE_DEVICE")
    if len(shape) != 2 or uniform.shape != shape[:1] or (shape[1] > 1 and logits.stride(1) != 1) or \
            (shape[0] > 1 and uniform.stride(0) != 1):
        raise shape_error("E_SAMPLE_SHAPE")
    rows, vocab = shape
    t, t_all = _each(temperature, rows, index, wide, 0.0, math.inf)
    p, p_all = _each(top_p, rows, index, wide, 0.0, math.inf)
    m, m_all = _each(min_p, rows, index, wide, 0.0, 1.0)
    k, k_all = _each(top_k, rows, index, attention._int32, 0, 2 ** 31 - 1)
    if logits.requires_grad or uniform.requires_grad:
        _no_gradients("E_SAMPLE_GRADIENT")
    if out is None:
        out = logits.new_empty((rows,), dtype=torch.int64) if stream is None else \
            _result(stream, index, logits.new_empty, (rows,), dtype=torch.int64)
    elif out.shape != (rows,) or out.dtype is not torch.int64 or out.get_device() != index or (rows > 1 and out.stride(0) != 1):
        raise shape_error("E_SAMPLE_OUT")
    if rows:
        L = lib()
        size = L.praghip_sample_workspace(rows, vocab)
        work = _work(size, logits, stream)
        args = _SAMPLE(logits.data_ptr(), logits.stride(0), rows, vocab, uniform.data_ptr(), t, p, m, k, t_all, p_all, m_all, k_all,
                       out.data_ptr(), kind)
        check(L.praghip_sample_tokens(index, args, work.data_ptr(), size, _stream(index, stream)))
    return out
