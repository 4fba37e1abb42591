"""Root-mean-square norms with the residual's addition (streams and gradients as in
:mod:`praghip.attention`)."""
from __future__ import annotations

import struct

from . import attention
from ._lib import check, lib, shape_error
from .attention import _kind, _no_gradients, _result, _stream, _type_error

_NORM = struct.Struct("5P4q2Qfi").pack  # praghip_norm


def _row(t) -> int:
    return t.stride(0)


def add_norm(x, weight, residual=None, *, eps: float = 1e-6, out=None, total=None, stream=None):
    """out[i][j] = s[i][j] w[j] / sqrt(mean_j s[i][j]^2 + eps), with s = x + residual.

    x [rows][n] bfloat16 or float16, residual of x's shape and type or None, weight [n] of
    its type; rows of any stride, their values contiguous.  s is summed in 32 bits, read by
    the norm before any rounding, and rounded once into total.  Returns out, and with a
    residual (out, total).  out and total may be x or residual themselves.
    """
    kind, index, shape = _kind(x, "E_NORM_TYPE"), x.get_device(), x.shape
    type = x.dtype
    if weight.dtype is not type or (residual is not None and residual.dtype is not type):
        raise _type_error("E_NORM_TYPE")
    if not weight.get_device() == index >= 0 or (residual is not None and residual.get_device() != index):
        raise _type_error("E_NORM_DEVICE")
    if len(shape) != 2 or weight.shape != shape[1:] or (residual is not None and residual.shape != shape):
        raise shape_error("E_NORM_SHAPE")
    rows, n = shape
    if n > 1 and (x.stride(1) != 1 or weight.stride(0) != 1 or (residual is not None and residual.stride(1) != 1)):
        raise shape_error("E_NORM_SHAPE")
    if x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad):
        _no_gradients("E_NORM_GRADIENT")
    if residual is None and total is not None:
        raise shape_error("E_NORM_OUT")
    made = []
    for t in (out, total):
        if t is None:
            t = attention._torch.empty_like(x) if stream is None else _result(stream, index, attention._torch.empty_like, x)
        elif t.shape != shape or t.dtype is not type or t.get_device() != index or (n > 1 and t.stride(1) != 1):
            raise shape_error("E_NORM_OUT")
        made.append(t)
        if residual is None:
            break
    out = made[0]
    total, at, row = (made[1], made[1].data_ptr(), _row(made[1])) if residual is not None else (None, 0, 0)
    args = _NORM(x.data_ptr(), 0 if residual is None else residual.data_ptr(), weight.data_ptr(), out.data_ptr(), at, _row(x),
                 0 if residual is None else _row(residual), _row(out), row, rows, n, eps, kind)
    check(lib().praghip_add_norm(index, args, _stream(index, stream)))
    return out if residual is None else (out, total)
