"""Products of a few rows with 4-bit weights and group scales (streams and gradients as
in :mod:`praghip.attention`)."""
from __future__ import annotations

import struct

from . import attention
from ._lib import check, lib, shape_error
from .attention import _kind, _no_gradients, _result, _stream, _type_error

_W4 = struct.Struct("PqPqPq4Qi4x").pack  # praghip_w4


def matvec_w4(x, weights, scales, zeros=None, *, group: int = 128, out=None, stream=None):
    """y[m][n] = sum_k x[m][k] (w[n][k] - z[n][k // group]) s[n][k // group].

    x [rows][k] bfloat16 or float16; weights uint8 [n][width], two 4-bit values a byte
    with the lower bits first (width >= (k + 1) // 2); scales [n][groups] of x's type;
    zeros uint8 [n][groups] or None for 8 everywhere; group a multiple of 32, the last
    group may be short.  Sums are 32-bit, rounded once to x's type.  Reads the weights
    once per 32 rows: meant for few rows.
    """
    kind, index = _kind(x, "E_W4_TYPE"), x.get_device()
    if weights.dtype is not attention._uint8 or scales.dtype is not x.dtype or \
            (zeros is not None and zeros.dtype is not weights.dtype):
        raise _type_error("E_W4_TYPE")
    if not weights.get_device() == scales.get_device() == index >= 0 or \
            (zeros is not None and zeros.get_device() != index):
        raise _type_error("E_W4_DEVICE")
    xs, ws, ss = x.stride(), weights.stride(), scales.stride()
    try:
        (m, k), (n, width) = x.shape, weights.shape
    except ValueError:
        raise shape_error("E_W4_SHAPE") from None
    if group <= 0 or group % 32 or width < (k + 1) // 2 or scales.shape != (n, -(-k // group)) or \
            (xs[1] != 1 and k > 1) or (ws[1] != 1 and width > 1) or (ss[1] != 1 and k > group):
        raise shape_error("E_W4_SHAPE")
    if x.requires_grad or scales.requires_grad:
        _no_gradients("E_W4_GRADIENT")
    zero, zs = 0, 0
    if zeros is not None:
        if zeros.shape != scales.shape or (zeros.stride(1) != 1 and k > group):
            raise shape_error("E_W4_SHAPE")
        zero, zs = zeros.data_ptr(), zeros.stride(0)
    if out is None:
        out = x.new_empty((m, n)) if stream is None else _result(stream, index, x.new_empty, (m, n))
    elif out.shape != (m, n) or out.dtype is not x.dtype or out.get_device() != index or \
            (n > 1 and out.stride(1) != 1):
        raise shape_error("E_W4_OUT")
    w = _W4(weights.data_ptr(), ws[0], scales.data_ptr(), ss[0], zero, zs, n, k, width, group, kind)
    check(lib().praghip_matvec_w4(index, w, x.data_ptr(), xs[0], m, out.data_ptr(), out.stride(0),
                                  _stream(index, stream)))
    return out


def quantize_w4(weight, group: int = 128, *, zeros: bool = False):
    """Rounds weights [n][k] to 4 bits with a scale (and a zero point) per group of k.

    Returns (packed uint8 [n][width], scales [n][groups] of the weights' type, zeros
    uint8 or None) as :func:`matvec_w4` takes them, width a multiple of 16.  Without
    zero points a group spans -8 .. 7 times its scale, with them 0 .. 15 from its
    smallest value on (0 included, so that a weight of 0 stays 0).  No gradients pass.
    """
    import torch
    _kind(weight, "E_W4_TYPE")
    if weight.dim() != 2 or group <= 0 or group % 32:
        raise shape_error("E_W4_SHAPE")
    weight = weight.detach()
    n, k = weight.shape
    groups, width = -(-k // group), -(-k // 32) * 16
    w = torch.zeros((n, groups * group), dtype=torch.float32, device=weight.device)
    w[:, :k] = weight
    w = w.view(n, groups, group)
    if zeros:
        low, high = w.amin(-1).clamp(max=0), w.amax(-1).clamp(min=0)
        scales = ((high - low) / 15).to(weight.dtype)
    else:
        low = None
        scales = (w.abs().amax(-1) / 7).to(weight.dtype)
    s = scales.float()
    s = torch.where(s == 0, torch.ones_like(s), s)
    zero = torch.round(-low / s).clamp(0, 15) if zeros else torch.full_like(s, 8)
    digits = (torch.round(w / s[..., None]) + zero[..., None]).clamp(0, 15).to(torch.uint8).flatten(1)
    if digits.shape[1] < 2 * width:
        digits = torch.nn.functional.pad(digits, (0, 2 * width - digits.shape[1]))
    digits = digits[:, : 2 * width]
    packed = (digits[:, ::2] | (digits[:, 1::2] << 4)).contiguous()
    return packed, scales, zero.to(torch.uint8) if zeros else None
