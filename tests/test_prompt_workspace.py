"""The prompt attention takes the workspace that its function names for the same arguments,
without a GPU: calls whose workspace is enough come as far as the device, and there is none."""
import ctypes
import itertools

import pytest
import torch

from praghip import _lib

AT = 1 << 40  # an address, 16-byte aligned, that is nobody's

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="a GPU would run these calls")


def cache(width, heads, dim, seqs):
    strides = (ctypes.c_int64 * 3)(16 * dim * heads, 16 * dim, dim)
    return _lib.Cache(k=AT, v=AT, k_strides=strides, v_strides=strides, pages=9, kv_heads=heads, page_size=16, head_dim=dim, type=0,
                      tables=AT, table_stride=width, table_width=width, lengths=AT, seqs=seqs)


def call(c, heads, tokens, max_rows, window, max_length, work, size):
    strides = (ctypes.c_int64 * 2)(heads * c.head_dim, c.head_dim)
    rc = _lib.lib().praghip_paged_prompt(0, ctypes.byref(c), AT, strides, heads, AT, tokens, max_rows, AT, strides, None, 1.0,
                                         window, 4, max_length, work, size, None)
    return rc, _lib.lib().praghip_last_error().decode()


def test_a_call_takes_the_size_that_was_named():
    L = _lib.lib()
    split = 0
    for kv, dim, seqs, width, window in itertools.product((1, 8), (64, 256), (1, 5), (64, 1024), (0, 700)):
        c, heads = cache(width, kv, dim, seqs), 32
        for max_rows, max_length in itertools.product((1, 5, 77, 512, 2048, 8192, 1 << 22, 1 << 40), (0, 900, 8192)):
            need = L.praghip_paged_prompt_workspace(ctypes.byref(c), heads, max_rows, window, 4, max_length)
            for tokens in (1, 3, 100, 5000):
                rc, said = call(c, heads, tokens, max_rows, window, max_length, AT if need else None, need)
                assert rc and said.startswith("E_ATTENTION_HIP"), (kv, dim, seqs, width, window, max_rows, max_length, tokens, rc, said)
            split += need > 0
    assert split  # (some of them are split over their keys)


def test_too_small_a_workspace_is_refused():
    c = cache(1024, 1, 64, 1)
    need = _lib.lib().praghip_paged_prompt_workspace(ctypes.byref(c), 32, 5, 0, 4, 0)
    assert need > 0
    for work, size in ((AT, need - 1), (AT, 0), (None, need)):
        assert call(c, 32, 5, 5, 0, 0, work, size) == (_lib.E_SHAPE, "E_ATTENTION_WORKSPACE")
