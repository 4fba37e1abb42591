"""The serving calls' checks of their arguments, without a GPU: every refusal comes back
before a device call, with addresses that nothing may touch; and the structures as Python
packs them are the header's."""
import ctypes
import os
import re
import subprocess

import pytest

from praghip import _lib, attention, matvec, pages

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
AT = 1 << 40  # an address, 16-byte aligned, that is nobody's
TWO = (ctypes.c_int64 * 2)
THREE = (ctypes.c_int64 * 3)


def refused(code, text, rc):
    said = _lib.lib().praghip_last_error().decode()
    assert rc == code and said == text, (rc, said)


def cache(**other):
    c = dict(k=AT, v=AT, k_strides=THREE(16 * 128 * 8, 16 * 128, 128), v_strides=THREE(16 * 128 * 8, 16 * 128, 128), pages=9,
             kv_heads=8, page_size=16, head_dim=128, type=0, tables=AT, table_stride=4, table_width=4, lengths=AT, seqs=2)
    return _lib.Cache(**{**c, **other})


def decode(c=None, q=AT, q_strides=(2048, 128), heads=16, out=AT, out_strides=(2048, 128), lse=None, scale=1.0, window=0, sinks=0,
           max_length=0, work=AT, size=1 << 40):
    c = ctypes.byref(cache() if c is None else c)
    return _lib.lib().praghip_paged_decode(0, c, q, q_strides and TWO(*q_strides), heads, out, out_strides and TWO(*out_strides), lse,
                                           scale, window, sinks, max_length, work, size, None)


def prompt(c=None, q=AT, q_strides=(2048, 128), heads=16, starts=AT, tokens=5, max_rows=5, out=AT, out_strides=(2048, 128), lse=None,
           scale=1.0, window=0, sinks=0, max_length=0, work=AT, size=1 << 40):
    c = ctypes.byref(cache() if c is None else c)
    return _lib.lib().praghip_paged_prompt(0, c, q, q_strides and TWO(*q_strides), heads, starts, tokens, max_rows, out,
                                           out_strides and TWO(*out_strides), lse, scale, window, sinks, max_length, work, size, None)


SHAPES = [dict(page_size=24), dict(page_size=8), dict(page_size=65536), dict(head_dim=0), dict(head_dim=12), dict(head_dim=264),
          dict(pages=0), dict(pages=1 << 31), dict(kv_heads=0), dict(kv_heads=65537), dict(seqs=(1 << 20) + 1), dict(table_width=0),
          dict(k_strides=THREE(1 << 31, 2048, 128)), dict(v_strides=THREE(16384, -8, 128)), dict(v_strides=THREE(16384, 2048, 1 << 26))]
ALIGNMENT = [dict(k=AT + 8), dict(v=AT + 2), dict(tables=AT + 2), dict(lengths=AT + 1), dict(k_strides=THREE(16384, 2048, 132)),
             dict(v_strides=THREE(16388, 2048, 128))]


@pytest.mark.parametrize("call", [decode, prompt])
def test_a_cache_that_does_not_fit(call):
    for other in SHAPES:
        refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", call(cache(**other)))
    for other in ALIGNMENT:
        refused(_lib.E_ARGUMENT, "E_ATTENTION_ALIGNMENT", call(cache(**other)))
    for name in ("k", "v", "tables", "lengths"):
        refused(_lib.E_ARGUMENT, "E_NULL", call(cache(**{name: None})))
    refused(_lib.E_ARGUMENT, "E_ATTENTION_TYPE", call(cache(type=2)))


@pytest.mark.parametrize("call", [decode, prompt])
def test_attention_arguments(call):
    for other in (dict(q=None), dict(q_strides=None), dict(out=None), dict(out_strides=None)):
        refused(_lib.E_ARGUMENT, "E_NULL", call(**other))
    for other in (dict(heads=0), dict(heads=12), dict(heads=1 << 17), dict(scale=float("nan")), dict(scale=float("inf"))):
        refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", call(**other))
    for other in (dict(q=AT + 8), dict(out=AT + 4), dict(work=AT + 8), dict(lse=AT + 2), dict(q_strides=(2048, 4)),
                  dict(out_strides=(2052, 128))):
        refused(_lib.E_ARGUMENT, "E_ATTENTION_ALIGNMENT", call(**other))
    # launches beyond 32 bits
    refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", call(cache(seqs=1 << 20)))
    assert _lib.lib().praghip_paged_decode_workspace(ctypes.byref(cache(seqs=1 << 20)), 16, 0) == 0


def test_decode_and_prompt_sizes():
    L = _lib.lib()
    refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", decode(cache(seqs=1 << 19, table_width=1 << 22)))
    refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", prompt(cache(seqs=1000), tokens=1 << 30, max_rows=1 << 30))
    refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", prompt(tokens=1 << 40, max_rows=1))
    assert L.praghip_paged_prompt_workspace(ctypes.byref(cache(seqs=1000)), 16, 1 << 40, 0, 0, 0) == 0
    refused(_lib.E_ARGUMENT, "E_NULL", decode(work=None))
    need = L.praghip_paged_decode_workspace(ctypes.byref(cache()), 16, 0)
    assert need > 0
    refused(_lib.E_SHAPE, "E_ATTENTION_WORKSPACE", decode(size=need - 1))
    long = cache(table_width=512)
    need = L.praghip_paged_prompt_workspace(ctypes.byref(long), 16, 5, 0, 0, 0)
    assert need > 0  # few rows over many keys are split
    refused(_lib.E_SHAPE, "E_ATTENTION_WORKSPACE", prompt(long, size=need - 1))
    refused(_lib.E_SHAPE, "E_ATTENTION_WORKSPACE", prompt(long, work=None))
    # nothing to do is no error, whatever else is there
    assert decode(cache(seqs=0, k=None)) == prompt(cache(seqs=0)) == prompt(tokens=0, q=None) == prompt(max_rows=0) == _lib.OK


def table(**other):
    t = dict(tables=AT, stride=4, width=4, seqs=3, lengths=AT, refs=AT, pages=9, page_size=16, status=None)
    return ctypes.byref(_lib.PageTable(**{**t, **other}))


def pool(**other):
    p = dict(base=AT, plane_bytes=1 << 20, page_bytes=4096, planes=2, pages=9)
    return ctypes.byref(_lib.PagePool(**{**p, **other}))


def test_pages():
    L = _lib.lib()
    calls = [lambda t: L.praghip_page_reserve(0, t, AT, AT, 2, None), lambda t: L.praghip_page_free(0, t, AT, 2, None),
             lambda t: L.praghip_page_trim(0, t, AT, 2, 5, 0, None),
             lambda t: L.praghip_page_fork(0, t, pool(), AT, AT, 2, AT, 1 << 20, None),
             lambda t: L.praghip_page_compact(0, t, pool(), AT, 1 << 20, None)]
    for call in calls:
        for other in (dict(page_size=12), dict(page_size=65536), dict(width=0), dict(width=1 << 31), dict(pages=0),
                      dict(pages=(1 << 28) + 1), dict(seqs=131073)):
            refused(_lib.E_SHAPE, "E_PAGES_SHAPE", call(table(**other)))
        for other in (dict(tables=AT + 1), dict(lengths=AT + 2), dict(refs=AT + 3), dict(status=AT + 2)):
            refused(_lib.E_ARGUMENT, "E_PAGES_ALIGNMENT", call(table(**other)))
        for name in ("tables", "lengths", "refs"):
            refused(_lib.E_ARGUMENT, "E_NULL", call(table(**{name: None})))
    t = table()
    refused(_lib.E_ARGUMENT, "E_NULL", L.praghip_page_reserve(0, t, AT, None, 2, None))
    refused(_lib.E_SHAPE, "E_PAGES_SHAPE", L.praghip_page_free(0, t, AT, 8193, None))
    refused(_lib.E_ARGUMENT, "E_PAGES_ALIGNMENT", L.praghip_page_free(0, t, AT + 2, 2, None))
    refused(_lib.E_ARGUMENT, "E_PAGES_WINDOW", L.praghip_page_trim(0, t, AT, 2, 0, 4, None))
    assert L.praghip_page_reserve(0, None, None, None, 0, None) == _lib.OK


def test_pools():
    L, t = _lib.lib(), table()
    calls = [lambda p: L.praghip_page_fork(0, t, p, AT, AT, 2, AT, 1 << 20, None),
             lambda p: L.praghip_page_compact(0, t, p, AT, 1 << 20, None), lambda p: L.praghip_page_copy(0, p, AT, AT, 2, None)]
    for call in calls:
        for other in (dict(page_bytes=0), dict(page_bytes=24), dict(page_bytes=1 << 31), dict(planes=0), dict(pages=0)):
            refused(_lib.E_SHAPE, "E_PAGES_SHAPE", call(pool(**other)))
        for other in (dict(base=AT + 8), dict(plane_bytes=(1 << 20) + 4)):
            refused(_lib.E_ARGUMENT, "E_PAGES_ALIGNMENT", call(pool(**other)))
        refused(_lib.E_ARGUMENT, "E_NULL", call(pool(base=None)))
    for call in calls[:2]:
        refused(_lib.E_SHAPE, "E_PAGES_SHAPE", call(pool(pages=8)))
    size = L.praghip_page_fork_workspace(2)
    refused(_lib.E_SHAPE, "E_PAGES_WORKSPACE", L.praghip_page_fork(0, t, pool(), AT, AT, 2, AT, size - 1, None))
    refused(_lib.E_ARGUMENT, "E_NULL", L.praghip_page_fork(0, t, pool(), AT, AT, 2, None, 0, None))
    size = L.praghip_page_compact_workspace(9)
    refused(_lib.E_SHAPE, "E_PAGES_WORKSPACE", L.praghip_page_compact(0, t, pool(), AT, size - 1, None))
    refused(_lib.E_ARGUMENT, "E_PAGES_ALIGNMENT", L.praghip_page_copy(0, pool(), AT + 2, AT, 2, None))
    refused(_lib.E_ARGUMENT, "E_NULL", L.praghip_page_copy(0, pool(), AT, None, 2, None))


def test_write():
    def write(c=None, k=AT, ks=(1024, 128), v=AT, vs=(1024, 128), starts=AT, tokens=3):
        return _lib.lib().praghip_page_write(0, ctypes.byref(cache() if c is None else c), k, ks and TWO(*ks), v, vs and TWO(*vs),
                                             starts, tokens, None)
    for other in SHAPES:
        refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", write(cache(**other)))
    for other in (dict(k=None), dict(ks=None), dict(v=None), dict(vs=None), dict(starts=None)):
        refused(_lib.E_ARGUMENT, "E_NULL", write(**other))
    for other in (dict(k=AT + 8), dict(v=AT + 4), dict(ks=(1024, 132)), dict(vs=(1028, 128)), dict(starts=AT + 2)):
        refused(_lib.E_ARGUMENT, "E_ATTENTION_ALIGNMENT", write(**other))
    refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", write(tokens=1 << 31))
    assert write(tokens=0, k=None) == _lib.OK


def test_products():
    def product(x=AT, m=2, y=AT, **other):
        w = dict(w=AT, w_stride=64, scales=AT, scale_stride=1, zeros=None, zero_stride=0, n=16, k=128, width=64, group=128, type=0)
        return _lib.lib().praghip_matvec_w4(0, ctypes.byref(_lib.W4(**{**w, **other})), x, 128, m, y, 16, None)
    for other in (dict(w=None), dict(scales=None), dict(x=None), dict(y=None)):
        refused(_lib.E_ARGUMENT, "E_NULL", product(**other))
    refused(_lib.E_ARGUMENT, "E_W4_TYPE", product(type=2))
    for other in (dict(group=0), dict(group=48), dict(width=63), dict(k=129), dict(n=(1 << 27) + 1), dict(m=(1 << 20) + 1),
                  dict(k=1 << 31)):
        refused(_lib.E_SHAPE, "E_W4_SHAPE", product(**other))
    for other in (dict(x=AT + 1), dict(y=AT + 1), dict(scales=AT + 1)):
        refused(_lib.E_ARGUMENT, "E_W4_ALIGNMENT", product(**other))
    assert product(m=0, y=None) == product(n=0, y=None) == _lib.OK


def test_structures_are_the_headers(tmp_path):
    """Sizes, and each member's place, as a C compiler sees them, against the packed forms."""
    with open(os.path.join(ROOT, "include", "praghip.h")) as f:
        text = f.read()
    made = {"praghip_cache": (_lib.Cache, attention._CACHE), "praghip_page_table": (_lib.PageTable, pages._TABLE.__self__),
            "praghip_page_pool": (_lib.PagePool, pages._POOL.__self__), "praghip_w4": (_lib.W4, matvec._W4.__self__)}
    lines = []
    for name, (of, _) in made.items():
        assert re.search(r"\} %s;" % name, text), name
        lines.append('printf("%%zu", sizeof(%s));' % name)
        lines += ['printf(" %%zu", offsetof(%s, %s));' % (name, field[0]) for field in of._fields_]
        lines.append('printf("\\n");')
    source = tmp_path / "sizes.c"
    source.write_text('#include <stdio.h>\n#include "praghip.h"\nint main(void) {\n%s\nreturn 0; }\n' % "\n".join(lines))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(source), "-o", str(tmp_path / "sizes")], check=True)
    said = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, (name, (of, packed)) in zip(said, made.items()):
        want = [ctypes.sizeof(of)] + [getattr(of, field[0]).offset for field in of._fields_]
        assert [int(x) for x in line.split()] == want, name
        assert packed.size == want[0], name
    # each value of the packed cache is read back from its own member
    values = list(range(1, 19))
    c = _lib.Cache.from_buffer_copy(attention._CACHE.pack(*values))
    assert [c.k, c.v, *c.k_strides, *c.v_strides, c.pages, c.kv_heads, c.page_size, c.head_dim, c.type, c.tables, c.table_stride,
            c.table_width, c.lengths, c.seqs] == values
