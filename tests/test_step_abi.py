"""The checks of arguments of the calls of a model's step (new tokens into the cache, shared
prefixes, norms, draws), without a GPU: every refusal comes back before a device call, with
addresses that nothing may touch; and their structures as Python packs them are the header's."""
import ctypes
import os
import re
import subprocess

import pytest

from praghip import _lib, append, norm, sample
from test_serving_abi import ALIGNMENT, AT, SHAPES, TWO, cache, refused

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NAN, INF = float("nan"), float("inf")


def shared(c=None, q=AT, q_strides=(2048, 128), heads=16, groups=AT, prefixes=AT, count=1, out=AT, out_strides=(2048, 128), lse=None, scale=1.0,
           max_length=0, work=AT, size=1 << 40):
    c = ctypes.byref(cache() if c is None else c)
    return _lib.lib().praghip_paged_shared(0, c, q, q_strides and TWO(*q_strides), heads, groups, prefixes, count, out,
                                           out_strides and TWO(*out_strides), lse, scale, max_length, work, size, None)


def test_shared_prefixes():
    L = _lib.lib()
    for other in SHAPES:
        refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", shared(cache(**other)))
    for other in ALIGNMENT:
        refused(_lib.E_ARGUMENT, "E_ATTENTION_ALIGNMENT", shared(cache(**other)))
    for other in (dict(q=None), dict(q_strides=None), dict(out=None), dict(out_strides=None), dict(work=None), dict(groups=None), dict(prefixes=None)):
        refused(_lib.E_ARGUMENT, "E_NULL", shared(**other))
    for other in (dict(heads=0), dict(heads=12), dict(heads=1 << 17), dict(scale=NAN), dict(scale=INF), dict(count=(1 << 20) + 1)):
        refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", shared(**other))
    for other in (dict(q=AT + 8), dict(out=AT + 4), dict(work=AT + 8), dict(lse=AT + 2), dict(groups=AT + 2), dict(prefixes=AT + 1),
                  dict(q_strides=(2048, 4)), dict(out_strides=(2052, 128))):
        refused(_lib.E_ARGUMENT, "E_ATTENTION_ALIGNMENT", shared(**other))
    # more blocks than 32 bits count
    refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", shared(cache(seqs=1 << 19, table_width=1 << 22)))
    refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", shared(cache(seqs=1, table_width=1 << 22), count=1 << 20))
    assert L.praghip_paged_shared_workspace(ctypes.byref(cache(seqs=1 << 19, table_width=1 << 22)), 16, 1, 0) == 0
    assert L.praghip_paged_shared_workspace(ctypes.byref(cache(head_dim=12)), 16, 1, 0) == 0
    need = L.praghip_paged_shared_workspace(ctypes.byref(cache()), 16, 1, 0)
    assert need > 0
    refused(_lib.E_SHAPE, "E_ATTENTION_WORKSPACE", shared(size=need - 1))
    assert shared(cache(seqs=0, k=None)) == _lib.OK


def appended(c=None, starts=AT, null=False, **other):
    p = dict(q=AT, k=AT, v=AT, q_strides=TWO(4096, 128), k_strides=TWO(4096, 128), v_strides=TWO(4096, 128), out=AT, out_strides=TWO(2048, 128),
             q_norm=AT, k_norm=AT, cos=AT, sin=AT, cos_row=64, sin_row=64, positions=64, half=64, heads=16, tokens=3, eps=1e-6, interleaved=0)
    return _lib.lib().praghip_page_append(0, ctypes.byref(cache() if c is None else c), None if null else ctypes.byref(_lib.Append(**{**p, **other})),
                                          starts, None)


def test_new_tokens():
    for other in SHAPES:
        refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", appended(cache(**other)))
    for other in ALIGNMENT:
        refused(_lib.E_ARGUMENT, "E_ATTENTION_ALIGNMENT", appended(cache(**other)))
    for name in ("q", "k", "v", "out", "cos", "sin"):
        refused(_lib.E_ARGUMENT, "E_NULL", appended(**{name: None}))
    refused(_lib.E_ARGUMENT, "E_NULL", appended(starts=None))
    refused(_lib.E_ARGUMENT, "E_NULL", appended(null=True))
    for other in (dict(heads=0), dict(heads=65537), dict(tokens=1 << 31), dict(tokens=1 << 26)):
        refused(_lib.E_SHAPE, "E_ATTENTION_SHAPE", appended(**other))
    for other in (dict(half=65), dict(positions=63), dict(positions=1 << 31), dict(eps=-1.0), dict(eps=NAN), dict(eps=INF)):
        refused(_lib.E_SHAPE, "E_ROTARY_SHAPE", appended(**other))
    for other in (dict(q=AT + 8), dict(k=AT + 2), dict(v=AT + 4), dict(out=AT + 8), dict(q_norm=AT + 8), dict(k_norm=AT + 2), dict(cos=AT + 2),
                  dict(sin=AT + 1), dict(q_strides=TWO(4100, 128)), dict(k_strides=TWO(4096, 4)), dict(v_strides=TWO(4, 128)),
                  dict(out_strides=TWO(2048, 132))):
        refused(_lib.E_ARGUMENT, "E_ATTENTION_ALIGNMENT", appended(**other))
    refused(_lib.E_ARGUMENT, "E_ATTENTION_ALIGNMENT", appended(starts=AT + 2))
    assert appended(tokens=0, q=None) == appended(cache(seqs=0, k=None)) == _lib.OK


def normed(null=False, **other):
    p = dict(x=AT, residual=AT, weight=AT, out=AT, total=AT, x_row=64, residual_row=64, out_row=64, total_row=64, rows=2, n=64, eps=1e-6, type=0)
    return _lib.lib().praghip_add_norm(0, None if null else ctypes.byref(_lib.Norm(**{**p, **other})), None)


def test_norms():
    for name in ("x", "weight", "out"):
        refused(_lib.E_ARGUMENT, "E_NULL", normed(**{name: None}))
    refused(_lib.E_ARGUMENT, "E_NULL", normed(null=True))
    for bad in (2, 3, -1):
        refused(_lib.E_ARGUMENT, "E_NORM_TYPE", normed(type=bad))
    for other in (dict(rows=1 << 31), dict(n=(1 << 30) + 1), dict(eps=-1.0), dict(eps=NAN), dict(eps=INF)):
        refused(_lib.E_SHAPE, "E_NORM_SHAPE", normed(**other))
    for name in ("x", "residual", "weight", "out", "total"):
        refused(_lib.E_ARGUMENT, "E_NORM_ALIGNMENT", normed(**{name: AT + 1}))
    assert normed(rows=0, x=None) == normed(n=0, x=None) == _lib.OK


def drawn(null=False, work=AT, size=1 << 40, **other):
    p = dict(logits=AT, row=100, rows=2, vocab=100, uniform=AT, temperature=AT, top_p=AT, min_p=AT, top_k=AT, temperature_all=0, top_p_all=0, min_p_all=0,
             top_k_all=0, out=AT, type=0)
    return _lib.lib().praghip_sample_tokens(0, None if null else ctypes.byref(_lib.Sample(**{**p, **other})), work, size, None)


def test_draws():
    L = _lib.lib()
    for name in ("logits", "uniform", "out"):
        refused(_lib.E_ARGUMENT, "E_NULL", drawn(**{name: None}))
    refused(_lib.E_ARGUMENT, "E_NULL", drawn(work=None))
    refused(_lib.E_ARGUMENT, "E_NULL", drawn(null=True))
    refused(_lib.E_ARGUMENT, "E_SAMPLE_TYPE", drawn(type=3))
    for other in (dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(rows=65536)):
        refused(_lib.E_SHAPE, "E_SAMPLE_SHAPE", drawn(**other))
    for other in (dict(logits=AT + 1), dict(logits=AT + 2, type=2), dict(uniform=AT + 2), dict(temperature=AT + 1), dict(top_p=AT + 2), dict(min_p=AT + 3),
                  dict(top_k=AT + 2), dict(out=AT + 4)):
        refused(_lib.E_ARGUMENT, "E_SAMPLE_ALIGNMENT", drawn(**other))
    refused(_lib.E_ARGUMENT, "E_SAMPLE_ALIGNMENT", drawn(work=AT + 8))
    need = L.praghip_sample_workspace(2, 100)
    refused(_lib.E_SHAPE, "E_SAMPLE_WORKSPACE", drawn(size=need - 1))
    assert L.praghip_sample_workspace(65536, 100) == L.praghip_sample_workspace(1, (1 << 20) + 1) == 0
    assert drawn(rows=0, logits=None) == _lib.OK


def test_structures_are_the_headers(tmp_path):
    """Sizes, and each member's place, as a C compiler sees them, against the packed forms."""
    with open(os.path.join(ROOT, "include", "praghip.h")) as f:
        text = f.read()
    made = {"praghip_append": (_lib.Append, append._APPEND), "praghip_norm": (_lib.Norm, norm._NORM), "praghip_sample": (_lib.Sample, sample._SAMPLE)}
    lines = []
    for name, (of, _) in made.items():
        assert re.search(r"\} %s;" % name, text), name
        lines.append('printf("%%zu", sizeof(%s));' % name)
        lines += ['printf(" %%zu", offsetof(%s, %s));' % (name, field[0]) for field in of._fields_]
        lines.append('printf("\\n");')
    source = tmp_path / "sizes.c"
    source.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "praghip.h"\nint main(void) {\n%s\nreturn 0; }\n' % "\n".join(lines))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(source), "-o", str(tmp_path / "sizes")], check=True)
    said = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.splitlines()
    for line, (name, (of, packed)) in zip(said, made.items()):
        want = [ctypes.sizeof(of)] + [getattr(of, field[0]).offset for field in of._fields_]
        assert [int(x) for x in line.split()] == want, name
        assert packed.__self__.size == want[0], name
    # each packed value is read back from its own member
    a = _lib.Append.from_buffer_copy(append._APPEND(*range(1, 23), 0.5, 7))
    assert [a.q, a.k, a.v, *a.q_strides, *a.k_strides, *a.v_strides, a.out, *a.out_strides, a.q_norm, a.k_norm, a.cos, a.sin, a.cos_row, a.sin_row,
            a.positions, a.half, a.heads, a.tokens, a.eps, a.interleaved] == [*range(1, 23), 0.5, 7]
    n = _lib.Norm.from_buffer_copy(norm._NORM(*range(1, 12), 0.5, 1))
    assert [n.x, n.residual, n.weight, n.out, n.total, n.x_row, n.residual_row, n.out_row, n.total_row, n.rows, n.n, n.eps, n.type] == [*range(1, 12), 0.5, 1]
    s = _lib.Sample.from_buffer_copy(sample._SAMPLE(*range(1, 10), 0.25, 0.5, 0.75, 13, 14, 2))
    assert [s.logits, s.row, s.rows, s.vocab, s.uniform, s.temperature, s.top_p, s.min_p, s.top_k, s.temperature_all, s.top_p_all, s.min_p_all, s.top_k_all,
            s.out, s.type] == [*range(1, 10), 0.25, 0.5, 0.75, 13, 14, 2]


@pytest.mark.parametrize("name", ["paged_shared", "page_append", "rotary_table", "add_norm", "sample_tokens"])
def test_they_are_the_packages(name):
    import praghip
    assert callable(getattr(praghip, name))
