"""Tensors of another rank than a serving call takes are refused in its own words."""
import pytest
import torch

import attention_plain as plain
import praghip

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def refused(text, call):
    with pytest.raises(praghip.PraghipError) as e:
        call()
    assert e.value.text == text, e.value.text


def test_products(gpu):
    x, w, s, z = torch.zeros((2, 64), dtype=BF16), torch.zeros((16, 32), dtype=torch.uint8), torch.zeros((16, 2), dtype=BF16), \
        torch.zeros((16, 2), dtype=torch.uint8)
    x, w, s, z = (t.to("cuda") for t in (x, w, s, z))
    F = praghip.matvec_w4
    for bad in ((x[0], w, s, z), (x[None], w, s, z), (x[0, 0], w, s, z), (x, w[0], s, z), (x, w[None], s, z), (x, w, s[0], z),
                (x, w, s[0, 0], z), (x, w, s, z[0]), (x, w, s[None], z[None])):
        refused("E_W4_SHAPE", lambda: F(*bad, group=32))
    refused("E_W4_OUT", lambda: F(x, w, s, z, group=32, out=x[0, :16]))


def test_attention(gpu):
    c = plain.make([20, 30], 4, 2, 64, 16, BF16, seed=61)
    k, v, tables, lengths = (c[x].to("cuda") for x in ("k", "v", "tables", "lengths"))
    q, starts = torch.zeros((2, 4, 64), dtype=BF16, device="cuda"), torch.arange(3, dtype=torch.int32, device="cuda")
    good = (q, k, v, tables, lengths)
    bad = [(0, q[0]), (0, q[None]), (0, q[0, 0, 0]), (1, k[0]), (1, k[None]), (2, v[0]), (3, tables[0]), (3, tables[None]),
           (3, tables[0, 0]), (4, lengths[None]), (4, lengths[0])]
    for at, t in bad:
        args = good[:at] + (t,) + good[at + 1:]
        refused("E_ATTENTION_SHAPE", lambda: praghip.paged_decode(*args))
        refused("E_ATTENTION_SHAPE", lambda: praghip.paged_prompt(*args, starts, 1))
        if at:
            refused("E_ATTENTION_SHAPE", lambda: praghip.page_write(q[:, :2], q[:, :2], *args[1:], starts))
    for t in (starts[0], starts[None]):
        refused("E_ATTENTION_SHAPE", lambda: praghip.paged_prompt(*good, t, 1))
        refused("E_ATTENTION_SHAPE", lambda: praghip.page_write(q[:, :2], q[:, :2], *good[1:], t))
    refused("E_ATTENTION_OUT", lambda: praghip.paged_decode(*good, out=q[0]))


def test_pages(gpu):
    def ints(*shape):
        return torch.zeros(shape, dtype=torch.int32, device="cuda")

    pool = torch.zeros((1, 2, 9, 1, 16, 16), dtype=BF16, device="cuda")
    good = (ints(4, 8), ints(4), ints(9))
    one, none = ints(1), ints(1)[0]
    for at, t in ((0, ints(8)), (0, none), (1, none), (1, ints(1, 4)), (2, none), (2, ints(1, 9))):
        bad = good[:at] + (t,) + good[at + 1:]
        refused("E_PAGES_SHAPE", lambda: praghip.page_reserve(*bad, 16, one, one))
        refused("E_PAGES_SHAPE", lambda: praghip.page_free(*bad, one))
        refused("E_PAGES_SHAPE", lambda: praghip.page_trim(*bad, 16, one, 5))
        refused("E_PAGES_SHAPE", lambda: praghip.page_fork(pool, *bad, one, one))
        if at != 1:
            refused("E_PAGES_SHAPE", lambda: praghip.page_compact(pool, bad[0], bad[2]))
    for t in (none, ints(1, 1)):
        refused("E_PAGES_SHAPE", lambda: praghip.page_reserve(*good, 16, t, one))
        refused("E_PAGES_SHAPE", lambda: praghip.page_reserve(*good, 16, one, t))
        refused("E_PAGES_SHAPE", lambda: praghip.page_free(*good, t))
        refused("E_PAGES_SHAPE", lambda: praghip.page_trim(*good, 16, t, 5))
        refused("E_PAGES_SHAPE", lambda: praghip.page_fork(pool, *good, t, one))
        refused("E_PAGES_SHAPE", lambda: praghip.page_fork(pool, *good, one, t))
        refused("E_PAGES_SHAPE", lambda: praghip.page_copy(pool, t, one))
        refused("E_PAGES_SHAPE", lambda: praghip.page_copy(pool, one, t))
    for p in (pool[0, 0, 0], pool[0, 0, 0, 0, 0, 0]):
        refused("E_PAGES_POOL", lambda: praghip.page_fork(p, *good, one, one))
        refused("E_PAGES_POOL", lambda: praghip.page_compact(p, good[0], good[2]))
        refused("E_PAGES_POOL", lambda: praghip.page_copy(p, one, one))
    assert not any(t.any() for t in good)
