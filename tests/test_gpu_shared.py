"""paged_shared against attention in 64 bits (attention_plain.py): groups of every size, prefixes
that end inside a page or a block, heads and types, sequences that take no part."""
import pytest
import torch

import attention_plain as plain
import praghip

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def make(groups, heads, kv, dim, page, type, seed, layout="phtd", fill=None, before=(), after=()):
    """groups: (shared, [lengths]); before, after: lengths of sequences of no group.  Whole pages
    of a prefix are the same pages, the one that it ends in is a copy for each."""
    lengths = list(before) + [n for _, group in groups for n in group] + list(after)
    c = plain.make(lengths, heads, kv, dim, page, type, seed, layout=layout, fill=fill)
    starts, s = [len(before)], len(before)
    for shared, group in groups:
        for i in range(s + 1, s + len(group)):
            have = min(shared, lengths[i], lengths[s])
            for p in range(-(-have // page)):
                rows = min(page, have - p * page)
                a, b = int(c["tables"][s, p]), int(c["tables"][i, p])
                if rows == page:
                    c["tables"][i, p] = a
                else:
                    for x in "kv":
                        c[x][b, :, :rows] = c[x][a, :, :rows]
        s += len(group)
        starts.append(s)
    c["groups"] = torch.tensor(starts, dtype=torch.int32)
    c["shared"] = torch.tensor([n for n, _ in groups], dtype=torch.int32)
    c["q"] = torch.randn((len(lengths), heads, dim), generator=c["g"]).to(type)
    return c


def call(c, **kw):
    q, k, v, tables, lengths, groups, shared = (c[x].cuda() for x in ("q", "k", "v", "tables", "lengths", "groups", "shared"))
    return praghip.paged_shared(q, k, v, tables, lengths, groups, shared, lse=True, **kw)


def check(c, scale=None, **kw):
    out, lse = call(c, scale=scale, **kw)
    want, want_lse, size = plain.attention(c, c["q"], list(range(len(c["q"]) + 1)), scale)
    plain.check(out, want, size, c["q"].dtype, False)
    plain.check_lse(lse, want_lse)
    return out, lse


GROUPS = [
    [(40, [40])], [(40, [41, 57])], [(1, [1, 2, 3])], [(64, [64, 64, 64, 64])], [(100, [100 + i for i in range(16)])],
    [(33, [34] * 17)], [(300, [301] * 33)], [(16, [20, 16, 30]), (200, [201, 333]), (5, [7])], [(0, [5, 6])],
    [(31, [50, 33]), (32, [50, 33]), (33, [50, 33])],
]


@pytest.mark.parametrize("groups", GROUPS, ids=lambda g: "-".join(f"{n}x{len(x)}" for n, x in g))
@pytest.mark.parametrize("heads,kv,dim,type", [(4, 2, 64, F16), (16, 8, 128, BF16)])
def test_groups(gpu, groups, heads, kv, dim, type):
    print("[shared]", groups[0][0], heads, dim, flush=True)
    check(make(groups, heads, kv, dim, 16, type, seed=heads + len(groups)))


@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 8), (3, 3, 24), (12, 1, 96), (28, 4, 128), (40, 1, 64), (6, 2, 72), (8, 2, 256), (4, 1, 136),
                                         (2, 1, 200)])
@pytest.mark.parametrize("page,layout", [(16, "phtd"), (64, "pthd")])
def test_heads(gpu, heads, kv, dim, page, layout):
    print("[shared] heads", heads, kv, dim, page, flush=True)
    check(make([(150, [150, 190, 151]), (70, [71] * 9)], heads, kv, dim, page, BF16 if page == 16 else F16, seed=dim, layout=layout))


@pytest.mark.parametrize("members,heads,kv,dim", [(64, 4, 2, 64), (40, 8, 1, 64), (20, 28, 4, 128), (70, 8, 2, 256), (300, 2, 2, 64)])
def test_many_columns(gpu, members, heads, kv, dim):
    """More columns of a head than a workgroup's waves hold at once."""
    print("[shared] columns", members * heads // kv, flush=True)
    check(make([(90, [90 + i % 5 for i in range(members)])], heads, kv, dim, 16, BF16, seed=members))


def test_long_prefixes(gpu):
    """Prefixes over many workgroups, and a sequence's own keys too."""
    print("[shared] long", flush=True)
    check(make([(5000, [5003, 9000, 5000])], 4, 2, 64, 16, BF16, seed=31))
    check(make([(3000, [3001] * 5), (2, [4000, 3])], 2, 1, 128, 64, F16, seed=32))


def test_sequences_that_take_no_part(gpu):
    """Sequences around the groups, empty ones, ones that are shorter than their group's prefix,
    a first one that is, groups of none, and no groups at all."""
    print("[shared] no part", flush=True)
    c = make([(80, [100, 0, 81, 30, 90]), (64, [20, 70, 64]), (50, [0, 60])], 4, 2, 64, 16, BF16, seed=33, before=[44, 0], after=[77, 1])
    check(c)
    c["groups"], c["shared"] = torch.tensor([2, 2, 7, 7, 10, 12], dtype=torch.int32), torch.tensor([9, 80, 5, 64, 50], dtype=torch.int32)
    first = check(c)
    c["groups"], c["shared"] = torch.zeros(1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    for a, b in zip(first, check(c)):
        assert torch.equal(a.isfinite(), b.isfinite())


def test_against_the_decode(gpu):
    """The same sequences without their groups."""
    c = make([(700, [711, 702, 1000]), (32, [90, 40])], 16, 8, 128, 16, BF16, seed=34)
    out, lse = call(c)
    q, k, v, tables, lengths = (c[x].cuda() for x in ("q", "k", "v", "tables", "lengths"))
    want, want_lse = praghip.paged_decode(q, k, v, tables, lengths, lse=True)
    # (both off by half a step of the result and their sums)
    assert bool(((out.float() - want.float()).abs() <= 2.0 ** -7 * want.float().abs() + 1e-3).all())
    assert bool(((lse - want_lse).abs() <= 2 * plain.SUMS).all())


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0, 30.0])
def test_scales(gpu, scale):
    c = make([(60, [61, 75])], 2, 1, 64, 16, F16, seed=35)
    if abs(scale) > 1:  # (scores of some hundred: their rounding in 32 bits is that of their size)
        c["q"] = (c["q"].float() / 8).half()
    check(c, scale=scale)


def test_places_without_a_page(gpu):
    """Entries of the first sequence that are no page: no member sees those positions; a member's
    own entries below the prefix are not looked at."""
    c = make([(100, [110, 120, 130])], 4, 2, 64, 16, BF16, seed=36)
    c["tables"][1:, :6] = 10 ** 6
    out, lse = call(c)
    c["tables"][1:, :6] = c["tables"][0, :6]
    want, want_lse, size = plain.attention(c, c["q"], [0, 1, 2, 3])
    plain.check(out, want, size, BF16, False)
    c["tables"][0, 2], c["tables"][0, 4] = -1, len(c["k"])
    out, lse = call(c)
    c["tables"][1:, :6] = c["tables"][0, :6]
    want, want_lse, size = plain.attention(c, c["q"], [0, 1, 2, 3])
    plain.check(out, want, size, BF16, False)
    plain.check_lse(lse, want_lse)


def test_lengths_and_groups_out_of_range(gpu):
    """Lengths outside the tables, shared positions below 0 and beyond everything, and groups that
    reach beyond the sequences."""
    c = make([(64, [64, 64, 64])], 4, 2, 64, 16, BF16, seed=37, after=[30])
    for shared in (-5, 2 ** 31 - 1, 64):
        c["shared"] = torch.tensor([shared], dtype=torch.int32)
        check(c)
    c["lengths"][1] = 2 ** 31 - 1
    c["lengths"][2] = -3
    check(c)
    c["lengths"][:3] = 64
    want = call(c)
    for groups in ([0, 3, 9], [0, 3, 3]):
        c["groups"], c["shared"] = torch.tensor(groups, dtype=torch.int32), torch.tensor([64, 7], dtype=torch.int32)
        got = call(c)
        assert all(torch.equal(a[:3], b[:3]) for a, b in zip(got, want))


def test_values_that_are_not_finite(gpu):
    """Those of a prefix reach every member that has it and nobody else; those of one's own keys
    only that one; those that nobody sees, nobody."""
    c = make([(50, [60, 55, 20, 70])], 4, 2, 64, 16, BF16, seed=38, after=[33])
    want = call(c)
    c["v"][int(c["tables"][1, 3]), 0, 3] = float("inf")  # position 51 of sequence 1
    got = call(c)
    assert torch.equal(got[0][[0, 2, 3, 4]], want[0][[0, 2, 3, 4]]) and not bool(got[0][1, :2].isfinite().all())
    c["v"][int(c["tables"][0, 0]), 0, 3] = float("nan")
    got = call(c)
    assert torch.equal(got[0][4], want[0][4]) and bool(got[0][[0, 1, 3], :2].isnan().all())
    # (the shorter sequence reads position 3 from its own page, which is a prefix's too)
    assert torch.equal(got[1][[0, 3, 4]], want[1][[0, 3, 4]])


def test_strides_and_results(gpu):
    c = make([(90, [91, 95, 120])], 4, 2, 64, 16, BF16, seed=39)
    want = call(c)
    q = torch.randn((3, 9, 2, 72), device="cuda").to(BF16)[:, ::2][:, :4, 1, 8:]
    q.copy_(c["q"].cuda())
    k, v, tables, lengths, groups, shared = (c[x].cuda() for x in ("k", "v", "tables", "lengths", "groups", "shared"))
    named = torch.full((3, 40), -1, dtype=torch.int32, device="cuda")
    named[:, 7: 7 + tables.shape[1]] = tables
    wide = torch.full((3, 8, 80), 5.0, dtype=BF16, device="cuda")
    out = praghip.paged_shared(q, k, v, named[:, 7: 7 + tables.shape[1]], lengths, groups, shared, out=wide[:, ::2, 8:72])
    assert torch.equal(out, want[0])
    wide[:, ::2, 8:72] = 5.0
    assert bool((wide == 5.0).all())


def test_the_same_bits_and_a_captured_call(gpu):
    """Replayed with other queries, lengths and groups, against the eager call."""
    c = make([(400, [410, 500, 401, 444]), (90, [100, 95])], 16, 8, 128, 16, BF16, seed=40)
    dev = [c[x].cuda() for x in ("q", "k", "v", "tables", "lengths", "groups", "shared")]

    def run():
        return praghip.paged_shared(*dev, lse=True)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for shared, less in (([400, 90], 0), ([350, 0], 1), ([0, 64], 3), ([400, 90], 0)):
        dev[0].copy_(torch.randn_like(dev[0]))
        dev[4].copy_(c["lengths"] - less)
        dev[6].copy_(torch.tensor(shared, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(run(), got))
        assert all(torch.equal(a, b) for a, b in zip(run(), got))


def test_a_bound_of_the_lengths(gpu):
    c = make([(200, [210, 220, 230])], 4, 2, 64, 16, BF16, seed=41)
    for bound in (0, 230, 1, 10 ** 9):  # (one that is too small sizes the launch alone)
        check(c, max_length=bound)


def test_far_pages(gpu):
    """A cache of more than 2^31 values."""
    pages, page, kv, dim = 270000, 64, 2, 64
    c = make([(70, [90, 100, 71])], 4, kv, dim, page, BF16, seed=42)
    small = c["tables"] >= 0
    k, v = (torch.zeros((pages, kv, page, dim), dtype=BF16, device="cuda") for _ in "kv")
    n = len(c["k"])
    k[pages - n:], v[pages - n:] = c["k"].cuda().nan_to_num(0), c["v"].cuda().nan_to_num(0)
    want = call(c)
    tables = torch.where(small, c["tables"] + (pages - n), -1).cuda()
    got = praghip.paged_shared(c["q"].cuda(), k, v, tables, c["lengths"].cuda(), c["groups"].cuda(), c["shared"].cuda(), lse=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(gpu):
    c = make([(20, [30, 25])], 4, 2, 64, 16, BF16, seed=43)
    good = [c[x].cuda() for x in ("q", "k", "v", "tables", "lengths", "groups", "shared")]
    q, k, v, tables, lengths, groups, shared = good

    def refused(text, at=None, t=None, **kw):
        args = list(good)
        if at is not None:
            args[at] = t
        with pytest.raises(praghip.PraghipError) as e:
            praghip.paged_shared(*args, **kw)
        assert e.value.text == text, e.value.text

    for at, t in ((0, q[0]), (0, q[:1]), (0, q[:, :3]), (0, q[..., :32]), (1, k[0]), (2, v[:2]), (3, tables[0]), (4, lengths[:1]), (5, groups[:1]),
                  (5, groups[None]), (6, shared[None]), (6, shared.repeat(2)), (5, groups.repeat(2)[:3:2][:1])):
        refused("E_ATTENTION_SHAPE", at, t)
    for at, t in ((0, q.float()), (1, k.half()), (2, v.half())):
        refused("E_ATTENTION_TYPE", at, t)
    refused("E_ATTENTION_DEVICE", 1, k.cpu())
    for at, t in ((3, tables.long()), (4, lengths.cpu()), (5, groups.long()), (5, groups.cpu()), (6, shared.long()), (6, shared.cpu())):
        refused("E_ATTENTION_INTS", at, t)
    refused("E_ATTENTION_SHAPE", scale=float("nan"))
    refused("E_ATTENTION_SHAPE", max_length=-1)
    refused("E_ATTENTION_OUT", out=q[:1])
    for at in range(3):
        refused("E_ATTENTION_GRADIENT", at, good[at].clone().requires_grad_())
    with torch.no_grad():
        assert not praghip.paged_shared(q.clone().requires_grad_(), *good[1:]).requires_grad
    empty = praghip.paged_shared(q[:0], k, v, tables[:0], lengths[:0], groups[:1], shared[:0])
    assert empty.shape == (0, 4, 64)
