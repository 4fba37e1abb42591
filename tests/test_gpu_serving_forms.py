"""Every form of the attention kernels (types, head sizes at and below a kernel's, masked and
not, split over keys and not), large scores, values that are not finite, and a cache whose
offsets pass 32 bits, against 64 bits."""
import math

import pytest
import torch

import attention_plain as plain
import praghip

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def to_gpu(c):
    return [c[x].to("cuda") for x in ("k", "v", "tables", "lengths")]


@pytest.mark.parametrize("type", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 56, 128, 120, 256, 248])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 5)])
def test_forms(gpu, type, dim, window, sinks):
    """One token, a chunk whose keys are split over workgroups, and a prompt from its start,
    of one cache: more tiles than there are LDS slots, a last tile that ends anywhere."""
    print("[forms]", type, dim, window, sinks, flush=True)
    c = plain.make([730, 331], 6, 2, dim, 32, type, seed=dim + window)
    on = to_gpu(c)
    q = torch.randn((2, 6, dim), generator=c["g"]).to(type)
    want, wlse, size = plain.attention(c, q, [0, 1, 2], window=window, sinks=sinks)
    out, lse = praghip.paged_decode(q.to("cuda"), *on, window=window, sinks=sinks, lse=True)
    torch.cuda.synchronize()
    plain.check(out, want, size, type, rounded=False)
    plain.check_lse(lse, wlse)
    for rows in ([40, 9], [730, 331]):
        starts = [0, rows[0], sum(rows)]
        q = torch.randn((sum(rows), 6, dim), generator=c["g"]).to(type)
        out, lse = praghip.paged_prompt(q.to("cuda"), *on, torch.tensor(starts, dtype=torch.int32, device="cuda"), max(rows),
                                        window=window, sinks=sinks, lse=True)
        torch.cuda.synchronize()
        # (of the prompt from its start every seventh row, and the last ones)
        see = sorted({r for s in (0, 1) for r in list(range(starts[s], starts[s + 1], 7 if sum(rows) > 100 else 1)) +
                      [starts[s + 1] - 1]})
        want, wlse, size = rows_of(c, q, starts, see, window, sinks)
        plain.check(out[see], want, size, type, rounded=True)
        plain.check_lse(lse[see], wlse)


@pytest.mark.parametrize("type", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 56, 128, 120, 256, 248])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 5)])
def test_decode_of_wide_tables(gpu, type, dim, window, sinks):
    """Tables with room for a cache that is read past the caches, and short sequences in them;
    with a window through the caches.  Poison in what no query sees."""
    print("[forms] wide tables", type, dim, window, sinks, flush=True)
    width = (64 << 20) // (2 * 2 * dim * 4) // 32 + 2
    c = plain.make([730, 331], 6, 2, dim, 32, type, seed=dim + window + 1, width=width)
    q = torch.randn((2, 6, dim), generator=c["g"]).to(type)
    want, wlse, size = plain.attention(c, q, [0, 1, 2], window=window, sinks=sinks)
    out, lse = praghip.paged_decode(q.to("cuda"), *to_gpu(c), window=window, sinks=sinks, lse=True)
    torch.cuda.synchronize()
    plain.check(out, want, size, type, rounded=False)
    plain.check_lse(lse, wlse)


def rows_of(c, q, starts, see, window, sinks):
    """attention() of some of the rows, each with its keys at once."""
    heads, dim = q.shape[1:]
    want, size = torch.zeros((2, len(see), heads, dim), dtype=torch.float64)
    lse = torch.full((len(see), heads), -math.inf, dtype=torch.float64)
    held = [plain.rows_of(c, s) for s in range(len(starts) - 1)]
    for i, row in enumerate(see):
        s = max(s for s in range(len(starts) - 1) if starts[s] <= row)
        at, k, v = held[s]
        place = int(c["lengths"][s]) - (starts[s + 1] - row)
        seen = at <= place
        if window:
            seen &= (at > place - window) | (at < sinks)
        k, v = (x[seen].repeat_interleave(heads // c["kv"], 1) for x in (k, v))
        score = torch.einsum("khd,hd->hk", k, q[row].double()) * dim ** -0.5
        lse[i] = torch.logsumexp(score, 1)
        p = torch.exp(score - lse[i][:, None])
        want[i] = torch.einsum("hk,khd->hd", p, v)
        size[i] = torch.einsum("hk,khd->hd", p, v.abs())
    return want, lse, size


@pytest.mark.parametrize("type,dim", [(BF16, 128), (F16, 64)])
def test_prompt_large_scores(gpu, type, dim):
    """Scores in the hundreds that rise along the keys: the maximum moves all the time."""
    print("[forms] large scores", type, dim, flush=True)
    c = plain.make([500], 4, 2, dim, 16, type, seed=31)
    rise = torch.linspace(0.1, 24, 500)
    for at in range(500):
        page = c["tables"][0, at // 16]
        c["k"][page, :, at % 16] = (c["k"][page, :, at % 16].float() * rise[at]).to(type)
    q = (24 * torch.randn((200, 4, dim), generator=c["g"])).to(type)
    out, lse = praghip.paged_prompt(q.to("cuda"), *to_gpu(c), torch.tensor([0, 200], dtype=torch.int32, device="cuda"), 200, lse=True)
    torch.cuda.synchronize()
    want, wlse, size = rows_of(c, q, [0, 200], list(range(200)), 0, 0)
    # dim products of up to 100 * 100 and their sums' roundings, relative in the probabilities
    off = dim * 2.0 ** -24 * 1e4 * dim ** -0.5 * 4
    got = out.double().cpu()
    unit = plain.UNIT[type]
    assert ((got - want).abs() <= unit * want.abs() + (off + 2 * unit) * size + 1e-7).all()
    assert ((lse.double().cpu() - wlse).abs() <= off + 1e-6 * wlse.abs()).all()


@pytest.mark.parametrize("type,dim", [(BF16, 128), (F16, 96)])
def test_values_that_are_not_finite(gpu, type, dim):
    """An infinity among the values reaches the queries that see it, in its column alone, and
    no others: those before it, and those whose window it has left."""
    print("[forms] not finite", type, dim, flush=True)
    c = plain.make([400], 4, 2, dim, 16, type, seed=33)
    q = torch.randn((400, 4, dim), generator=c["g"]).to(type)
    see = list(range(400))
    want, wlse, size = rows_of(c, q, [0, 400], see, 100, 3)
    c["v"][c["tables"][0, 150 // 16], 1, 150 % 16, 5] = math.inf
    out, lse = praghip.paged_prompt(q.to("cuda"), *to_gpu(c), torch.tensor([0, 400], dtype=torch.int32, device="cuda"), 400,
                                    window=100, sinks=3, lse=True)
    torch.cuda.synchronize()
    out = out.cpu()
    hit = torch.zeros(out.shape, dtype=torch.bool)
    hit[150:250, 2:, 5] = True
    assert torch.equal(torch.isfinite(out), ~hit)
    out[hit] = want[hit].to(type)
    plain.check(out, want, size, type, rounded=True)
    plain.check_lse(lse, wlse)
    c["lengths"][0] = 240  # the decode of row 239, which sees it
    out = praghip.paged_decode(q[239:240].to("cuda"), *to_gpu(c), window=100, sinks=3).cpu()
    assert torch.equal(torch.isfinite(out), ~hit[239:240])


def test_offsets_beyond_32_bits(gpu):
    """Pages 4.9e9 values into a cache: written, read by a token and a prompt, and copied."""
    print("[forms] long offsets", flush=True)
    pages, kv, page, dim = 300_000, 8, 16, 128
    pool = torch.empty((2, pages, kv, page, dim), dtype=BF16, device="cuda")
    c = plain.make([75, 200], 16, kv, dim, page, BF16, seed=34)
    count = c["k"].shape[0]
    at = pages - count
    tables = torch.where(c["tables"] >= 0, c["tables"] + at, -1).to(torch.int32).to("cuda")
    lengths = c["lengths"].to("cuda")
    new = [torch.cat([x[c["tables"][s, i // page], :, i % page][None] for s, n in enumerate((75, 200)) for i in range(n)])
           for x in (c["k"], c["v"])]
    starts = torch.tensor([0, 75, 275], dtype=torch.int32, device="cuda")
    praghip.page_write(new[0].to("cuda"), new[1].to("cuda"), pool[0], pool[1], tables, lengths, starts)
    q = torch.randn((275, 16, dim), generator=c["g"]).to(BF16)
    see = [0, 1, 74, 75, 150, 274]
    want, wlse, size = rows_of(c, q, [0, 75, 275], see, 0, 0)
    out, lse = praghip.paged_prompt(q.to("cuda"), pool[0], pool[1], tables, lengths, starts, 200, lse=True)
    torch.cuda.synchronize()
    plain.check(out[see], want, size, BF16, rounded=True)
    plain.check_lse(lse[see], wlse)
    last = [2, 5]
    out = praghip.paged_decode(q[[74, 274]].to("cuda"), pool[0], pool[1], tables, lengths)
    plain.check(out, want[last], size[last], BF16, rounded=False)
    pairs = [[pages - 1, pages - 2], [3, 7]]
    praghip.page_copy(pool, *(torch.tensor(x, dtype=torch.int32, device="cuda") for x in pairs))
    assert torch.equal(pool[:, 3].view(torch.int16), pool[:, pages - 1].view(torch.int16))
    assert torch.equal(pool[:, 7].view(torch.int16), pool[:, pages - 2].view(torch.int16))
