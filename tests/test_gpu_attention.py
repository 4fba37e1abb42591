"""Paged attention on the GPU against its definition in 64 bits: lengths of zero and
one, pages that end inside a block, windows and sinks, head layouts, strides, missing
pages, NaN in memory that no position names, streams, graphs, refusals."""
import math

import pytest
import torch

import attention_plain as plain
import praghip

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def to_gpu(c):
    # strides are kept: .to() of a permuted tensor preserves its layout
    return [c[x].to("cuda") for x in ("k", "v", "tables", "lengths")]


def decode(c, q, **kw):
    out, lse = praghip.paged_decode(q.to("cuda"), *to_gpu(c), lse=True, **kw)
    torch.cuda.synchronize()
    return out, lse


def say(*a):
    print("[attention]", *a, flush=True)


DECODE = [
    # lengths, heads, kv, dim, page, window, sinks, type
    ([1], 16, 8, 128, 16, 0, 0, BF16),
    ([2], 2, 2, 64, 16, 0, 0, F16),
    ([0, 1, 15, 16, 17, 31, 32, 33, 0, 63, 64, 65], 16, 8, 128, 16, 0, 0, BF16),
    ([0, 0, 0], 4, 2, 64, 32, 0, 0, F16),
    ([1000, 3, 0, 517, 2049], 16, 8, 128, 16, 0, 0, BF16),
    ([700, 41], 8, 8, 64, 64, 0, 0, F16),
    ([700, 41, 5], 28, 4, 128, 32, 0, 0, BF16),
    ([333, 90], 12, 1, 96, 16, 0, 0, F16),
    ([333, 90, 1], 20, 1, 128, 16, 0, 0, BF16),   # a group of more than 16
    ([200, 77], 64, 2, 64, 16, 0, 0, F16),        # two full turns of 16 heads
    ([130, 33], 4, 2, 256, 16, 0, 0, BF16),
    ([130, 33], 4, 2, 200, 16, 0, 0, F16),
    ([65, 40], 6, 3, 8, 16, 0, 0, BF16),
    ([65, 40], 6, 3, 40, 128, 0, 0, F16),
    ([1000, 100, 7], 16, 8, 128, 16, 64, 4, BF16),
    ([1000, 64, 65, 66, 0, 1], 32, 4, 64, 64, 64, 0, F16),
    ([1000, 257], 16, 8, 128, 16, 100, 33, BF16),  # sinks end inside a block
    ([500, 90], 16, 8, 128, 16, 1, 0, F16),        # a window of one
    ([500, 90], 16, 8, 128, 16, 470, 40, BF16),    # sinks that reach the window
    ([500, 90], 16, 8, 128, 16, 5000, 3, BF16),    # a window nothing reaches
]


@pytest.mark.parametrize("lengths,heads,kv,dim,page,window,sinks,type", DECODE)
def test_decode_against_64_bits(gpu, lengths, heads, kv, dim, page, window, sinks, type):
    say("decode", lengths, heads, kv, dim, page, window, sinks, type)
    c = plain.make(lengths, heads, kv, dim, page, type, seed=len(lengths) * 1000 + dim)
    q = torch.randn((len(lengths), heads, dim), generator=c["g"]).to(type)
    out, lse = decode(c, q, window=window, sinks=sinks)
    want, wlse, size = plain.attention(c, q, list(range(len(lengths) + 1)), window=window, sinks=sinks)
    plain.check(out, want, size, type, rounded=False)
    plain.check_lse(lse, wlse)


def test_decode_many_sequences(gpu):
    """More sequences than a workgroup has threads: several to a thread's stretch."""
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 60, (700,), generator=g).tolist()
    say("decode of 700 sequences")
    c = plain.make(lengths, 4, 2, 64, 16, BF16, seed=6)
    q = torch.randn((700, 4, 64), generator=g).to(BF16)
    out, lse = decode(c, q)
    want, wlse, size = plain.attention(c, q, list(range(701)))
    plain.check(out, want, size, BF16, rounded=False)
    plain.check_lse(lse, wlse)


@pytest.mark.parametrize("max_length", [0, 1, 5000, 1 << 40])
def test_decode_max_length_sizes_the_launch_alone(gpu, max_length):
    say("max_length", max_length)
    c = plain.make([3000, 10, 800], 8, 4, 128, 16, F16, seed=7, width=400)
    q = torch.randn((3, 8, 128), generator=c["g"]).to(F16)
    out, lse = decode(c, q, max_length=max_length)
    want, wlse, size = plain.attention(c, q, [0, 1, 2, 3])
    plain.check(out, want, size, F16, rounded=False)
    plain.check_lse(lse, wlse)


def test_decode_missing_pages_and_lengths_out_of_range(gpu):
    """Entries that are no page are seen by nobody, whole rows of them included; lengths
    beyond the tables count as the tables' width, negative ones as 0."""
    say("missing pages")
    c = plain.make([300, 200, 100, 64, 96], 8, 4, 64, 16, BF16, seed=8)
    c["tables"][0, 3] = -1
    c["tables"][0, 7] = 1 << 30
    c["tables"][1, :] = -5
    c["tables"][2, 6] = c["k"].shape[0]
    c["lengths"][3] = -7
    c["lengths"][4] = 2 ** 31 - 1   # six pages are named, the row's others are none
    for x in ("k", "v"):
        c[x].nan_to_num_(0.0)
    q = torch.randn((5, 8, 64), generator=c["g"]).to(BF16)
    out, lse = decode(c, q)
    want, wlse, size = plain.attention(c, q, list(range(6)))
    assert math.isinf(wlse[1, 0]) and math.isinf(wlse[3, 0])
    plain.check(out, want, size, BF16, rounded=False)
    plain.check_lse(lse, wlse)


def test_decode_strides(gpu):
    """Pages in [page][token][head][dim] order, a slice of wider rows of q, of out and of
    the tables, one tensor that holds keys and values side by side."""
    say("strides")
    c = plain.make([150, 77], 8, 4, 64, 16, F16, seed=9, layout="pthd")
    q = torch.randn((2, 8, 64), generator=c["g"]).to(F16)
    want, wlse, size = plain.attention(c, q, [0, 1, 2], scale=0.3)
    wide = torch.zeros((2, 24, 64), dtype=F16, device="cuda")
    wide[:, 8:16] = q.to("cuda")
    tables = torch.full((2, 40), 1 << 29, dtype=torch.int32, device="cuda")
    tables[:, : c["tables"].shape[1]] = c["tables"].to("cuda")
    both = torch.stack([c["k"].transpose(1, 2), c["v"].transpose(1, 2)], 1).to("cuda")  # [page][2][token][head][dim]
    k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    room = torch.zeros((2, 10, 72), dtype=F16, device="cuda")
    out, lse = praghip.paged_decode(wide[:, 8:16], k, v, tables[:, : c["tables"].shape[1]], c["lengths"].to("cuda"),
                                    scale=0.3, lse=True, out=room[:, 1:9, :64])
    torch.cuda.synchronize()
    plain.check(out, want, size, F16, rounded=False)
    plain.check_lse(lse, wlse)
    assert not room[:, 0].any() and not room[:, 9].any() and not room[:, :, 64:].any()


def test_decode_masked_keys_may_hold_anything(gpu):
    """Infinities and NaN in keys and values that the window hides."""
    say("poisoned window")
    c = plain.make([200], 4, 2, 64, 16, BF16, seed=10)
    q = torch.randn((1, 4, 64), generator=c["g"]).to(BF16)
    want, wlse, size = plain.attention(c, q, [0, 1], window=70, sinks=5)
    for at in range(5, 130):
        for x, bad in (("k", math.inf), ("v", math.nan)):
            c[x][c["tables"][0, at // 16], :, at % 16] = bad
    out, lse = decode(c, q, window=70, sinks=5)
    plain.check(out, want, size, BF16, rounded=False)
    plain.check_lse(lse, wlse)


def test_decode_large_scores(gpu):
    """Scores in the hundreds: one key takes all, the exponentials of the others vanish."""
    say("large scores")
    c = plain.make([400, 50], 4, 2, 64, 16, F16, seed=11)
    c["k"] *= 30
    q = 30 * torch.randn((2, 4, 64), generator=c["g"]).to(F16)
    out, lse = decode(c, q)
    want, wlse, size = plain.attention(c, q, [0, 1, 2])
    # scores of some hundreds are sums of 64 products of up to 10^4: off by 64 2^-24 10^5,
    # which is relative in the probabilities
    got = out.double().cpu()
    assert ((got - want).abs() <= 2.0 ** -11 * want.abs() + 64 * 2.0 ** -24 * 1e5 * size).all()
    assert ((lse.double().cpu() - wlse).abs() <= 64 * 2.0 ** -24 * 1e5 + 1e-6 * wlse.abs()).all()


def test_decode_split_is_the_same_every_time(gpu):
    say("same bits")
    c = plain.make([5000, 100], 16, 8, 128, 16, BF16, seed=12)
    q = torch.randn((2, 16, 128), generator=c["g"]).to(BF16).to("cuda")
    k, v, tables, lengths = to_gpu(c)
    first = praghip.paged_decode(q, k, v, tables, lengths, lse=True)
    for _ in range(5):
        again = praghip.paged_decode(q, k, v, tables, lengths, lse=True)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


PROMPT = [
    # (before, rows) of each sequence, heads, kv, dim, page, window, sinks, type
    ([(0, 1)], 16, 8, 128, 16, 0, 0, BF16),
    ([(0, 2), (0, 1), (5, 3)], 2, 1, 64, 16, 0, 0, F16),
    ([(0, 77), (0, 0), (0, 41)], 16, 8, 128, 16, 0, 0, BF16),
    ([(0, 64), (0, 65), (0, 63)], 4, 4, 64, 32, 0, 0, F16),
    ([(0, 130)], 14, 2, 128, 16, 0, 0, BF16),
    ([(100, 30), (0, 0), (63, 1)], 8, 2, 64, 64, 0, 0, BF16),
    ([(600, 20), (900, 3)], 16, 8, 128, 16, 0, 0, F16),     # few rows, many keys: split
    ([(300, 5)], 4, 2, 256, 16, 0, 0, BF16),
    ([(0, 90)], 4, 2, 200, 16, 0, 0, F16),
    ([(40, 33)], 3, 1, 96, 16, 0, 0, BF16),
    ([(40, 33)], 5, 5, 8, 32, 0, 0, F16),
    ([(0, 300)], 4, 2, 64, 16, 50, 4, F16),
    ([(500, 100), (10, 7)], 16, 8, 128, 16, 64, 20, BF16),
    ([(500, 40)], 8, 4, 64, 64, 1, 0, BF16),
    ([(200, 150)], 4, 4, 64, 16, 128, 130, F16),           # sinks beyond the first tiles
    ([(700, 10)], 20, 1, 128, 128, 300, 1, BF16),
]


@pytest.mark.parametrize("parts,heads,kv,dim,page,window,sinks,type", PROMPT)
def test_prompt_against_64_bits(gpu, parts, heads, kv, dim, page, window, sinks, type):
    say("prompt", parts, heads, kv, dim, page, window, sinks, type)
    c = plain.make([a + b for a, b in parts], heads, kv, dim, page, type, seed=len(parts) * 1000 + dim + 1)
    starts = [sum(b for _, b in parts[:i]) for i in range(len(parts) + 1)]
    q = torch.randn((starts[-1], heads, dim), generator=c["g"]).to(type)
    out, lse = praghip.paged_prompt(q.to("cuda"), *to_gpu(c), torch.tensor(starts, dtype=torch.int32, device="cuda"),
                                    max(b for _, b in parts), window=window, sinks=sinks, lse=True)
    torch.cuda.synchronize()
    want, wlse, size = plain.attention(c, q, starts, window=window, sinks=sinks)
    plain.check(out, want, size, type, rounded=True)
    plain.check_lse(lse, wlse)


def test_prompt_rows_before_the_cache_and_missing_pages(gpu):
    """More new rows than tokens: the first see nothing.  Entries that are no page."""
    say("prompt rows before the cache")
    c = plain.make([20, 90], 4, 2, 64, 16, BF16, seed=21)
    c["tables"][1, 2] = -1
    q = torch.randn((60, 4, 64), generator=c["g"]).to(BF16)
    starts = [0, 30, 60]
    out, lse = praghip.paged_prompt(q.to("cuda"), *to_gpu(c), torch.tensor(starts, dtype=torch.int32, device="cuda"), 30,
                                    lse=True)
    torch.cuda.synchronize()
    want, wlse, size = plain.attention(c, q, starts)
    assert math.isinf(wlse[0, 0]) and not math.isinf(wlse[10, 0])
    plain.check(out, want, size, BF16, rounded=True)
    plain.check_lse(lse, wlse)


def test_prompt_of_one_row_is_the_decode(gpu):
    say("prompt of one row")
    lengths = [700, 1, 33]
    c = plain.make(lengths, 16, 8, 128, 16, BF16, seed=22)
    q = torch.randn((3, 16, 128), generator=c["g"]).to(BF16)
    starts = torch.arange(4, dtype=torch.int32, device="cuda")
    out = praghip.paged_prompt(q.to("cuda"), *to_gpu(c), starts, 1, window=100, sinks=2)
    want, _, size = plain.attention(c, q, [0, 1, 2, 3], window=100, sinks=2)
    plain.check(out, want, size, BF16, rounded=True)
    plain.check(praghip.paged_decode(q.to("cuda"), *to_gpu(c), window=100, sinks=2), want, size, BF16, rounded=False)


def test_prompt_strides(gpu):
    say("prompt strides")
    c = plain.make([150, 77], 8, 4, 64, 16, F16, seed=23, layout="pthd")
    q = torch.randn((60, 8, 64), generator=c["g"]).to(F16)
    starts = [0, 40, 60]
    want, _, size = plain.attention(c, q, starts, scale=0.2)
    wide = torch.zeros((60, 16, 64), dtype=F16, device="cuda")  # q beside k and v of a joint projection
    wide[:, :8] = q.to("cuda")
    room = torch.zeros((60, 8, 128), dtype=F16, device="cuda")
    k, v, tables, lengths = to_gpu(c)
    assert k.stride(1) == 64
    out = praghip.paged_prompt(wide[:, :8], k, v, tables, lengths, torch.tensor(starts, dtype=torch.int32, device="cuda"),
                               40, scale=0.2, out=room[:, :, :64])
    torch.cuda.synchronize()
    plain.check(out, want, size, F16, rounded=True)
    assert not room[:, :, 64:].any()


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1.0])
def test_scales(gpu, scale):
    """Negative scales turn the order of the scores; with 0 all visible keys weigh the same."""
    say("scale", scale)
    c = plain.make([150, 41], 8, 4, 64, 16, BF16, seed=28)
    q = (torch.randn((60, 8, 64), generator=c["g"]) * (0.1 if scale == 1.0 else 1)).to(BF16)
    starts = [0, 40, 60]
    want, wlse, size = plain.attention(c, q, starts, scale=scale, window=50, sinks=3)
    out, lse = praghip.paged_prompt(q.to("cuda"), *to_gpu(c), torch.tensor(starts, dtype=torch.int32, device="cuda"), 40,
                                    scale=scale, window=50, sinks=3, lse=True)
    plain.check(out, want, size, BF16, rounded=True)
    plain.check_lse(lse, wlse)
    want, wlse, size = plain.attention(c, q[:2], [0, 1, 2], scale=scale, window=50, sinks=3)
    out, lse = decode(c, q[:2], scale=scale, window=50, sinks=3)
    plain.check(out, want, size, BF16, rounded=False)
    plain.check_lse(lse, wlse)


@pytest.mark.parametrize("dim,type", [(64, BF16), (128, F16), (96, BF16), (256, F16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
def test_prompt_masked_keys_may_hold_anything(gpu, dim, type, window, sinks):
    """NaN and infinities in keys and values reach the rows that see them and no others:
    later rows of the same tile, earlier ones, and those whose window has moved on."""
    say("poisoned prompt", dim, type, window, sinks)
    n, rows, heads, kv = 230, 150, 4, 2
    c = plain.make([n], heads, kv, dim, 16, type, seed=dim + window)
    q = torch.randn((rows, heads, dim), generator=c["g"]).to(type)
    want, _, size = plain.attention(c, q, [0, rows], window=window, sinks=sinks)
    bad = {100: ("v", math.nan), 171: ("k", math.nan), 190: ("v", math.inf), 207: ("v", -math.inf)}
    for at, (x, value) in bad.items():
        c[x][c["tables"][0, at // 16], 1, at % 16, 5] = value
    out = praghip.paged_prompt(q.to("cuda"), *to_gpu(c), torch.tensor([0, rows], dtype=torch.int32, device="cuda"), rows,
                               window=window, sinks=sinks).cpu()
    place = torch.arange(n - rows, n)
    hit = torch.zeros(rows, dtype=torch.bool)
    for at in bad:
        hit |= (at <= place) & ((place - at < window) if window else torch.ones(rows, dtype=torch.bool))
    clean = torch.ones(rows, heads, dtype=torch.bool)
    clean[hit, 2:] = False  # the heads of key/value head 1
    assert bool(hit.any()) and not bool(hit.all())
    assert torch.isfinite(out[clean]).all()
    plain.check(out[clean], want[clean], size[clean], type, rounded=True)
    # column 5 of the rows that see a bad value is not finite
    assert not torch.isfinite(out[hit][:, 2:, 5].float()).any()


def test_prompt_over_a_long_cache(gpu):
    """More tiles than a workgroup keeps the pages of; few of the rows, by their definition."""
    say("long cache")
    n, rows = 70000, 300
    g = torch.Generator(device="cuda").manual_seed(29)
    k, v = (torch.randn((n // 16 + 2, 1, 16, 64), generator=g, device="cuda").to(F16) for _ in range(2))
    tables = torch.randperm(n // 16 + 2, generator=g, device="cuda").to(torch.int32)[None]
    q = torch.randn((rows, 1, 64), generator=g, device="cuda").to(F16)
    lengths, starts = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([n], [0, rows]))
    c = {"k": k.cpu(), "v": v.cpu(), "tables": tables.cpu(), "lengths": lengths.cpu(), "page": 16, "kv": 1}
    for window, sinks in ((0, 0), (40000, 3)):
        out = praghip.paged_prompt(q.repeat(1, 32, 1), k, v, tables, lengths, starts, rows, window=window, sinks=sinks)
        for row in (0, 150, 299):
            part = dict(c, lengths=torch.tensor([n - rows + row + 1]))
            want, _, size = plain.attention(part, q[row:row + 1].cpu(), [0, 1], window=window, sinks=sinks)
            for head in (0, 31):
                plain.check(out[row:row + 1, head:head + 1], want, size, F16, rounded=True)


def test_zero_sequences_and_rows(gpu):
    c = plain.make([20], 4, 2, 64, 16, BF16, seed=24)
    k, v, tables, lengths = to_gpu(c)
    q = torch.zeros((0, 4, 64), dtype=BF16, device="cuda")
    assert praghip.paged_decode(q, k, v, tables[:0], lengths[:0]).shape == (0, 4, 64)
    none = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert praghip.paged_prompt(q, k, v, tables, lengths, none, 5).shape == (0, 4, 64)


def test_another_stream(gpu):
    """Calls on a stream of their own, whose inputs are made on it, and many in a row."""
    say("another stream")
    c = plain.make([900, 50], 16, 8, 128, 16, BF16, seed=25)
    q = torch.randn((2, 16, 128), generator=c["g"]).to(BF16)
    want, _, size = plain.attention(c, q, [0, 1, 2])
    k, v, tables, lengths = to_gpu(c)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        qs = q.to("cuda", non_blocking=True)
        outs = [praghip.paged_decode(qs, k, v, tables, lengths) for _ in range(8)]
    one = praghip.paged_prompt(qs, k, v, tables, lengths, torch.arange(3, dtype=torch.int32, device="cuda"), 1,
                               stream=torch.cuda.current_stream()) if side.synchronize() is None else None
    given = torch.empty_like(qs)
    torch.cuda.synchronize()
    praghip.paged_decode(qs, k, v, tables, lengths, out=given, stream=side)
    torch.cuda.synchronize()
    for o in outs + [given]:
        plain.check(o, want, size, BF16, rounded=False)
    plain.check(one, want, size, BF16, rounded=True)


def test_graph_replays(gpu):
    """A captured decode and prompt follow lengths that change between the replays."""
    say("graph")
    c = plain.make([500, 300, 40], 8, 4, 64, 16, BF16, seed=26)
    q = torch.randn((3, 8, 64), generator=c["g"]).to(BF16).to("cuda")
    k, v, tables, lengths = to_gpu(c)
    starts = torch.arange(4, dtype=torch.int32, device="cuda")
    a, b = torch.empty_like(q), torch.empty_like(q)

    def work(a, b):
        praghip.paged_decode(q, k, v, tables, lengths, out=a)
        praghip.paged_prompt(q, k, v, tables, lengths, starts, 1, out=b)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(a, b)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work(a, b)
    for held in ([500, 300, 40], [1, 0, 39], [499, 17, 2], [500, 300, 40]):
        lengths.copy_(torch.tensor(held, dtype=torch.int32))
        ea, eb = torch.empty_like(q), torch.empty_like(q)
        work(ea, eb)
        torch.cuda.synchronize()
        a.zero_()
        b.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, ea) and torch.equal(b, eb), held


def test_refusals(gpu):
    c = plain.make([20, 30], 4, 2, 64, 16, BF16, seed=27)
    k, v, tables, lengths = to_gpu(c)
    q = torch.zeros((2, 4, 64), dtype=BF16, device="cuda")
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")

    def refused(text, call):
        with pytest.raises(praghip.PraghipError) as e:
            call()
        assert text in e.value.text, e.value.text

    D, P = praghip.paged_decode, praghip.paged_prompt
    refused("E_ATTENTION_TYPE", lambda: D(q.float(), k, v, tables, lengths))
    refused("E_ATTENTION_TYPE", lambda: D(q.half(), k, v, tables, lengths))
    refused("E_ATTENTION_SHAPE", lambda: D(q[:1], k, v, tables, lengths))
    refused("E_ATTENTION_SHAPE", lambda: D(q[:, :3].contiguous(), k, v, tables, lengths))
    refused("E_ATTENTION_SHAPE", lambda: D(q[..., :32].contiguous(), k, v, tables, lengths))
    refused("E_ATTENTION_SHAPE", lambda: D(q.transpose(1, 2), k, v, tables, lengths))
    refused("E_ATTENTION_SHAPE", lambda: D(q, k, v[:, :1], tables, lengths))
    refused("E_ATTENTION_SHAPE", lambda: D(q, k, v, tables[:1], lengths))
    refused("E_ATTENTION_INTS", lambda: D(q, k, v, tables.long(), lengths))
    refused("E_ATTENTION_INTS", lambda: D(q, k, v, tables.cpu(), lengths))
    refused("E_ATTENTION_DEVICE", lambda: D(q, k.cpu(), v, tables, lengths))
    refused("E_ATTENTION_SHAPE", lambda: D(q, k, v, tables, lengths, window=-1))
    refused("E_ATTENTION_SHAPE", lambda: D(q, k, v, tables, lengths, scale=math.nan))
    refused("E_ATTENTION_OUT", lambda: D(q, k, v, tables, lengths, out=q.half()))
    # pages of 24 tokens; rows that are not on 16 bytes
    odd = torch.zeros((3, 2, 24, 64), dtype=BF16, device="cuda")
    refused("E_ATTENTION_SHAPE", lambda: D(q, odd, odd, tables, lengths))
    wide = torch.zeros((2, 4, 68), dtype=BF16, device="cuda")
    refused("E_ATTENTION_ALIGNMENT", lambda: D(wide[..., :64], k, v, tables, lengths))
    flat = torch.zeros(2 * 4 * 64 + 4, dtype=BF16, device="cuda")
    refused("E_ATTENTION_ALIGNMENT", lambda: D(flat[4:].view(2, 4, 64), k, v, tables, lengths))
    refused("E_ATTENTION_SHAPE", lambda: P(q, k, v, tables, lengths, starts[:2], 1))
    refused("E_ATTENTION_INTS", lambda: P(q, k, v, tables, lengths, starts.long(), 1))
    refused("E_ATTENTION_SHAPE", lambda: P(q, k, v, tables, lengths, starts, -1))
