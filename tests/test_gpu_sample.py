"""sample_tokens against the definition in 64 bits: the same tokens, whatever the vocabulary, the
type, the filters, ties and values that are no numbers.

Both sides' weights are off by some 2^-42 of themselves, so a row's token could differ where its
random number, or a cut, falls within vocab x 2^-42 of a border: below 10^-6 a row.  Where borders
are hit on purpose (equal logits) the sums are exact on both sides."""
import math

import numpy as np
import pytest
import torch

import praghip

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def plain(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row's token."""
    x = logits.double().numpy()
    x = np.minimum(np.where(np.isnan(x), -np.inf, x), float(torch.finfo(F32).max))
    top = x.max()
    if top == -np.inf:
        return -1
    if not temperature > 0:
        return int(np.argmax(x))
    with np.errstate(over="ignore", invalid="ignore"):
        w = np.where(x == top, 1.0, np.exp((x - top) / temperature))
    w[x == -np.inf] = 0
    order = np.argsort(-x, kind="stable")
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        sums = np.cumsum(w[order])
        order = order[: 1 + int(np.count_nonzero(sums[:-1] < np.float64(top_p) * sums[-1]))]
    if min_p > 0:
        order = order[w[order] >= min(min_p, 1.0)]
    order = np.sort(order)
    order = order[w[order] > 0]
    sums = np.cumsum(w[order])
    return int(order[min(int(np.count_nonzero(sums <= np.float64(u) * sums[-1])), len(order) - 1)])


def f32(x):
    return float(np.float32(x))


def check(logits, uniform, **filters):
    """All rows; filters are numbers or lists."""
    rows = len(logits)
    each = {n: v if isinstance(v, list) else [v] * rows for n, v in filters.items()}
    want = [plain(logits[i].cpu(), f32(uniform[i]), **{n: f32(v[i]) if n != "top_k" else v[i] for n, v in each.items()}) for i in range(rows)]
    given = {n: torch.tensor(v, dtype=torch.int32 if n == "top_k" else F32, device="cuda") if isinstance(v, list) else v
             for n, v in filters.items()}
    got = praghip.sample_tokens(logits.cuda(), torch.tensor(uniform, dtype=F32, device="cuda"), **given)
    assert got.dtype == torch.int64
    assert got.tolist() == want, [(i, a, b, uniform[i]) for i, (a, b) in enumerate(zip(got.tolist(), want)) if a != b]
    return want


def make(rows, vocab, type, seed, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g) * spread
    at = torch.randint(0, vocab, (rows, min(vocab, 9)), generator=g)
    x.scatter_add_(1, at, torch.rand(at.shape, generator=g) * 5 * spread)
    return x.to(type), torch.rand(rows, generator=g).tolist()


FILTERS = [{}, {"temperature": 0.6}, {"top_k": 1}, {"top_k": 40, "temperature": 1.3}, {"top_p": 0.9}, {"top_p": 0.4, "temperature": 2.0},
           {"min_p": 0.05}, {"top_k": 60, "top_p": 0.8, "min_p": 0.02, "temperature": 0.8}, {"top_k": 7, "top_p": 0.97},
           {"top_p": 0.999, "min_p": 0.3}, {"top_k": 3000, "min_p": 1e-4}, {"temperature": 0.0, "top_k": 5}]


@pytest.mark.parametrize("vocab", [1, 2, 3, 8, 9, 63, 1000, 16383, 16384, 16385, 32768, 50257, 155648])
@pytest.mark.parametrize("type", [BF16, F16, F32])
def test_vocabularies(gpu, vocab, type):
    print("[sample]", vocab, type, flush=True)
    for i, filters in enumerate(FILTERS):
        logits, u = make(5 if vocab < 50000 else 3, vocab, type, seed=vocab + 100 * i)
        check(logits, u, **filters)


@pytest.mark.parametrize("spread", [0.0, 0.01, 0.5, 1.0, 6.0, 30.0])
def test_spreads(gpu, spread):
    """From flat rows, where nearly every token is a candidate, to rows of one that counts."""
    print("[sample] spread", spread, flush=True)
    for i, filters in enumerate(({}, {"top_p": 0.95}, {"top_k": 20000}, {"top_k": 20000, "top_p": 0.7}, {"min_p": 0.4})):
        logits, u = make(4, 40000, F32, seed=i, spread=spread)
        check(logits, u, **filters)
        check(logits.to(BF16), u, **filters)


def test_the_largest_vocabulary(gpu):
    logits, u = make(2, 2 ** 20, BF16, seed=1, spread=1.5)
    for filters in ({}, {"top_p": 0.9, "top_k": 100000}, {"min_p": 0.001}):
        check(logits, u, **filters)


@pytest.mark.parametrize("rows", [1, 7, 64, 300])
def test_rows_of_their_own_filters(gpu, rows):
    print("[sample] rows", rows, flush=True)
    logits, u = make(rows, 3001, BF16, seed=rows)
    g = np.random.default_rng(rows)
    check(logits, u, temperature=[float(x) for x in g.choice([0.0, 0.3, 1.0, 1.7], rows)],
          top_k=[int(x) for x in g.choice([0, -3, 1, 5, 200, 3000, 3001, 2 ** 31 - 1], rows)],
          top_p=[float(x) for x in g.choice([0.0, 0.1, 0.5, 0.95, 1.0, 7.0], rows)],
          min_p=[float(x) for x in g.choice([-1.0, 0.0, 0.01, 0.2, 1.0, 3.0], rows)])


@pytest.mark.parametrize("vocab", [1, 5, 64, 1000, 40000])
@pytest.mark.parametrize("value", [0.0, -7.25, 1e4])
def test_equal_logits(gpu, vocab, value):
    """Ties: the lower indexes stay, and sums are exact, so that borders are hit."""
    print("[sample] equal", vocab, value, flush=True)
    u = [0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1.0]
    logits = torch.full((len(u), vocab), value)
    for filters in ({}, {"top_k": 3}, {"top_k": max(1, vocab // 2)}, {"top_p": 0.5}, {"top_p": 0.25, "top_k": max(1, vocab - 1)}, {"min_p": 1.0}):
        want = check(logits, u, **filters)
        if not filters and vocab == 64:
            assert want[:4] == [0, 16, 32, 48] and want[5] == 63


def test_few_values(gpu):
    """Logits of a handful of values, as 8-bit models have them: each cut falls among ties."""
    g = torch.Generator().manual_seed(2)
    logits = torch.randint(-6, 3, (40, 30000), generator=g).float()
    u = torch.rand(40, generator=g).tolist()
    for filters in ({}, {"top_k": 5000}, {"top_p": 0.3}, {"top_p": 0.77, "top_k": 9000}, {"min_p": f32(math.exp(-2.5))}):
        check(logits, u, **filters)


@pytest.mark.parametrize("near", [1, 2, 63, 64, 65, 127, 128, 129, 300, 1100, 5000])
def test_tokens_near_a_cut(gpu, near):
    """So many logits within 1/100, some of them equal, among lower ones: cuts fall among them."""
    print("[sample] near a cut", near, flush=True)
    g = torch.Generator().manual_seed(near)
    logits = torch.randn((6, 12000), generator=g) - 9
    for row in logits:
        row[torch.randperm(12000, generator=g)[:near]] = 2 + torch.randint(0, 40, (near,), generator=g) / 4000
    u = torch.rand(6, generator=g).tolist()
    some = max(1, near // 2)
    for filters in ({"top_k": 1}, {"top_k": some}, {"top_k": near}, {"top_k": near + 3}, {"top_p": 0.3}, {"top_p": 0.6, "top_k": some},
                    {"top_p": 0.99, "top_k": near}, {"top_k": some, "top_p": 0.5, "min_p": f32(0.995)}):
        check(logits, u, **filters)


def test_masked_and_values_that_are_no_numbers(gpu):
    inf, nan, low = math.inf, math.nan, float(torch.finfo(BF16).min)
    logits, u = make(10, 20000, BF16, seed=3)
    logits[0] = -inf
    logits[1] = nan
    logits[2], logits[2, 17000] = -inf, -3.0
    logits[3] = low                      # all of the type's lowest value: any of them
    logits[4, :19000] = -inf
    logits[5, ::3] = nan
    logits[6, [5, 19999]] = inf          # the two share everything
    logits[7], logits[7, 18000:] = low, -1.0
    logits[8], logits[8, 19999] = -inf, low
    logits[9, 16384:] = -1e4             # a part whose weights are all nothing
    for filters in ({}, {"top_k": 50}, {"top_p": 0.9}, {"min_p": 0.1}, {"top_k": 100, "top_p": 0.5, "temperature": 0.7}, {"temperature": 0.0}):
        want = check(logits, u, **filters)
        assert want[:3] == [-1, -1, 17000] and want[6] in (5, 19999) and want[8] == 19999
    logits = logits.half().float()
    logits[3] = -3.4e38
    check(logits, u, top_p=0.9)


@pytest.mark.parametrize("temperature", [1e-30, 1e-6, 0.01, 100.0, 1e30, math.inf])
def test_temperatures(gpu, temperature):
    logits, u = make(6, 20000, F32, seed=4)
    for filters in ({}, {"top_p": 0.9}, {"top_k": 11}):
        check(logits, u, temperature=temperature, **filters)


@pytest.mark.parametrize("size", [1e3, 1e6, 1e20, 3e38])
def test_large_logits(gpu, size):
    """Differences far beyond the weights' range, ties of the largest value among them."""
    g = torch.Generator().manual_seed(5)
    logits = (torch.rand((6, 20000), generator=g) * 2 - 1) * size
    logits[2:4, [3, 9000, 19000]] = size
    logits[4] = -size
    u = torch.rand(6, generator=g).tolist()
    for filters in ({}, {"top_k": 3}, {"top_p": 0.9}, {"min_p": 0.5}):
        check(logits, u, **filters)


def test_the_distribution(gpu):
    """As many of an even grid of random numbers draw a token as its probability says."""
    n, vocab = 4096, 37
    logits, _ = make(1, vocab, F32, seed=6, spread=1.0)
    u = ((torch.arange(n) + 0.5) / n).cuda()
    got = praghip.sample_tokens(logits.cuda().expand(n, -1).contiguous(), u, temperature=0.9)
    count = torch.bincount(got.cpu(), minlength=vocab).double()
    p = torch.softmax(logits[0].double() / f32(0.9), 0)
    assert bool(((count - n * p).abs() <= 1.0 + 1e-6).all())


def test_strides_and_results(gpu):
    logits, u = make(5, 2003, F16, seed=7)
    want = check(logits, u, top_p=0.9)
    wide = torch.full((9, 4100), 9.0, dtype=F16, device="cuda")
    wide[::2, 33: 33 + 2003] = logits.cuda()
    out = torch.full((9,), 7, dtype=torch.int64, device="cuda")
    got = praghip.sample_tokens(wide[::2, 33: 33 + 2003], torch.tensor(u, device="cuda"), top_p=0.9, out=out[2:7])
    assert got.data_ptr() == out[2:].data_ptr() and out.tolist() == [7, 7] + want + [7, 7]
    # one row for all, by a stride of 0
    row = logits[:1].cuda().expand(5, -1)
    assert praghip.sample_tokens(row, torch.tensor(u, device="cuda")).tolist() == [plain(logits[0], f32(x)) for x in u]


def test_a_captured_call(gpu):
    """Replayed with other logits, numbers and filters, against the eager call."""
    logits, u = make(9, 70000, BF16, seed=8)
    x, uniform = logits.cuda(), torch.tensor(u, device="cuda")
    made = {"temperature": torch.full((9,), 0.8, device="cuda"), "top_k": torch.full((9,), 50, dtype=torch.int32, device="cuda"),
            "top_p": torch.full((9,), 0.9, device="cuda"), "min_p": torch.zeros(9, device="cuda")}
    praghip.sample_tokens(x, uniform, **made)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = praghip.sample_tokens(x, uniform, **made)
    for seed in range(9, 13):
        logits, u = make(9, 70000, BF16, seed=seed)
        x.copy_(logits), uniform.copy_(torch.tensor(u))
        made["top_k"].fill_(seed - 9)
        graph.replay()
        torch.cuda.synchronize()
        assert got.tolist() == praghip.sample_tokens(x, uniform, **made).tolist()
        assert got.tolist() == [plain(logits[i], f32(u[i]), f32(0.8), seed - 9, f32(0.9)) for i in range(9)]


def test_logits_and_workspace_beyond_32_bits(gpu):
    """2.2 x 10^9 logits, whose candidates' list is 8.7 GB: the same tokens as row by row."""
    rows, vocab = 14000, 155648
    g = torch.Generator(device="cuda").manual_seed(4)
    logits = torch.empty((rows, vocab), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    uniform = torch.rand(rows, device="cuda", generator=g)
    draw = dict(temperature=0.9, top_k=5000, top_p=0.9, min_p=1e-4)
    got = praghip.sample_tokens(logits, uniform, **draw)
    for first in (0, rows // 2, rows - 300):
        some = slice(first, first + 300)
        assert torch.equal(got[some], praghip.sample_tokens(logits[some], uniform[some], **draw))


def test_refusals(gpu):
    logits, u = torch.zeros((3, 40), device="cuda"), torch.zeros(3, device="cuda")

    def refused(text, *args, **kw):
        with pytest.raises(praghip.PraghipError) as e:
            praghip.sample_tokens(*args, **kw)
        assert e.value.text == text, e.value.text

    for bad in ((logits[0], u), (logits, u[:2]), (logits, u[None]), (logits.t(), u), (logits[:, ::2], u), (logits, u.repeat(2)[::2])):
        refused("E_SAMPLE_SHAPE", *bad)
    refused("E_SAMPLE_SHAPE", logits[:, :0], u)
    refused("E_SAMPLE_SHAPE", torch.zeros((1, 2 ** 20 + 1), device="cuda"), u[:1])
    refused("E_SAMPLE_SHAPE", logits[:1].expand(65536, -1), torch.zeros(65536, device="cuda"))
    for bad in ((logits.double(), u), (logits.long(), u), (logits, u.double()), (logits, u.half())):
        refused("E_SAMPLE_TYPE", *bad)
    for bad in ((logits, u.cpu()), (logits.cpu(), u.cpu())):
        refused("E_SAMPLE_DEVICE", *bad)
    for name in ("temperature", "top_p", "min_p"):
        refused("E_SAMPLE_TYPE", logits, u, **{name: u.double()})
        refused("E_SAMPLE_DEVICE", logits, u, **{name: u.cpu()})
        refused("E_SAMPLE_SHAPE", logits, u, **{name: u[:2]})
        refused("E_SAMPLE_FILTER", logits, u, **{name: -0.5})
        refused("E_SAMPLE_FILTER", logits, u, **{name: math.nan})
        refused("E_SAMPLE_GRADIENT", logits, u, **{name: u.clone().requires_grad_()})
    refused("E_SAMPLE_FILTER", logits, u, min_p=1.5)
    refused("E_SAMPLE_FILTER", logits, u, top_k=-1)
    refused("E_SAMPLE_TYPE", logits, u, top_k=u.long())
    for out in (torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(3, dtype=torch.int64)):
        refused("E_SAMPLE_OUT", logits, u, out=out)
    refused("E_SAMPLE_GRADIENT", logits.clone().requires_grad_(), u)
    with torch.no_grad():
        assert praghip.sample_tokens(logits.clone().requires_grad_(), u).tolist() == [0, 0, 0]
    assert praghip.sample_tokens(logits[:0], u[:0]).shape == (0,)
