"""page_append against 64 bits: layouts of the rotation, norms, heads, strides, places without a
page, and everything that it is not to touch."""
import pytest
import torch

import praghip

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
UNIT = {BF16: 2.0 ** -8, F16: 2.0 ** -11}
# Sums of up to 256 squares by 8 values a lane and 5 exchanges: 13 roundings, a root, a quotient
# and products: below 2^-19 of each of a pair's products, which are added.
SUMS = 2.0 ** -19


def make(rows, before, heads, kv, dim, half, type, page=16, seed=0, norms=(True, True), spare=3, extra=0, before_rows=0, layout="phtd"):
    """Sequences with rows[s] new tokens after before[s]; `before_rows` and `extra` rows of no
    stretch around them."""
    g = torch.Generator().manual_seed(seed)
    lengths = [a + b for a, b in zip(rows, before)]
    need = [-(-n // page) for n in lengths]
    width = max(need + [1]) + 1
    count = sum(need) + spare
    tables = torch.full((len(rows), width), -1, dtype=torch.int32)
    order, at = torch.randperm(count, generator=g).to(torch.int32), 0
    for s, n in enumerate(need):
        tables[s, :n] = order[at: at + n]
        at += n
    starts = [before_rows + sum(rows[:s]) for s in range(len(rows) + 1)]
    joint = torch.randn((starts[-1] + extra, heads + 2 * kv, dim), generator=g).to(type)
    pools = [torch.randn((count, kv, page, dim), generator=g).to(type) for _ in "kv"]
    if layout == "pthd":
        pools = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in pools]
    cos, sin = praghip.rotary_table(width * page, 2 * half, device="cpu")
    return {"q": joint[:, :heads], "k": joint[:, heads: heads + kv], "v": joint[:, heads + kv:], "pools": pools, "tables": tables,
            "lengths": torch.tensor(lengths, dtype=torch.int32), "starts": torch.tensor(starts, dtype=torch.int32), "cos": cos, "sin": sin,
            "norms": [(1 + 0.3 * torch.randn(dim, generator=g)).to(type) if x else None for x in norms]}


def turned(x, norm, cos, sin, interleaved, eps):
    """One token's heads in 64 bits, and for each value the products' sizes."""
    x = x.double()
    if norm is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * norm.double()
    y, size = x.clone(), x.abs()
    half = cos.numel()
    i = torch.arange(half)
    one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    a, b, c, s = x[..., one], x[..., two], cos.double(), sin.double()
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    size[..., one], size[..., two] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, size


def check(m, interleaved=False, eps=1e-6, out=None):
    type = m["q"].dtype
    page, (tokens, heads, dim) = m["pools"][0].shape[2], m["q"].shape
    dev = {x: t.cuda() if x not in ("pools", "norms") else [None if p is None else p.cuda() for p in t] for x, t in m.items()}
    if m["pools"][0].stride(2) != dim:  # (copies keep the strides of dense memory)
        assert dev["pools"][0].stride() == m["pools"][0].stride()
    marked = torch.full((tokens, heads, dim), 5.0, dtype=type, device="cuda") if out is None else out(dev)
    got = praghip.page_append(dev["q"], dev["k"], dev["v"], *dev["pools"], dev["tables"], dev["lengths"], dev["starts"], dev["cos"],
                              dev["sin"], q_norm=dev["norms"][0], k_norm=dev["norms"][1], eps=eps, interleaved=interleaved, out=marked)
    assert got is marked
    got = got.cpu().double()
    want = [p.double().clone() for p in m["pools"]]
    bound = [torch.zeros_like(p) for p in want]
    written = torch.zeros(tokens, dtype=torch.bool)
    starts = m["starts"].tolist()
    for s, n in enumerate(m["lengths"].tolist()):
        for row in range(starts[s], starts[s + 1]):
            written[row] = True
            at = n - (starts[s + 1] - row)
            place = min(max(at, 0), m["cos"].shape[0] - 1)
            y, size = turned(m["q"][row], m["norms"][0], m["cos"][place], m["sin"][place], interleaved, eps)
            err = (got[row] - y).abs() / (UNIT[type] * y.abs() + SUMS * size + 2.0 ** -25)
            assert float(err.max()) <= 1, (s, row, float(err.max()))
            if at < 0 or at // page >= m["tables"].shape[1]:
                continue
            entry = int(m["tables"][s, at // page])
            if not 0 <= entry < len(want[0]):
                continue
            y, size = turned(m["k"][row], m["norms"][1], m["cos"][place], m["sin"][place], interleaved, eps)
            want[0][entry, :, at % page] = y
            bound[0][entry, :, at % page] = UNIT[type] * y.abs() + SUMS * size + 2.0 ** -25
            want[1][entry, :, at % page] = m["v"][row].double()
    for pool, w, b in zip(dev["pools"], want, bound):  # (places without a new key have a bound of 0)
        assert bool(((pool.cpu().double() - w).abs() <= b).all())
    if out is None:
        assert bool((got[~written] == 5.0).all())
    return dev


SHAPES = [(16, 8, 128, 64), (16, 8, 128, 32), (32, 4, 64, 32), (4, 4, 8, 4), (3, 1, 24, 12), (12, 1, 96, 48), (12, 2, 96, 12), (6, 3, 80, 40),
          (28, 4, 128, 64), (8, 2, 256, 128), (8, 2, 256, 24), (5, 5, 136, 68), (2, 1, 64, 0), (2, 2, 72, 5)]


@pytest.mark.parametrize("heads,kv,dim,half", SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_shapes(gpu, heads, kv, dim, half, interleaved):
    print("[append]", heads, kv, dim, half, interleaved, flush=True)
    for type, norms in ((BF16, (True, True)), (F16, (False, False))):
        check(make([1, 7, 0, 20], [40, 0, 3, 13], heads, kv, dim, half, type, seed=dim + half, norms=norms), interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("half", [16, 20, 21])
def test_infinities_stay_in_their_pairs(gpu, half, interleaved):
    """A head's first values are turned; infinite ones reach no value behind them."""
    m = make([4], [9], 4, 2, 64, half, BF16, seed=half, norms=(False, False))
    finite = m["q"].clone()
    m["q"][:, 1, 0], m["q"][:, 2, 2 * half - 1], m["k"][:, 0, 1] = float("inf"), float("-inf"), float("nan")
    cache = [p.cuda() for p in m["pools"]]
    rest = [m[x].cuda() for x in ("tables", "lengths", "starts", "cos", "sin")]
    got = praghip.page_append(m["q"].cuda(), m["k"].cuda(), m["v"].cuda(), *cache, *rest, interleaved=interleaved).cpu()
    assert torch.equal(got[..., 2 * half:], finite[..., 2 * half:])
    place = m["tables"][0, 0]  # of positions 9 .. 12
    assert torch.equal(cache[0][place, :, 9:13].transpose(0, 1).cpu()[..., 2 * half:], m["k"][..., 2 * half:])
    others = [h for h in range(4) if h not in (1, 2)]
    assert bool(got[:, others].isfinite().all())


@pytest.mark.parametrize("norms", [(True, False), (False, True)])
def test_one_norm(gpu, norms):
    check(make([3, 2], [5, 16], 4, 2, 64, 32, F16, seed=1, norms=norms), eps=1e-3)


@pytest.mark.parametrize("rows,before,page", [([1], [0], 16), ([1] * 64, [i * 7 for i in range(64)], 16), ([300], [0], 16), ([513, 1, 90], [1, 0, 700], 64),
                                             ([129] * 5, [0, 15, 16, 17, 127], 128)])
def test_lengths(gpu, rows, before, page):
    print("[append] lengths", len(rows), page, flush=True)
    check(make(rows, before, 8, 4, 128, 64, BF16, page=page, seed=2))


@pytest.mark.parametrize("layout", ["phtd", "pthd"])
def test_rows_of_no_stretch(gpu, layout):
    check(make([4, 9], [20, 1], 6, 2, 64, 16, BF16, seed=3, before_rows=3, extra=5, layout=layout))


def test_no_tokens_and_no_sequences(gpu):
    m = make([0, 0], [20, 0], 4, 2, 64, 32, BF16, seed=4)
    check(m)
    for x, shape in (("tables", (0, 3)), ("lengths", (0,)), ("starts", (1,))):
        m[x] = torch.zeros(shape, dtype=torch.int32)
    check(m)
    m = make([], [], 4, 2, 64, 32, BF16, seed=4, extra=3)
    check(m)


def test_places_without_a_page(gpu):
    """Entries that are no page, more rows than positions, and lengths beyond the tables."""
    m = make([20, 20, 20, 5], [30, 0, 40, 0], 4, 2, 64, 32, BF16, seed=5)
    m["tables"][0, 2] = -1
    m["tables"][0, 3] = -7
    m["tables"][2, 3] = len(m["pools"][0])
    m["tables"][2, 2] = 2 ** 31 - 1
    m["lengths"][1] = 12           # eight rows at positions below 0
    m["lengths"][3] = m["tables"].shape[1] * 16 + 3  # three rows beyond the tables
    check(m)
    m["lengths"][1], m["lengths"][3] = -2 ** 31, 2 ** 31 - 1
    check(m)


@pytest.mark.parametrize("interleaved,half", [(False, 64), (False, 20), (True, 64)])
def test_in_place(gpu, interleaved, half):
    """The queries over themselves, a view of the joint projection whose other columns stay."""
    m = make([3, 130], [9, 50], 16, 8, 128, half, BF16, seed=6)
    m["joint"] = torch.cat((m["q"], m["k"], m["v"]), 1)
    base = m["joint"].cuda()

    def out(dev):
        dev["q"], dev["k"], dev["v"] = base[:, :16], base[:, 16:24], base[:, 24:]
        return dev["q"]

    check(m, interleaved, out=out)
    assert torch.equal(base[:, 16:].cpu(), m["joint"][:, 16:])


def test_strided_results(gpu):
    m = make([2, 9], [5, 6], 4, 2, 64, 32, F16, seed=7)
    wide = torch.full((11, 9, 80), 5.0, dtype=F16, device="cuda")
    check(m, out=lambda dev: wide[:, ::2][:, :4, 8:72])
    wide[:, ::2][:, :4, 8:72] = 5.0
    assert bool((wide == 5.0).all())


def test_far_positions(gpu):
    """A cache of more than 2^31 values, and positions whose angles 32 bits would not hold."""
    pages, page, kv, dim = 270000, 64, 2, 64
    assert pages * page * kv * dim > 2 ** 31
    k, v = (torch.zeros((pages, kv, page, dim), dtype=BF16, device="cuda") for _ in "kv")
    tables = torch.full((2, 16384), -1, dtype=torch.int32, device="cuda")
    tables[0, 16383], tables[1, 0] = pages - 1, pages - 2
    cos, sin = praghip.rotary_table(16384 * page, dim)
    g = torch.Generator().manual_seed(8)
    q, new, value = (torch.randn((2, n, dim), generator=g).to(BF16).cuda() for n in (4, kv, kv))
    lengths = torch.tensor([16384 * page, 1], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    got = praghip.page_append(q, new, value, k, v, tables, lengths, starts, cos, sin)
    for s, (entry, row, place) in enumerate(((pages - 1, page - 1, 16384 * page - 1), (pages - 2, 0, 0))):
        angle = place * 1e6 ** (-torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))
        for x, y in ((q[s], got[s]), (new[s], k[entry, :, row])):
            a, b = x.cpu().double().chunk(2, -1)
            want = torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)
            size = (a.abs() + b.abs()).repeat(1, 2)
            assert bool(((y.cpu().double() - want).abs() <= UNIT[BF16] * want.abs() + 2.0 ** -22 * size).all())
        assert torch.equal(v[entry, :, row], value[s])
        k[entry, :, row], v[entry, :, row] = 0, 0
    assert not bool(k[pages - 2:].any()) and not bool(v[pages - 2:].any()) and not bool(k[:100].any())


def test_a_captured_call(gpu):
    """Replayed with other tokens and lengths, against the eager call."""
    m = make([1] * 4, [3, 40, 15, 16], 16, 8, 128, 64, BF16, seed=9)
    dev = {x: t.cuda() if x not in ("pools", "norms") else [p.cuda() for p in t] for x, t in m.items()}
    base = torch.randn((4, 32, 128), device="cuda").to(BF16)

    def call():
        return praghip.page_append(base[:, :16], base[:, 16:24], base[:, 24:], *dev["pools"], dev["tables"], dev["lengths"], dev["starts"],
                                   dev["cos"], dev["sin"], q_norm=dev["norms"][0], k_norm=dev["norms"][1])

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for step in range(4):
        base.copy_(torch.randn_like(base))
        dev["lengths"].copy_(m["lengths"] - step)
        kept = [p.clone() for p in dev["pools"]]
        graph.replay()
        torch.cuda.synchronize()
        after = [p.clone() for p in dev["pools"]]
        for p, k in zip(dev["pools"], kept):
            p.copy_(k)
        assert torch.equal(call(), got)
        assert all(torch.equal(a, b) for a, b in zip(dev["pools"], after))


def test_refusals(gpu):
    m = make([2, 3], [5, 6], 4, 2, 64, 32, BF16, seed=10)
    dev = [m["q"].cuda(), m["k"].cuda(), m["v"].cuda(), *(p.cuda() for p in m["pools"]), *(m[x].cuda() for x in ("tables", "lengths", "starts",
                                                                                                                 "cos", "sin"))]
    w = m["norms"][0].cuda()

    def refused(text, at=None, t=None, **kw):
        args = list(dev)
        if at is not None:
            args[at] = t
        with pytest.raises(praghip.PraghipError) as e:
            praghip.page_append(*args, **kw)
        assert e.value.text == text, e.value.text

    q, k, v, kp, vp, tables, lengths, starts, cos, sin = dev
    for at, t in ((0, q[0]), (0, q[:4]), (0, q[..., :56]), (0, q[:, :0]), (1, k[:, :1]), (1, k[0]), (2, v[:4]), (2, v[..., :32]), (3, kp[0]),
                  (4, vp[:2]), (5, tables[0]), (6, lengths[:1]), (7, starts[:2]), (7, starts[None]), (0, q.transpose(1, 2).contiguous().transpose(1, 2))):
        refused("E_ATTENTION_SHAPE", at, t)
    for at, t in ((0, q.half()), (0, q.float()), (1, k.half()), (2, v.float()), (3, kp.half()), (4, vp.half())):
        refused("E_ATTENTION_TYPE", at, t)
    for at, t in ((1, k.cpu()), (3, kp.cpu()), (4, vp.cpu())):
        refused("E_ATTENTION_DEVICE", at, t)
    for at, t in ((5, tables.long()), (6, lengths.cpu()), (7, starts.long())):
        refused("E_ATTENTION_INTS", at, t)
    for at, t in ((8, cos.double()), (9, sin.to(BF16))):
        refused("E_ROTARY_TYPE", at, t)
    refused("E_ROTARY_DEVICE", 8, cos.cpu())
    for at, t in ((8, cos[0]), (9, sin[:-1]), (8, cos[:, :5]), (8, cos.t().contiguous().t())):
        refused("E_ROTARY_SHAPE", at, t)
    dev[8], dev[9] = cos[:-1], sin[:-1]  # shorter than the tables' positions
    refused("E_ROTARY_SHAPE")
    dev[8], dev[9] = torch.zeros((len(cos), 33), device="cuda"), torch.zeros((len(cos), 33), device="cuda")
    refused("E_ROTARY_SHAPE")
    dev[8], dev[9] = cos, sin
    refused("E_ROTARY_SHAPE", eps=-1.0)
    refused("E_ATTENTION_SHAPE", q_norm=w[:32])
    refused("E_ATTENTION_SHAPE", k_norm=w.repeat(2)[::2])
    refused("E_ATTENTION_TYPE", k_norm=w.float())
    refused("E_ATTENTION_DEVICE", q_norm=w.cpu())
    refused("E_ATTENTION_OUT", out=q[:2])
    refused("E_ATTENTION_ALIGNMENT", out=torch.zeros(5 * 4 * 64 + 1, dtype=BF16, device="cuda")[1:].view(5, 4, 64))
    refused("E_ATTENTION_ALIGNMENT", q_norm=w.repeat(2)[1:65])
    for at, t in ((0, q), (1, k), (2, v), (3, kp), (4, vp), (8, cos), (9, sin)):
        refused("E_ATTENTION_GRADIENT", at, t.clone().requires_grad_())
    refused("E_ATTENTION_GRADIENT", k_norm=w.clone().requires_grad_())
    with torch.no_grad():
        assert not praghip.page_append(q.clone().requires_grad_(), *dev[1:]).requires_grad


def test_more_workgroups_than_a_grid_row_has_threads_for(gpu):
    """2^24 workgroups of 256 threads; all but the last tokens stand before position 0."""
    tokens, type = 2 ** 26 + 5, BF16
    m = make([3], [0], 1, 1, 8, 4, type, seed=5)
    q, k, v = (m[x][:1].cuda().expand(tokens, 1, 8) for x in ("q", "k", "v"))
    cache = [torch.zeros_like(p).cuda() for p in m["pools"]]
    starts = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    out = torch.full((tokens, 1, 8), 5.0, dtype=type, device="cuda")
    praghip.page_append(q, k, v, *cache, m["tables"].cuda(), m["lengths"].cuda(), starts, m["cos"].cuda(), m["sin"].cuda(), out=out)
    assert bool((out[:-2] == q[:-2]).all())  # (position 0 turns nothing)
    for at in (1, 2):
        want, size = turned(q[0].cpu(), None, m["cos"][at], m["sin"][at], False, 0)
        assert bool(((out[at - 3].cpu().double() - want).abs() <= UNIT[type] * want.abs() + SUMS * size).all())
    page = m["tables"][0, 0]
    assert bool((cache[1][page, 0, :3] == v[0, 0]).all()) and not bool(cache[1][page, 0, 3:].any())
