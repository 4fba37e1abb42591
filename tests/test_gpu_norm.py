"""add_norm against 64 bits: types, widths around each of its kernels' limits, strides, memory
that is read and written, values at the types' ends."""
import pytest
import torch

import praghip

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]
# half a step of the type; the mean's terms are all positive, so its sum of depth d is off by d
# 2^-24 relatively (d at most 8 x 4 + 6 + 16 up to n = 32768, and 60 more at 65000), which the
# root halves, and a handful of products follow
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SUMS = 2.0 ** -17


def plain(x, weight, residual, eps):
    s = x.cpu().double() if residual is None else x.cpu().double() + residual.cpu().double()
    return s, s / (s.square().mean(-1, keepdim=True) + eps).sqrt() * weight.cpu().double()


def close(got, want, type, more=0.0):
    got = got.cpu().double()
    # (below the smallest normal value a step is the smallest subnormal one)
    least = 2.0 ** -25 if type is torch.float16 else 2.0 ** -134
    bound = (UNIT[type] + more) * want.abs() + least
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


def make(rows, n, type, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x, r = (torch.randn((rows, n), generator=g) * scale for _ in range(2))
    w = 1 + 0.3 * torch.randn(n, generator=g)
    return x.to(type).cuda(), w.to(type).cuda(), (3 * r).to(type).cuda()


def check(x, w, r, eps=1e-6, **kw):
    s, y = plain(x, w, r, eps)  # before the call, which may write to its inputs
    got = praghip.add_norm(x, w, r, eps=eps, **kw)
    if r is None:
        close(got, y, x.dtype, SUMS)
    else:
        close(got[0], y, x.dtype, SUMS)
        close(got[1], s, x.dtype, 2.0 ** -23)
    return got


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 63, 511, 512, 513, 1024, 1031, 2047, 2048, 2049, 4096, 4099, 8192, 8200, 16384, 16391,
                               32768, 32769, 65000])
def test_widths(gpu, type, n):
    print("[norm]", type, n, flush=True)
    for rows in (1, 5):
        x, w, r = make(rows, n, type, seed=n)
        check(x, w, r)
        check(x, w, None)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("rows", [1, 3, 64, 257, 5000])
def test_rows(gpu, type, rows):
    print("[norm] rows", type, rows, flush=True)
    x, w, r = make(rows, 640, type, seed=rows)
    check(x, w, r, eps=1e-5)


@pytest.mark.parametrize("n", [40, 1027, 3000, 9001, 33000])
def test_strides_and_what_lies_between(gpu, n):
    """Rows apart, at odd addresses; what lies between them stays."""
    print("[norm] strides", n, flush=True)
    x, w, r = make(6, 2 * n + 3, torch.bfloat16, seed=n)
    wide = [torch.full((6, n + 5), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    out, total = (t[:, 3: 3 + n] for t in wide)
    got = check(x[::2, 1: 1 + n], w[1: 1 + n], r[1:4, n: 2 * n], out=out[:3], total=total[3:])
    assert got[0].data_ptr() == out.data_ptr()
    for t, used in ((wide[0], range(3)), (wide[1], range(3, 6))):
        rest = t.clone()
        rest[list(used), 3: 3 + n] = 7.0
        assert bool((rest == 7.0).all())


@pytest.mark.parametrize("n", [5, 1024, 1029, 4001, 20000, 40000])
@pytest.mark.parametrize("where", ["total is residual", "out is x", "out is residual, total is x"])
def test_memory_that_is_read(gpu, n, where):
    print("[norm]", where, n, flush=True)
    x, w, r = make(9, n, torch.float16, seed=n)
    check(x, w, r, **({"total": r} if where == "total is residual" else {"out": x} if where == "out is x" else {"out": r, "total": x}))


def test_values_at_the_ends(gpu):
    """Zeros (eps alone), subnormal and large values, and rows that are not finite, which leave
    the others as they are."""
    x, w, r = make(8, 1000, torch.bfloat16, seed=3)
    x[0] = 0
    r[0] = 0
    x[1] *= 1e-30
    r[1] *= 1e-30
    x[2] *= 1e15
    check(x, w, r)
    h = (x[3:6] * 1000).half()
    h[0] *= 2.0 ** -24 / 1000
    check(h, w.half(), None, eps=0.0 + 1e-12)
    want = praghip.add_norm(x, w, r)
    x[5, 17], r[6, 0] = float("inf"), float("nan")
    got = praghip.add_norm(x, w, r)
    for a, b in zip(got, want):
        assert torch.equal(a[[0, 1, 2, 3, 4, 7]], b[[0, 1, 2, 3, 4, 7]])
    assert bool(got[0][6].isnan().all()) and not bool(got[0][5].isfinite().all())


def test_the_same_bits(gpu):
    """A captured call replayed with other inputs, and the same call again."""
    x, w, r = make(33, 5000, torch.bfloat16, seed=4)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side):
        praghip.add_norm(x, w, r)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = praghip.add_norm(x, w, r)
    for seed in range(5, 9):
        x2, _, r2 = make(33, 5000, torch.bfloat16, seed)
        x.copy_(x2), r.copy_(r2)
        graph.replay()
        torch.cuda.synchronize()
        want = praghip.add_norm(x, w, r)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(gpu):
    x, w, r = make(4, 64, torch.bfloat16, seed=5)
    F = praghip.add_norm

    def refused(text, *args, **kw):
        with pytest.raises(praghip.PraghipError) as e:
            F(*args, **kw)
        assert e.value.text == text

    for bad in ((x[0], w, r[0]), (x, w[:63], r), (x, w[None], r), (x, w, r[:3]), (x, w, r[0]), (x.t(), w[:4], r.t()), (x, w[::2], r),
                (x[:, ::2], w[:32], None)):
        refused("E_NORM_SHAPE", *bad)
    for bad in ((x.float(), w.float(), None), (x, w.half(), r), (x, w, r.half()), (x.long(), w, r)):
        refused("E_NORM_TYPE", *bad)
    for bad in ((x, w.cpu(), r), (x, w, r.cpu()), (x.cpu(), w.cpu(), r.cpu())):
        refused("E_NORM_DEVICE", *bad)
    for kw in (dict(out=x[:3]), dict(out=x.half()), dict(total=r.cpu()), dict(total=r.t()), dict(out=torch.empty_like(x).t().contiguous().t())):
        refused("E_NORM_OUT", x, w, r, **kw)
    refused("E_NORM_OUT", x, w, None, total=r)
    for eps in (-1.0, float("nan"), float("inf")):
        refused("E_NORM_SHAPE", x, w, r, eps=eps)
    for some in ((x.clone().requires_grad_(), w, r), (x, w.clone().requires_grad_(), r), (x, w, r.clone().requires_grad_())):
        refused("E_NORM_GRADIENT", *some)
        with torch.no_grad():
            assert not F(*some)[0].requires_grad
    assert F(x[:0], w, r[:0])[0].shape == (0, 64) and F(x[:, :0], w[:0]).shape == (4, 0)


@pytest.mark.parametrize("rows,n", [(2 ** 22 + 3, 1), (2 ** 26 + 5, 8)])
def test_more_workgroups_than_a_grid_row_has_threads_for(gpu, rows, n):
    """2^22 workgroups of 1024 threads, and 2^24 of 256."""
    print("[norm]", rows, n, flush=True)
    x, w, _ = make(1024, n, torch.bfloat16, seed=n)
    want = praghip.add_norm(x, w)
    check(x, w, None)
    index = torch.arange(rows, device="cuda") % 1000
    got = praghip.add_norm(x[index], w)
    assert torch.equal(got, want[index])
