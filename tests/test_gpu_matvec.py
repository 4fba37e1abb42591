"""Few-row products with 4-bit weights on the GPU against their definition in 64 bits."""
import pytest
import torch

import praghip

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
UNIT = {BF16: 2.0 ** -8, F16: 2.0 ** -11}


def make(m, k, n, group, zeros, type, seed, width=None, positive=False):
    g = torch.Generator().manual_seed(seed)
    groups, width = -(-k // group), -(-k // 32) * 16 if width is None else width
    x = torch.randn((m, k), generator=g)
    x = (x.abs() if positive else x).to(type)
    w = torch.randint(0, 256, (n, width), generator=g, dtype=torch.uint8)
    s = (torch.rand((n, groups), generator=g) * 0.02 + 0.001).to(type)
    z = torch.randint(0, 16, (n, groups), generator=g, dtype=torch.uint8) if zeros else None
    return x, w, s, z


def plain(x, w, s, z, group):
    k = x.shape[1]
    digits = torch.stack((w & 15, w >> 4), -1).flatten(1)[:, :k].double()
    of = torch.arange(k) // group
    zero = z.double()[:, of] if z is not None else 8.0
    scale = s.double()[:, of] if k else digits
    want = x.double() @ ((digits - zero) * scale).T
    # the kernel sums x (16 + w) and (16 + z) x over a group in 32 bits
    size = x.double().abs() @ ((digits + 32 + 8) * scale).T
    return want, size


def check(y, want, size, type, group):
    # a group's sums are off by at most group 2^-24 of their terms' sizes, the sum over
    # the groups by far less; then one rounding
    bound = UNIT[type] * want.abs() + group * 2.0 ** -24 * size + 1e-30
    worst = ((y.double().cpu() - want).abs() / bound).max().item() if want.numel() else 0
    assert worst <= 1, worst


SIZES = [
    # m, k, n, group, zeros, type
    (1, 32, 16, 32, False, BF16), (1, 1024, 4096, 128, False, BF16), (1, 1, 1, 32, True, F16),
    (2, 33, 17, 32, True, BF16), (3, 100, 15, 64, False, F16), (16, 128, 64, 128, True, F16),
    (17, 1000, 100, 96, True, BF16), (5, 535, 521, 32, True, F16), (33, 257, 48, 256, False, BF16),
    (64, 2048, 33, 64, True, BF16), (70, 4097, 40, 1024, False, F16), (8, 130, 31, 160, True, BF16),
    (16, 256, 65600, 64, True, F16), (20, 96, 65700, 32, False, BF16), (4, 8192, 50, 128, True, F16),
    (1, 8192, 4099, 128, True, BF16), (7, 4096, 2050, 64, False, F16), (18, 2048, 2100, 32, True, BF16),
    # many columns: whole turns of eight groups, in LDS as a whole or in parts, and others
    (1, 1024, 16400, 128, False, BF16), (16, 512, 16385, 64, True, F16), (18, 768, 16390, 32, True, BF16),
    (40, 4096, 16384, 128, True, F16), (3, 8192, 16400, 128, False, BF16), (17, 3072, 65540, 64, False, F16),
    (2, 256, 70001, 32, True, BF16), (33, 1184, 16400, 32, True, F16), (2, 1600, 65600, 64, False, BF16),
]


@pytest.mark.parametrize("m,k,n,group,zeros,type", SIZES)
def test_against_64_bits(gpu, m, k, n, group, zeros, type):
    print("[w4]", m, k, n, group, zeros, type, flush=True)
    x, w, s, z = make(m, k, n, group, zeros, type, seed=m * 7 + k)
    y = praghip.matvec_w4(*(t.to("cuda") for t in (x, w, s)), None if z is None else z.to("cuda"), group=group)
    torch.cuda.synchronize()
    check(y, *plain(x, w, s, z, group), type, group)


@pytest.mark.parametrize("k,width", [(101, 51), (64, 33), (535, 268), (1024, 517), (30, 15)])
def test_rows_that_end_anywhere(gpu, k, width):
    """Rows without padding, at odd addresses: weights, scales, x and y."""
    print("[w4] width", k, width, flush=True)
    x, w, s, z = make(3, k, 37, 32, True, BF16, seed=k, width=width)
    wide = torch.zeros((3, k + 3), dtype=BF16, device="cuda")
    wide[:, 1:k + 1] = x.to("cuda")
    ws = torch.full((37, width + 5), 255, dtype=torch.uint8, device="cuda")
    ws[:, 2:width + 2] = w.to("cuda")
    out = torch.zeros((3, 50), dtype=BF16, device="cuda")
    y = praghip.matvec_w4(wide[:, 1:k + 1], ws[:, 2:width + 2], s.to("cuda"), z.to("cuda"), group=32, out=out[:, 5:42])
    torch.cuda.synchronize()
    check(y, *plain(x, w, s, z, 32), BF16, 32)
    assert not out[:, :5].any() and not out[:, 42:].any()


def test_rows_of_one_sign(gpu):
    """All of x positive: the offset's share of a sum is largest."""
    x, w, s, z = make(2, 4096, 64, 128, True, F16, seed=3, positive=True)
    y = praghip.matvec_w4(*(t.to("cuda") for t in (x, w, s, z)), group=128)
    check(y, *plain(x, w, s, z, 128), F16, 128)


def test_empty(gpu):
    x, w, s, z = make(3, 64, 20, 32, True, BF16, seed=4)
    w, s, z = w.to("cuda"), s.to("cuda"), z.to("cuda")
    assert praghip.matvec_w4(x[:0].to("cuda"), w, s, z, group=32).shape == (0, 20)
    assert praghip.matvec_w4(x.to("cuda"), w[:0], s[:0], z[:0], group=32).shape == (3, 0)
    y = praghip.matvec_w4(x[:, :0].to("cuda"), w, s[:, :0], None, group=32)
    assert y.shape == (3, 20) and not y.any()


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("k,group", [(256, 64), (100, 32), (40, 128)])
def test_quantized_weights(gpu, zeros, k, group):
    """A round trip: each weight is off by at most half a step, and a little for the
    scale's rounding; a group of zeros stays zero."""
    w = torch.randn((24, k), generator=torch.Generator().manual_seed(k)).to(BF16)
    w[3] = 0
    packed, scales, z = praghip.quantize_w4(w.to("cuda"), group, zeros=zeros)
    y = praghip.matvec_w4(torch.eye(k, dtype=BF16, device="cuda"), packed, scales, z, group=group).cpu().float().T
    step = scales.cpu().float()[:, torch.arange(k) // group]
    assert ((y - w.float()).abs() <= step * (0.5 + 15 * 2.0 ** -8) + 2.0 ** -8 * y.abs()).all()
    assert not y[3].any()


def test_same_bits_and_another_stream(gpu):
    x, w, s, z = (t.to("cuda") for t in make(4, 2048, 300, 64, True, F16, seed=6))
    y = praghip.matvec_w4(x, w, s, z, group=64)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = [praghip.matvec_w4(x, w, s, z, group=64, stream=side, out=torch.empty_like(y)) for _ in range(4)]
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, y)


def test_refusals(gpu):
    x, w, s, z = (t.to("cuda") for t in make(2, 64, 16, 32, True, BF16, seed=5))

    def refused(text, call):
        with pytest.raises(praghip.PraghipError) as e:
            call()
        assert text in e.value.text, e.value.text

    F = praghip.matvec_w4
    refused("E_W4_TYPE", lambda: F(x.float(), w, s, z, group=32))
    refused("E_W4_TYPE", lambda: F(x.half(), w, s, z, group=32))
    refused("E_W4_TYPE", lambda: F(x, w.to(torch.int8), s, z, group=32))
    refused("E_W4_SHAPE", lambda: F(x, w, s, z, group=24))
    refused("E_W4_SHAPE", lambda: F(x, w, s, z, group=64))
    refused("E_W4_SHAPE", lambda: F(x, w[:, :31], s, z, group=32))
    refused("E_W4_SHAPE", lambda: F(x, w, s, z[:, :1], group=32))
    refused("E_W4_SHAPE", lambda: F(x.t().contiguous().t(), w, s, z, group=32))
    refused("E_W4_DEVICE", lambda: F(x, w.cpu(), s, z, group=32))
    refused("E_W4_OUT", lambda: F(x, w, s, z, group=32, out=torch.zeros((2, 15), dtype=BF16, device="cuda")))
