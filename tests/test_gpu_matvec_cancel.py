"""4-bit products whose terms nearly cancel: weights at and beside their zero points, against
the bound that the two sums' roundings give."""
import pytest
import torch

import praghip

pytestmark = pytest.mark.gpu
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [70, 16390])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("off", [0, 1])
def test_weights_near_their_zero_points(gpu, type, n, group, off):
    print("[w4] near", type, n, group, off, flush=True)
    g = torch.Generator().manual_seed(group + off)
    m, k = 5, 8 * group
    x = (torch.rand((m, k), generator=g) + 0.5).to(type)  # all of one sign: the sums are largest
    z = torch.randint(0, 15, (n, 8), generator=g, dtype=torch.uint8)
    digits = z.repeat_interleave(group, 1)
    digits[:, ::7] += off
    w = digits[:, ::2] | (digits[:, 1::2] << 4)
    s = (torch.rand((n, 8), generator=g) + 0.5).to(type)
    y = praghip.matvec_w4(x.cuda(), w.cuda(), s.cuda(), z.cuda(), group=group).double().cpu()
    d, zz, ss = digits.double(), z.double().repeat_interleave(group, 1), s.double().repeat_interleave(group, 1)
    want = x.double() @ ((d - zz) * ss).T
    bound = UNIT[type] * want.abs() + group * 2.0 ** -24 * (x.double().abs() @ ((32 + d + zz) * ss).T)
    assert ((y - want).abs() <= bound).all(), ((y - want).abs() / bound).max().item()
