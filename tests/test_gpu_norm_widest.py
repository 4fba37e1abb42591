"""add_norm of the widest rows that it takes: sums of 2^30 squares, which a 32-bit number does not
count one by one."""
import pytest
import torch

import praghip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type,unit", [(torch.float16, 2.0 ** -11), (torch.bfloat16, 2.0 ** -8)])
@pytest.mark.parametrize("n", [2 ** 26 + 3, 2 ** 28 + 7, 2 ** 30])
@pytest.mark.parametrize("add", [False, True])
def test_equal_values(gpu, n, type, unit, add):
    """The mean is the value's square, whatever the width."""
    print("[widest]", n, type, add, flush=True)
    value = torch.tensor(1.7, dtype=type)
    x = value.cuda().repeat(n)[None]
    w = torch.tensor(0.9, dtype=type).cuda().repeat(n)
    s = 2 * value.double() if add else value.double()
    got = praghip.add_norm(x, w, x if add else None, eps=0.5)
    if add:
        got, total = got
        assert bool((total == 2 * value.cuda()).all())
        del total
    want = float(w[0].double() * s / (s * s + 0.5).sqrt())
    # half a step of the type; the sum, the mean, the root, the quotient and two products in 32 bits
    worst = max(abs(float(got.min()) - want), abs(float(got.max()) - want)) / want
    assert worst <= unit + 16 * 2.0 ** -24, worst


def test_two_halves(gpu):
    """A row whose first half is small beside the second, against 64 bits."""
    n = 2 ** 27 + 8
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty((2, n), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    x[0, : n // 2] *= 2.0 ** -6
    w = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    got = praghip.add_norm(x, w)
    for i in range(2):
        mean = sum(float(part.double().square().sum()) for part in x[i].split(1 << 24)) / n
        want = x[i, ::999].double() / (mean + 1e-6) ** 0.5
        assert bool(((got[i, ::999].double() - want).abs() <= (2.0 ** -8 + 16 * 2.0 ** -24) * want.abs()).all())
