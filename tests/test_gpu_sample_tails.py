"""sample_tokens where whole parts of a row lie about 2^-44 below its largest weight, at the
ends of the random numbers' range: against weights in the units that the header names, 2^-43
of the power of two above the largest, rounded to whole numbers.

At 0 the token is the first with a unit, at 1 the last one, whatever the sums are; at 1 - 2^-24
it is one whose sums these tails are too small to change."""
import numpy as np
import pytest
import torch

import praghip

pytestmark = pytest.mark.gpu
ENDS = [0.0, 1 - 2.0 ** -24, 1.0]
PART = 8192  # tokens that the kernel's workgroups take at a time
FILTERS = [{}, {"top_k": "most"}, {"min_p": 1e-14}, {"top_k": "most", "min_p": 1e-14}, {"top_p": 1 - 2.0 ** -24, "top_k": "most"}]


def units(x, temperature):
    x = x.double().numpy()
    top, by = x.max(), 1.4426950408889634 / temperature
    anchor = np.ceil(top * by)
    return np.rint(np.exp2((x - top) * by + (top * by - anchor) + 43)).astype(object)


def plain(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    w = units(x, temperature)
    order = sorted(range(len(w)), key=lambda i: (-float(x[i]), i))
    if top_k:
        order = order[:top_k]
    if top_p < 1:
        sums = np.cumsum([w[i] for i in order])
        digits = int(top_p * 2 ** 24)  # (exact of a 32-bit number in [1/2, 1))
        order = order[: 1 + sum(1 for s in sums[:-1] if s * 2 ** 24 < digits * sums[-1])]
    if min_p:
        least = float(np.float32(min_p)) * float(w.max())
        order = [i for i in order if w[i] >= least]
    stay = sorted(i for i in order if w[i] > 0)
    sums = np.cumsum([w[i] for i in stay])
    at = min(int(u * 2 ** 24) * sums[-1] // 2 ** 24, sums[-1] - 1)
    return next(i for i, s in zip(stay, sums) if s > at)


def check(rows, **filters):
    rows = torch.stack(rows)
    vocab, n = rows.shape[1], len(rows)
    if filters.get("top_k") == "most":
        filters["top_k"] = vocab - 1
    want = [plain(row, u, **filters) for row in rows for u in ENDS]
    got = praghip.sample_tokens(rows.repeat_interleave(len(ENDS), 0).cuda(), torch.tensor(ENDS * n, device="cuda"), **filters)
    assert got.tolist() == want, [(i // 3, ENDS[i % 3], a, b) for i, (a, b) in enumerate(zip(got.tolist(), want)) if a != b]


@pytest.mark.parametrize("filters", FILTERS, ids=str)
@pytest.mark.parametrize("vocab,at", [(2 * PART, PART + 5), (2 * PART, PART - 2), (3 * PART + 77, PART + 5)])
def test_flat_tails(gpu, vocab, at, filters):
    """All logits but one are equal, in its part and in the others, 2^-42.3 to 2^-46.2 of it in
    weight: 1.7 to 0.06 units, none of them near a half."""
    print("[tails] flat", vocab, at, filters, flush=True)
    rows = []
    for top, tail in ((0, -29.3), (0, -29.9), (0, -30.2), (0, -30.4), (0, -30.8), (31, 0), (31.3, 0), (32, 0)):
        rows.append(torch.full((vocab,), float(tail)))
        rows[-1][at] = top
    check(rows, **filters)


@pytest.mark.parametrize("filters", FILTERS[:2], ids=str)
@pytest.mark.parametrize("temperature", [0.4, 1.0])
def test_random_tails(gpu, temperature, filters):
    """Tails of every distance around the last unit, whose parts hold some tokens with one,
    many or none; a few tokens far above them."""
    print("[tails] random", temperature, filters, flush=True)
    g = torch.Generator().manual_seed(int(10 * temperature))
    rows = []
    for i in range(24):
        x = -temperature * (29.5 + 0.125 * i + 3 * torch.rand(4 * PART - 100, generator=g))
        x[torch.randint(PART, 3 * PART, (3,), generator=g)] = torch.rand(3, generator=g)
        rows.append(x)
    check(rows, temperature=float(np.float32(temperature)), **filters)


def test_half_of_the_parts_count(gpu):
    """Parts in turn just above and just below the last unit."""
    x = torch.empty(6 * PART)
    for p in range(6):
        x[p * PART: (p + 1) * PART] = -30.9 if p % 2 == 0 else -30.2
    for at in (PART + 9, 2 * PART + 9, 4 * PART):
        row = x.clone()
        row[at] = 0
        for filters in FILTERS[:3]:
            check([row], **filters)
