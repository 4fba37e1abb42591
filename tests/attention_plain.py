"""Paged attention in 64 bits on the CPU, written from its definition, and the
tensors of a test."""
import math

import torch


def make(lengths, heads, kv, dim, page, type, seed, spare=3, width=None, layout="phtd", fill=None):
    """A cache with these lengths: pages at random places, keys and values on the CPU.

    fill: what every row that no position names holds (NaN by default).  layout
    "phtd" is [pages][kv][page][dim] in memory, "pthd" [pages][page][kv][dim].
    """
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    width = max(need + [1]) if width is None else width
    count = sum(need) + spare
    order = torch.randperm(count, generator=g).to(torch.int32)
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    shape = (count, kv, page, dim)
    pools = [torch.full(shape, math.nan if fill is None else fill, dtype=type) for _ in range(2)]
    for s, n in enumerate(lengths):
        tables[s, : need[s]] = order[at: at + need[s]]
        at += need[s]
        for i in range(need[s]):
            rows = min(page, n - i * page)
            for x in pools:
                x[tables[s, i], :, :rows] = torch.randn((kv, rows, dim), generator=g).to(type)
    if layout == "pthd":
        pools = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in pools]
    return {"k": pools[0], "v": pools[1], "tables": tables, "lengths": torch.tensor(lengths, dtype=torch.int32),
            "g": g, "heads": heads, "kv": kv, "dim": dim, "page": page}


def rows_of(c, s):
    """Positions of sequence s that have a page, and their keys and values in 64 bits."""
    n = int(c["lengths"][s])
    n = max(0, min(n, c["tables"].shape[1] * c["page"]))
    at = torch.arange(n)
    entry = c["tables"][s].long()[at // c["page"]]
    here = (entry >= 0) & (entry < c["k"].shape[0])
    at, entry = at[here], entry[here]
    return at, c["k"][entry, :, at % c["page"]].double(), c["v"][entry, :, at % c["page"]].double()


def attention(c, q, starts, scale=None, window=0, sinks=0):
    """out, lse and the sums of p |v| (for tolerances) of rows starts[s] .. of q, in 64 bits."""
    heads, dim = q.shape[1:]
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    size = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    for s in range(len(starts) - 1):
        at, k, v = rows_of(c, s)
        n = int(c["lengths"][s])
        n = max(0, min(n, c["tables"].shape[1] * c["page"]))
        for row in range(starts[s], starts[s + 1]):
            place = n - (starts[s + 1] - row)
            see = at <= place
            if window:
                see &= (at > place - window) | (at < sinks)
            if not bool(see.any()):
                continue
            for h in range(heads):
                g = h * c["kv"] // heads
                score = scale * (k[see, g] @ q[row, h].double())
                lse[row, h] = torch.logsumexp(score, 0)
                p = torch.exp(score - lse[row, h])
                out[row, h] = p @ v[see, g]
                size[row, h] = p @ v[see, g].abs()
    return out, lse, size


# Rounding of an output to its type, and what the sums leave.  Scores are 32-bit sums
# of dim products, off by less than dim 2^-24 sum |q k| scale, below 2^-13 for the
# tests' values; the probabilities are off by that relatively, and each output by that
# times sum p |v|.  Where P goes into the product rounded to the type, each
# probability is off by the type's unit more.
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SUMS = 2.0 ** -12


def check(got, want, size, type, rounded):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    bound = UNIT[type] * want.abs() + (SUMS + (UNIT[type] if rounded else 0)) * size + 1e-7
    worst = ((got - want).abs() / bound).max().item() if got.numel() else 0.0
    assert worst <= 1, f"{worst} of the bound"


def check_lse(got, want):
    got = got.double().cpu()
    empty = want == -math.inf
    assert torch.equal(got == -math.inf, empty)
    assert ((got - want)[~empty].abs() <= SUMS + 1e-6 * want[~empty].abs()).all()
