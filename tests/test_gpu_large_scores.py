"""Scores so large that a step of their 32 bits is a whole power of two of a probability and
more: the strongest key, or the equal ones that share it, have all of the output.

Each score is one product of two 16-bit numbers (exact in 32 bits), and the next smaller one
is 2^-7 of it lower, far more than the exponent's range."""
import pytest
import torch

import attention_plain as plain
import praghip

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def make(type, size, dim, sign):
    """Three sequences over one prefix of 150 keys; an even head's product with the strongest keys is 2^size 1.28."""
    lengths, prefix, page = [190, 150, 163], 150, 16
    c = plain.make(lengths, 4, 2, dim, page, type, seed=size + dim)
    high = size // 2
    for s, n in enumerate(lengths):
        at = torch.arange(n)
        entry, row = c["tables"][s].long()[at // page], at % page
        k = torch.zeros((n, 2, dim))
        # (the strongest are keys 3, 70 and 149 of the prefix, for head 1 also one of each's own)
        k[:, :, 5] = sign * 2.0 ** high * (1 - 2.0 ** -7 * (1 + at % 40))[:, None]
        k[[3, 70, 149], :, 5] = sign * 2.0 ** high
        k[prefix + 9:, 1, 5] = sign * 2.0 ** high * (1 + 2.0 ** -6)
        c["k"][entry, :, row] = k.to(type)
        if s:
            c["v"][entry[:prefix], :, row[:prefix]] = c["v"][c["tables"][0].long()[at[:prefix] // page], :, at[:prefix] % page]
    q = torch.zeros((3, 4, dim))
    q[:, ::2, 5] = 2.0 ** (size - high) * 1.28125
    q[:, 1::2, 5] = 2.0 ** -high * 1.28125  # beside them in a wave, scores of about 1
    c["q"] = q.to(type)
    c["groups"] = torch.tensor([0, 3], dtype=torch.int32)
    c["shared"] = torch.tensor([prefix], dtype=torch.int32)
    return c


# With a scale of 0.7 these are some 1.3 x 2^size in powers of two; in float16 a product
# of two is below 2^32.
SIZES = [(t, n) for t in (F16, BF16) for n in (12, 19, 20, 22, 23, 24, 25, 26, 27, 28, 30)] + [(BF16, n) for n in (31, 32, 33, 34, 36, 40, 60, 90)]


def attention(c, q, starts, scale):
    """As attention_plain.py's, whose probabilities are taken relative to the logarithm of their sum: of scores
    from 2^53 on 64 bits do not hold that beside the maximum."""
    out, sums = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:2], -float("inf"), dtype=torch.float64)
    for s in range(len(starts) - 1):
        _, k, v = plain.rows_of(c, s)
        for row in range(starts[s], starts[s + 1]):
            n = len(k) - (starts[s + 1] - 1 - row)
            for h in range(q.shape[1]):
                g = h * c["kv"] // q.shape[1]
                score = scale * (k[:n, g] @ q[row, h].double())
                lse[row, h] = torch.logsumexp(score, 0)
                p = torch.softmax(score, 0)
                out[row, h], sums[row, h] = p @ v[:n, g], p @ v[:n, g].abs()
    return out, lse, sums


def compare(out, lse, want, want_lse, sums, type, rounded):
    plain.check(out, want, sums, type, rounded)
    # (two roundings of the score and one of the scale, 2^-24 of it each)
    assert ((lse.double().cpu() - want_lse).abs() <= 2.0 ** -22 * want_lse.abs() + plain.SUMS).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("type,size", SIZES)
@pytest.mark.parametrize("scale", [0.7, -0.7])
def test_shared_prefixes(gpu, type, size, dim, scale):
    print("[large] shared", type, size, dim, scale, flush=True)
    c = make(type, size, dim, 1 if scale > 0 else -1)
    on = [c[x].cuda() for x in ("q", "k", "v", "tables", "lengths", "groups", "shared")]
    want = attention(c, c["q"], [0, 1, 2, 3], scale)
    out, lse = praghip.paged_shared(*on, scale=scale, lse=True)
    compare(out, lse, *want, type, False)


def test_a_score_that_overflows_in_a_shared_prefix(gpu):
    """Of a maximum that is no number in 32 bits the output is none either."""
    c = make(BF16, 130, 64, 1)
    out = praghip.paged_shared(*(c[x].cuda() for x in ("q", "k", "v", "tables", "lengths", "groups", "shared")))
    assert not bool(out[:, ::2].isfinite().any()) and bool(out[:, 1::2].isfinite().all())


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("type,size", SIZES)
@pytest.mark.parametrize("scale", [0.7, -0.7])
def test_single_tokens(gpu, type, size, dim, scale):
    print("[large] single", type, size, dim, scale, flush=True)
    c = make(type, size, dim, 1 if scale > 0 else -1)
    want = attention(c, c["q"], [0, 1, 2, 3], scale)
    out, lse = praghip.paged_decode(*(c[x].cuda() for x in ("q", "k", "v", "tables", "lengths")), scale=scale, lse=True)
    compare(out, lse, *want, type, False)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("type,size", SIZES)
@pytest.mark.parametrize("scale", [0.7, -0.7])
def test_prompts(gpu, type, size, dim, scale):
    print("[large] prompt", type, size, dim, scale, flush=True)
    c = make(type, size, dim, 1 if scale > 0 else -1)
    q = c["q"].repeat_interleave(20, 0)
    starts = [0, 20, 40, 60]
    want = attention(c, q, starts, scale)
    first = torch.tensor(starts, dtype=torch.int32, device="cuda")
    out, lse = praghip.paged_prompt(q.cuda(), *(c[x].cuda() for x in ("k", "v", "tables", "lengths")), first, 20, scale=scale, lse=True)
    compare(out, lse, *want, type, True)


def test_a_prompt_with_an_infinity_among_large_scores(gpu):
    """What is formed again from the cache (O that is not finite) takes the same exponents."""
    c = make(BF16, 34, 64, 1)
    q = c["q"].repeat_interleave(20, 0)
    c["v"][int(c["tables"][0, 160 // 16]), 1, 0, 5] = float("inf")  # position 160 of the first sequence, as long as 190
    starts = [0, 20, 40, 60]
    out, _ = praghip.paged_prompt(q.cuda(), *(c[x].cuda() for x in ("k", "v", "tables", "lengths")),
                                  torch.tensor(starts, dtype=torch.int32, device="cuda"), 20, scale=0.7, lse=True)
    # all of its queries see that key, which the second key/value head's even queries take a share of
    c["v"][int(c["tables"][0, 160 // 16]), 1, 0, 5] = 0
    want, _, sums = attention(c, q, starts, 0.7)
    held = torch.ones_like(want, dtype=torch.bool)
    held[:20, 2:, 5] = False
    assert not bool(out[:20, 2, 5].isfinite().any())
    plain.check(torch.where(held, out.cpu().double(), want), want, sums, BF16, True)
