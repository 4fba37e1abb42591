"""One strong key above many weak ones, by 16 to 18 in the exponent: each of the weak ones'
probabilities is near or below float16's smallest value, and together they are a part of
the output that counts, or all of it where the strong key's value is 0."""
import pytest
import torch

import attention_plain as plain
import praghip

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
DIM, PAGE = 64, 16


def make(n, strong, type, rows):
    """A sequence of n tokens; scores of the three heads are 24 / 8, 25.5 / 8.5 and 27 / 9."""
    c = plain.make([n], 3, 1, DIM, PAGE, type, seed=n + strong, width=-(-n // PAGE))
    at = torch.arange(n)
    page, place = c["tables"][0].long()[at // PAGE], at % PAGE
    c["k"][page, :, place] = 0
    c["k"][page, :, place, 0] = 2
    c["v"][page, :, place] = (torch.rand((n, 1, DIM), generator=c["g"]) + 0.5).to(type)
    c["k"][page[strong], :, place[strong], 0] = 6
    c["v"][page[strong], :, place[strong]] = torch.arange(DIM).ge(DIM // 2).to(type)
    q = torch.zeros((rows, 3, DIM))
    q[:, :, 0] = torch.tensor([4, 4.25, 4.5])
    return c, q.to(type), [c[x].to("cuda") for x in ("k", "v", "tables", "lengths")]


def place_of(strong, n):
    return {"first": 0, "middle": n // 2, "last": n - 8}[strong]


@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("strong", ["first", "middle", "last"])
@pytest.mark.parametrize("n", [32, 1000, 131072])
def test_decode(gpu, n, strong, type):
    print("[small] decode", n, strong, type, flush=True)
    c, q, on = make(n, place_of(strong, n), type, 1)
    out, lse = praghip.paged_decode(q.to("cuda"), *on, scale=1.0, lse=True)
    want, wlse, size = plain.attention(c, q, [0, 1], scale=1.0)
    plain.check(out, want, size, type, rounded=False)
    plain.check_lse(lse, wlse)


@pytest.mark.parametrize("type", [F16, BF16])
@pytest.mark.parametrize("strong", ["first", "middle", "last"])
@pytest.mark.parametrize("n", [32, 1000, 131072])
def test_prompt(gpu, n, strong, type):
    print("[small] prompt", n, strong, type, flush=True)
    c, q, on = make(n, place_of(strong, n), type, 4)
    starts = [0, 4]
    out, lse = praghip.paged_prompt(q.to("cuda"), *on, torch.tensor(starts, dtype=torch.int32, device="cuda"), 4, scale=1.0, lse=True)
    want, wlse, size = plain.attention(c, q, starts, scale=1.0)
    plain.check(out, want, size, type, rounded=True)
    plain.check_lse(lse, wlse)


@pytest.mark.parametrize("heads", [1, 130, 3200])
def test_all_of_a_heads_keys_in_one_wave(gpu, heads):
    """So many heads (which name the same keys) that none is split: one wave, or one workgroup
    of the prompt's, meets the strong key and the 20000 weak ones."""
    print("[small] heads", heads, flush=True)
    n = 20000
    for strong in (0, n // 2):
        c, q, (k, v, tables, lengths) = make(n, strong, F16, 2)
        want, wlse, size = plain.attention(c, q, [0, 2], scale=1.0)
        k, v = (x.expand(-1, heads, -1, -1) for x in (k, v))
        q = q.repeat(1, heads, 1).to("cuda")
        out, lse = praghip.paged_decode(q[1:], k, v, tables, lengths, scale=1.0, lse=True)
        both, sums = praghip.paged_prompt(q, k, v, tables, lengths, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), 2,
                                          scale=1.0, lse=True)
        for h in {0, heads // 2, heads - 1}:
            at = slice(3 * h, 3 * h + 3)
            plain.check(out[:, at], want[1:], size[1:], F16, rounded=False)
            plain.check_lse(lse[:, at], wlse[1:])
            plain.check(both[:, at], want, size, F16, rounded=True)
            plain.check_lse(sums[:, at], wlse)


@pytest.mark.parametrize("scale", [-0.1, 0.0, 0.125, 30.0])
def test_scales(gpu, scale):
    """float16 at scales of any size: what P's range is chosen by."""
    print("[small] scale", scale, flush=True)
    c = plain.make([150, 41], 8, 4, 64, 16, F16, seed=43)
    q = (torch.randn((60, 8, 64), generator=c["g"]) * (0.01 if scale == 30.0 else 1)).to(F16)
    on = [c[x].to("cuda") for x in ("k", "v", "tables", "lengths")]
    starts = [0, 40, 60]
    want, wlse, size = plain.attention(c, q, starts, scale=scale, window=50, sinks=3)
    out, lse = praghip.paged_prompt(q.to("cuda"), *on, torch.tensor(starts, dtype=torch.int32, device="cuda"), 40,
                                    scale=scale, window=50, sinks=3, lse=True)
    plain.check(out, want, size, F16, rounded=True)
    plain.check_lse(lse, wlse)
    want, wlse, size = plain.attention(c, q[:2], [0, 1, 2], scale=scale, window=50, sinks=3)
    out, lse = praghip.paged_decode(q[:2].to("cuda"), *on, scale=scale, window=50, sinks=3, lse=True)
    plain.check(out, want, size, F16, rounded=False)
    plain.check_lse(lse, wlse)
