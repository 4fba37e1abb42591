"""Infinite keys that a query sees: a score of minus infinity is weight 0, and leaves the output
to the other keys; any other score that is not finite makes it NaN."""
import math

import pytest
import torch

import attention_plain as plain
import praghip

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 5)])
def test_infinite_keys_that_are_seen(gpu, type, dim, window, sinks):
    print("[infinite keys]", type, dim, window, sinks, flush=True)
    n, rows = 300, 60
    c = plain.make([n], 4, 2, dim, 16, type, seed=dim + window + 2)
    q = torch.randn((rows, 4, dim), generator=c["g"])
    q[:, :, 7] = q[:, :, 7].abs() + 0.1
    q = q.to(type)
    for at in (2, 255, 280):  # a sink, one that all see, one that the later rows see
        c["k"][c["tables"][0, at // 16], 1, at % 16, 7] = -math.inf
    want, wlse, size = plain.attention(c, q, [0, rows], window=window, sinks=sinks)
    assert torch.isfinite(want).all()
    on = [c[x].to("cuda") for x in ("k", "v", "tables", "lengths")]
    starts = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    out, lse = praghip.paged_prompt(q.to("cuda"), *on, starts, rows, window=window, sinks=sinks, lse=True)
    plain.check(out, want, size, type, rounded=True)
    plain.check_lse(lse, wlse)
    out, lse = praghip.paged_decode(q[-1:].to("cuda"), *on, window=window, sinks=sinks, lse=True)
    plain.check(out, want[-1:], size[-1:], type, rounded=False)
    plain.check_lse(lse, wlse[-1:])
    # the same key as plus infinity
    on[0][c["tables"][0, 255 // 16].long(), 1, 255 % 16, 7] = math.inf
    for out in (praghip.paged_prompt(q.to("cuda"), *on, starts, rows, window=window, sinks=sinks)[-rows // 2:],
                praghip.paged_decode(q[-1:].to("cuda"), *on, window=window, sinks=sinks)):
        assert out[:, 2:].isnan().all() and torch.isfinite(out[:, :2]).all()


@pytest.mark.parametrize("type", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [5, 100])
def test_no_other_key_is_seen(gpu, type, n):
    """All scores are minus infinity: zeros and minus infinity, as where nothing is seen."""
    print("[infinite keys] all", type, n, flush=True)
    c = plain.make([n], 4, 2, 64, 16, type, seed=n)
    q = torch.randn((n, 4, 64), generator=c["g"]).abs().add(0.1).to(type).to("cuda")
    k, v, tables, lengths = (c[x].to("cuda") for x in ("k", "v", "tables", "lengths"))
    k[:, :, :, 7] = -math.inf
    starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    for out, lse in (praghip.paged_prompt(q, k, v, tables, lengths, starts, n, lse=True),
                     praghip.paged_decode(q[-1:], k, v, tables, lengths, lse=True)):
        assert not out.any() and bool((lse == -math.inf).all())
