"""Serving calls on another stream beside a busy current one, with no wait between them: the
current stream's memory, freed with work on it still to run, is not theirs."""
import pytest
import torch

import attention_plain as plain
import praghip

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def busy_then_free():
    """Some milliseconds of work on the current stream that end in writes of memory which is
    free again by the time this returns: blocks of all sizes that a workspace may have."""
    a = torch.ones((4096, 4096), device="cuda")
    for _ in range(4):
        a = a @ a
        a /= 4096
    for size in [1 << n for n in range(9, 27)]:
        for _ in range(2):
            torch.empty(size, dtype=torch.uint8, device="cuda").fill_(255)


def serving():
    """The calls that make a workspace or a result, and what they change."""
    c = plain.make([3000, 70], 16, 8, 128, 16, BF16, seed=41)
    k, v, tables, lengths = (c[x].to("cuda") for x in ("k", "v", "tables", "lengths"))
    q = torch.randn((20, 16, 128), generator=c["g"]).to(BF16).to("cuda")
    starts = torch.tensor([0, 12, 20], dtype=torch.int32, device="cuda")
    x = torch.randn((5, 1024), generator=c["g"]).to(BF16).to("cuda")
    w = praghip.quantize_w4(torch.randn((512, 1024), generator=c["g"]).to(BF16).to("cuda"), zeros=True)
    return {
        "decode": lambda **s: praghip.paged_decode(q[:2], k, v, tables, lengths, lse=True, **s),
        "prompt": lambda **s: praghip.paged_prompt(q, k, v, tables, lengths, starts, 12, lse=True, **s),
        "w4": lambda **s: (praghip.matvec_w4(x, *w, **s),),
    }


@pytest.mark.parametrize("name", ["decode", "prompt", "w4"])
def test_beside_a_busy_current_stream(gpu, name):
    print("[streams]", name, flush=True)
    call = serving()[name]
    want = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        busy_then_free()
        got = call(stream=side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", ["decode", "prompt", "w4"])
def test_results_let_go_while_they_are_read(gpu, name):
    """The current stream reads a result late; the next call on the side stream, made when the
    result is gone, does not write over it."""
    print("[streams] let go", name, flush=True)
    call = serving()[name]
    want = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        poison = [torch.empty_like(t) for t in want]
    torch.cuda.synchronize()
    del poison
    got = call(stream=side)
    torch.cuda.current_stream().wait_stream(side)
    busy_then_free()
    kept = [t.clone() for t in got]
    del got
    with torch.cuda.stream(side):  # in the blocks of the result, if those are free
        for t in want:
            for _ in range(4):
                torch.empty_like(t).fill_(-1)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_pages_beside_a_busy_current_stream(gpu):
    """A fork and a compaction: their lists of moves are their own."""
    print("[streams] pages", flush=True)

    def lists(*v):
        return [torch.tensor(x, dtype=torch.int32, device="cuda") for x in v]

    results = []
    for other in (False, True):
        g = torch.Generator(device="cuda").manual_seed(42)
        pool = torch.randn((4, 2, 200, 2, 16, 64), generator=g, device="cuda").to(BF16)
        tables = torch.full((12, 20), -1, dtype=torch.int32, device="cuda")
        lengths, refs = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (12, 200))
        status, = lists([0])
        rows, counts, parents, children, ended = lists([0, 1, 2], [250, 77, 90], [0, 0, 1, 2], [3, 4, 5, 6], [0, 2, 3])
        praghip.page_reserve(tables, lengths, refs, 16, rows, counts, status)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        on = dict(stream=side) if other else {}
        if other:
            busy_then_free()
        praghip.page_fork(pool, tables, lengths, refs, parents, children, status, **on)
        praghip.page_free(tables, lengths, refs, ended, status, **on)
        praghip.page_compact(pool, tables, refs, **on)
        torch.cuda.synchronize()
        assert int(status) == 0
        results.append((pool, tables, lengths, refs))
    assert all(torch.equal(a, b) for a, b in zip(*results))
