"""A step's calls on another stream beside a busy current one, with memory that others have
written over, and as graphs that run at the same time."""
import pytest
import torch

import praghip
from test_gpu_serving_streams import busy_then_free
from test_gpu_shared import make

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def step():
    """name -> (the call's results, given keywords; what it changes)."""
    c = make([(300, [310, 420, 301]), (40, [44, 41])], 16, 8, 128, 16, BF16, seed=71, fill=0.0)
    q, k, v, tables, lengths, groups, shared = (c[x].cuda() for x in ("q", "k", "v", "tables", "lengths", "groups", "shared"))
    joint = torch.randn((5, 32, 128), generator=c["g"]).to(BF16).cuda()
    starts = torch.arange(6, dtype=torch.int32, device="cuda")
    cos, sin = praghip.rotary_table(tables.shape[1] * 16, 128)
    x, r, w = (torch.randn(n, generator=c["g"]).to(BF16).cuda() for n in ((7, 3000), (7, 3000), (3000,)))
    logits, u = torch.randn((9, 60000), generator=c["g"]).cuda() * 2, torch.rand(9, generator=c["g"]).cuda()

    def appended(**s):
        pools = [p.clone() for p in (k, v)]
        torch.cuda.synchronize()
        if s.pop("busy", False):
            busy_then_free()
        got = praghip.page_append(joint[:, :16], joint[:, 16:24], joint[:, 24:], *pools, tables, lengths, starts, cos, sin, **s)
        return (got, *pools)

    def then(call):
        def run(**s):
            if s.pop("busy", False):
                busy_then_free()
            return call(**s)
        return run

    return {
        "shared": then(lambda **s: praghip.paged_shared(q, k, v, tables, lengths, groups, shared, lse=True, **s)),
        "append": appended,
        "norm": then(lambda **s: praghip.add_norm(x, w, r, **s)),
        "sample": then(lambda **s: (praghip.sample_tokens(logits, u, top_p=0.9, top_k=5000, min_p=1e-3, **s),)),
    }


@pytest.mark.parametrize("name", ["shared", "append", "norm", "sample"])
def test_beside_a_busy_current_stream(gpu, name):
    print("[step streams]", name, flush=True)
    call = step()[name]
    want = call()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        got = call(stream=side, busy=True)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", ["shared", "norm", "sample"])
def test_graphs_at_the_same_time(gpu, name):
    """Two graphs of one call, each with a workspace of its own, replayed on two streams at once."""
    print("[step streams] graphs", name, flush=True)
    call = step()[name]
    want = call()
    torch.cuda.synchronize()
    graphs, results = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            results.append(call())
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for got in results:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            for t in got:
                t.zero_()
        torch.cuda.synchronize()
