"""The cache's pages on the GPU against a model of them in Python: every call compared
exactly (tables, lengths, references, contents), and every refusal leaves all as it was."""
import pytest
import torch

import praghip

pytestmark = pytest.mark.gpu


class Model:
    """Tables, lengths, references and pages on the CPU."""

    def __init__(self, layers, pages, kv, page, dim, seqs, width, seed, type=torch.bfloat16):
        g = torch.Generator().manual_seed(seed)
        self.page, self.width = page, width
        self.pool = torch.randn((layers, 2, pages, kv, page, dim), generator=g).to(type)
        self.tables = torch.full((seqs, width), -1, dtype=torch.int32)
        self.lengths = torch.zeros(seqs, dtype=torch.int32)
        self.refs = torch.zeros(pages, dtype=torch.int32)

    def free_pages(self):
        return [p for p in range(len(self.refs)) if self.refs[p] <= 0]

    def reserve(self, seqs, counts):
        if len(set(seqs)) < len(seqs) or any(not 0 <= s < len(self.lengths) for s in seqs):
            return 1
        if any(c < 0 or self.lengths[s] + c > self.width * self.page for s, c in zip(seqs, counts)):
            return 2
        need = [(s, at) for s, c in zip(seqs, counts)
                for at in range(-(-int(self.lengths[s]) // self.page), -(-int(self.lengths[s] + c) // self.page))]
        free = self.free_pages()
        if len(free) < len(need):
            return 3
        for (s, at), p in zip(need, free):
            self.tables[s, at] = p
            self.refs[p] = 1
        for s, c in zip(seqs, counts):
            self.lengths[s] += c
        return 0

    def drop(self, s, at):
        if self.tables[s, at] >= 0:
            self.refs[self.tables[s, at]] -= 1
            self.tables[s, at] = -1

    def free(self, seqs):
        if len(set(seqs)) < len(seqs) or any(not 0 <= s < len(self.lengths) for s in seqs):
            return 1
        for s in seqs:
            for at in range(self.width):
                self.drop(s, at)
            self.lengths[s] = 0
        return 0

    def trim(self, seqs, window, sinks):
        for s in seqs:
            for at in range(self.width):
                seen = [j for j in range(at * self.page, (at + 1) * self.page)
                        if j < sinks or j > int(self.lengths[s]) - window]
                if not seen:
                    self.drop(s, at)
        return 0

    def fork(self, parents, children):
        if len(set(children)) < len(children) or set(parents) & set(children) or \
                any(not 0 <= s < len(self.lengths) for s in parents + children) or \
                any(self.lengths[s] for s in children):
            return 1
        last = {i: int(self.lengths[p]) // self.page for i, p in enumerate(parents) if int(self.lengths[p]) % self.page}
        apart = [i for i in last if self.tables[parents[i], last[i]] >= 0]
        free = self.free_pages()
        if len(free) < len(apart):
            return 3
        new = dict(zip(apart, free))
        for i, (p, c) in enumerate(zip(parents, children)):
            count = -(-int(self.lengths[p]) // self.page)
            row = torch.full_like(self.tables[c], -1)
            row[:count] = self.tables[p, :count]
            if i in new:
                self.pool[:, :, new[i]] = self.pool[:, :, row[last[i]]]
                row[last[i]] = new[i]
            self.tables[c] = row
            self.lengths[c] = self.lengths[p]
        for i, c in enumerate(children):
            for p in self.tables[c].tolist():
                if p >= 0:
                    self.refs[p] += 1
        return 0

    def compact(self):
        live = int((self.refs > 0).sum())
        holes = [p for p in range(live) if self.refs[p] <= 0]
        moved = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        for src, dst in zip(moved, holes):
            self.pool[:, :, dst] = self.pool[:, :, src]
            self.refs[dst], self.refs[src] = int(self.refs[src]), 0
            self.tables[self.tables == src] = dst
        return 0

    def write(self, layer, k, v, starts):
        for s in range(len(starts) - 1):
            for t in range(starts[s], starts[s + 1]):
                at = int(self.lengths[s]) - starts[s + 1] + t
                if at < 0 or at >= self.width * self.page or self.tables[s, at // self.page] < 0:
                    continue
                self.pool[layer, 0, self.tables[s, at // self.page], :, at % self.page] = k[t]
                self.pool[layer, 1, self.tables[s, at // self.page], :, at % self.page] = v[t]


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Pair:
    """A model and the same on the GPU; every call goes to both."""

    def __init__(self, *a, **kw):
        self.m = Model(*a, **kw)
        self.pool, self.tables, self.lengths, self.refs = (
            x.to("cuda") for x in (self.m.pool, self.m.tables, self.m.lengths, self.m.refs))
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def same(self, code):
        torch.cuda.synchronize()
        assert int(self.status) == code
        self.status.zero_()
        for name in ("tables", "lengths", "refs", "pool"):
            assert torch.equal(getattr(self, name).cpu(), getattr(self.m, name)), name

    def reserve(self, seqs, counts):
        praghip.page_reserve(self.tables, self.lengths, self.refs, self.m.page, ints(seqs), ints(counts), self.status)
        self.same(self.m.reserve(seqs, counts))

    def free(self, seqs):
        praghip.page_free(self.tables, self.lengths, self.refs, ints(seqs), self.status)
        self.same(self.m.free(seqs))

    def trim(self, seqs, window, sinks):
        praghip.page_trim(self.tables, self.lengths, self.refs, self.m.page, ints(seqs), window, sinks, self.status)
        self.same(self.m.trim(seqs, window, sinks))

    def fork(self, parents, children):
        praghip.page_fork(self.pool, self.tables, self.lengths, self.refs, ints(parents), ints(children), self.status)
        self.same(self.m.fork(parents, children))

    def compact(self):
        praghip.page_compact(self.pool, self.tables, self.refs)
        self.same(self.m.compact())

    def write(self, layer, starts, seed):
        g = torch.Generator().manual_seed(seed)
        shape = (starts[-1], self.pool.shape[3], self.pool.shape[5])
        k, v = (torch.randn(shape, generator=g).to(self.pool.dtype) for _ in range(2))
        praghip.page_write(k.to("cuda"), v.to("cuda"), self.pool[layer, 0], self.pool[layer, 1], self.tables,
                           self.lengths, ints(starts))
        self.m.write(layer, k, v, starts)
        self.same(0)


def test_a_life_of_sequences(gpu):
    print("[pages] a life", flush=True)
    p = Pair(2, 60, 2, 16, 24, seqs=9, width=12, seed=1)
    p.reserve([0, 1, 2], [40, 1, 16])
    p.write(1, [0, 40, 41, 57] + [57] * 6, seed=2)
    p.reserve([1, 0], [1, 0])
    p.reserve([3], [0])
    p.fork([0, 0, 2, 1], [4, 5, 6, 7])          # 40 % 16 != 0: copied; 16: shared whole
    p.reserve([4, 5, 0], [9, 1, 30])            # a forked sequence grows on its own pages
    p.write(0, [0, 30, 30, 30, 30, 39, 40, 40, 40, 40], seed=3)
    p.free([0, 2])
    p.compact()
    p.compact()
    p.reserve([8, 0], [100, 33])
    p.trim([8], 20, 3)
    p.trim([8, 4], 20, 3)
    p.fork([8], [2])                            # a parent with trimmed pages
    p.free([8, 4, 5, 6, 7])
    p.compact()
    p.fork([3], [4])                            # an empty parent
    p.free([0, 1, 2, 3, 4])
    p.compact()
    assert int(p.m.refs.abs().sum()) == 0


def test_refused_calls_change_nothing(gpu):
    print("[pages] refusals", flush=True)
    p = Pair(1, 10, 1, 16, 16, seqs=6, width=8, seed=4)
    p.reserve([0, 1], [50, 64])
    for seqs, counts in (([0, 0], [1, 1]), ([6], [1]), ([-1], [1]), ([0], [79]), ([2, 3], [1, -1]), ([2], [49]),
                         ([2], [2 ** 31 - 1]), ([2, 3], [16, 48])):
        p.reserve(seqs, counts)
    p.free([1, 1])
    p.free([9])
    p.reserve([2], [32])                        # the pool is full now
    p.fork([0], [3])                            # no page for the last one's copy
    p.fork([1], [3])                            # nothing to copy: 64 is four pages
    p.fork([0], [1])                            # a child that is not empty
    p.fork([0, 1], [4, 4])
    p.fork([0, 4], [4, 5])                      # a child that is a parent
    p.fork([0], [17])
    with pytest.raises(praghip.PraghipError) as e:
        praghip.page_free(p.tables, p.lengths, p.refs, ints([7]), p.status)
        praghip.page_check(p.status)
    assert e.value.text == "E_PAGES_SEQUENCE"
    praghip.page_check(p.status)


@pytest.mark.parametrize("pages,seqs", [(3, 1), (64, 5), (65, 7), (1025, 40), (5000, 130)])
def test_many_pages(gpu, pages, seqs):
    """Counts over stretches of the pages that are short, whole and ragged."""
    print("[pages] many", pages, flush=True)
    g = torch.Generator().manual_seed(pages)
    p = Pair(1, pages, 1, 16, 8, seqs=2 * seqs, width=60, seed=5)
    share = pages // seqs * 16
    p.reserve(list(range(seqs)), torch.randint(0, min(share, 500) + 1, (seqs,), generator=g).tolist())
    gone = [s for s in range(seqs) if s % 3 != 1]
    p.free(gone)
    p.reserve(gone[::-1], [min(share, 300)] * len(gone))
    p.free(gone[::2])
    p.compact()
    kept = [s for s in range(seqs) if int(p.m.lengths[s])][:5]
    p.fork(kept, [seqs + i for i in range(len(kept))])
    p.compact()


def test_copy(gpu):
    print("[pages] copy", flush=True)
    g = torch.Generator().manual_seed(9)
    for shape, type in (((3, 2, 20, 2, 16, 24), torch.bfloat16), ((1, 20, 1, 16, 8), torch.float16), ((9, 4, 32, 64), torch.float32)):
        pool = torch.randn(shape, generator=g).to(type)
        dim = pool.dim() - 4
        want, got = pool.clone(), pool.to("cuda")
        praghip.page_copy(got, ints([1, 3, -1, 5, 3, 99]), ints([0, 8, 2, 40, 7, 6]))
        for a, b in ((1, 0), (3, 8), (3, 7)):
            want.select(dim, b).copy_(pool.select(dim, a))
        assert torch.equal(got.cpu(), want)
        praghip.page_copy(got, ints([]), ints([]))
        assert torch.equal(got.cpu(), want)


def test_write_drops_what_has_no_place(gpu):
    print("[pages] write", flush=True)
    p = Pair(1, 12, 3, 16, 40, seqs=3, width=4, seed=6, type=torch.float16)
    p.reserve([0, 2], [5, 40])
    p.tables[2, 1] = p.m.tables[2, 1] = -1
    p.lengths[1] = p.m.lengths[1] = 7           # a length without pages
    p.write(0, [0, 9, 12, 52], seed=7)          # four of the nine lie before the first token
    p.write(0, [0, 0, 0, 0], seed=8)
    # rows of a joint projection: k and v beside one another
    both = torch.randn((5, 6, 40), generator=torch.Generator().manual_seed(9)).half()
    dev = both.to("cuda")
    praghip.page_write(dev[:, :3], dev[:, 3:], p.pool[0, 0], p.pool[0, 1], p.tables, p.lengths, ints([0, 5, 5, 5]))
    p.m.write(0, both[:, :3], both[:, 3:], [0, 5, 5, 5])
    p.same(0)


def test_graph_replays(gpu):
    """A fork, a release and a compaction in one graph, against the same calls made eagerly."""
    print("[pages] graph", flush=True)
    a, b = (Pair(2, 40, 2, 16, 16, seqs=8, width=8, seed=10) for _ in range(2))
    for x in (a, b):
        x.reserve([0, 1], [40, 70])
        x.reserve([2], [20])
    parents, children, ended = ints([0, 0, 1]), ints([4, 5, 6]), ints([4, 5])
    more, ones = ints([0, 1, 2]), ints([1, 2, 1])

    def work(x):
        praghip.page_fork(x.pool, x.tables, x.lengths, x.refs, parents, children, x.status)
        praghip.page_free(x.tables, x.lengths, x.refs, ended, x.status)
        praghip.page_reserve(x.tables, x.lengths, x.refs, 16, more, ones, x.status)
        praghip.page_free(x.tables, x.lengths, x.refs, children[2:], x.status)
        praghip.page_compact(x.pool, x.tables, x.refs)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        work(a)
    for _ in range(4):
        graph.replay()
        work(b)
        torch.cuda.synchronize()
        for name in ("tables", "lengths", "refs", "pool", "status"):
            assert torch.equal(getattr(a, name), getattr(b, name)), name
    assert int(a.status) == 0


def test_argument_refusals(gpu):
    p = Pair(1, 10, 1, 16, 16, seqs=4, width=8, seed=11)

    def refused(text, call):
        with pytest.raises(praghip.PraghipError) as e:
            call()
        assert text in e.value.text, e.value.text

    one, t = ints([0]), (p.tables, p.lengths, p.refs)
    refused("E_PAGES_SHAPE", lambda: praghip.page_reserve(*t, 24, one, one))
    refused("E_PAGES_INTS", lambda: praghip.page_reserve(*t, 16, one.long(), one))
    refused("E_PAGES_SHAPE", lambda: praghip.page_reserve(*t, 16, one, ints([1, 2])))
    refused("E_PAGES_SHAPE", lambda: praghip.page_reserve(p.tables, p.lengths[:2], p.refs, 16, one, one))
    refused("E_PAGES_INTS", lambda: praghip.page_free(*t, one.cpu()))
    refused("E_PAGES_SHAPE", lambda: praghip.page_free(*t, torch.zeros(9000, dtype=torch.int32, device="cuda")))
    refused("E_PAGES_WINDOW", lambda: praghip.page_trim(*t, 16, one, 0))
    refused("E_PAGES_POOL", lambda: praghip.page_fork(p.pool.transpose(4, 5), *t, one, ints([1])))
    refused("E_PAGES_SHAPE", lambda: praghip.page_fork(p.pool[:, :, :5].contiguous(), *t, one, ints([1])))
    refused("E_PAGES_POOL", lambda: praghip.page_copy(p.pool[0, 0, 0], one, ints([1])))
    k = torch.zeros((1, 1, 16), dtype=torch.bfloat16, device="cuda")
    starts = ints([0, 1, 1, 1, 1])
    refused("E_ATTENTION_TYPE", lambda: praghip.page_write(k.float(), k, p.pool[0, 0], p.pool[0, 1], p.tables, p.lengths, starts))
    refused("E_ATTENTION_SHAPE", lambda: praghip.page_write(k, k[:, :, :8], p.pool[0, 0], p.pool[0, 1], p.tables, p.lengths, starts))
    refused("E_ATTENTION_SHAPE", lambda: praghip.page_write(k, k, p.pool[0, 0], p.pool[0, 1], p.tables, p.lengths, starts[:3]))
    p.same(0)
