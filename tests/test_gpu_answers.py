"""A Qwen3-shaped model on the serving calls together against a forward in 64 bits over
whole sequences, without a cache, from the same 4-bit weights."""
import pytest
import torch

import praghip
from praghip.answers import Qwen3Answers, random_weights

pytestmark = pytest.mark.gpu

SHAPE = praghip.Qwen3Shape(layers=2, hidden=64, q_heads=4, kv_heads=2, head_dim=32, intermediate=96)
VOCAB, GROUP = 211, 32


def model(type, **more):
    weights = random_weights(SHAPE, VOCAB, seed=3, type=type, device="cpu")
    g = torch.Generator().manual_seed(4)  # norms that are not all one
    for t in [weights["norm"]] + [w for layer in weights["layers"] for w in layer.values() if w.dim() == 1]:
        t.copy_(1 + 0.2 * torch.randn(t.shape, generator=g))

    def to(w):
        return w.cuda() if isinstance(w, torch.Tensor) else [to(x) for x in w] if isinstance(w, list) else \
            {n: to(x) for n, x in w.items()}

    return Qwen3Answers(to(weights), SHAPE, group=GROUP, **more)


def wide(w):
    """The weights that 4 bits with scales and zero points stand for, in 64 bits."""
    packed, scales, zeros = (t.cpu() for t in w)
    digits = torch.stack((packed & 15, packed >> 4), -1).flatten(1).double()
    groups = scales.shape[1]
    digits = digits[:, : groups * GROUP].unflatten(1, (groups, -1))
    return ((digits - zeros.double()[..., None]) * scales.double()[..., None]).flatten(1)


def plain(m, tokens):
    """Logits after the last of the tokens."""
    def normed(x, weight):
        return x * (x.square().mean(-1, keepdim=True) + m.eps).rsqrt() * weight.cpu().double()

    def product(x, w):
        return x @ wide(w)[:, : x.shape[-1]].T

    n, d = len(tokens), SHAPE.head_dim
    angle = torch.arange(n).double()[:, None, None] * 1e6 ** (-torch.arange(0, d, 2).double() / d)

    def turned(x):
        a, b = x.chunk(2, -1)
        return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)

    i = torch.arange(n)
    seen = i[None] <= i[:, None]
    if m.window:
        seen &= (i[None] > i[:, None] - m.window) | (i[None] < m.sinks)
    x = m.embed.cpu().double()[tokens]
    for layer in m.layers:
        qkv = product(normed(x, layer["attention_norm"]), layer["qkv"]).unflatten(1, (-1, d))
        q, k, v = qkv.split((SHAPE.q_heads, SHAPE.kv_heads, SHAPE.kv_heads), 1)
        q, k = turned(normed(q, layer["q_norm"])), turned(normed(k, layer["k_norm"]))
        k, v = (t.repeat_interleave(SHAPE.q_heads // SHAPE.kv_heads, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) * d ** -0.5
        o = torch.einsum("hqk,khd->qhd", s.masked_fill(~seen, -torch.inf).softmax(-1), v)
        x = x + product(o.flatten(1), layer["o"])
        gate, up = product(normed(x, layer["mlp_norm"]), layer["gate_up"]).chunk(2, 1)
        x = x + product(torch.nn.functional.silu(gate) * up, layer["down"])
    return product(normed(x[-1:], m.norm), m.head)[0]


def near(got, want, type):
    # 14 roundings to 16 bits along each of two layers and three at the end, each passed on
    # with about its own relative size, add like a random walk; four times that
    u = 2.0 ** -11 if type is torch.float16 else 2.0 ** -8
    got = got.cpu().double()
    assert (got - want).norm() <= 4 * 31 ** 0.5 * u * want.norm(), float((got - want).norm() / want.norm())


@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 2)])
def test_answers_of_two_prompts(gpu, type, window, sinks):
    print("[answers]", type, window, sinks, flush=True)
    m = model(type, slots=6, pages=24, capacity=128, window=window, sinks=sinks)
    g = torch.Generator().manual_seed(5)
    said = {0: torch.randint(0, VOCAB, (61,), generator=g).tolist(), 1: torch.randint(0, VOCAB, (16,), generator=g).tolist()}
    m.extend([0], [said[0][:40]])  # a prompt in two pieces, the second with another beside it
    logits = m.extend([0, 1], [said[0][40:], said[1]])
    for s in (0, 1):
        near(logits[s], plain(m, said[s]), type)
    m.fork(0, [2, 3])
    m.fork(1, [4])
    said |= {2: list(said[0]), 3: list(said[0]), 4: list(said[1])}
    active = [3, 4, 2]
    for step in range(4):  # answers that go apart over the shared pages
        new = torch.randint(0, VOCAB, (3,), generator=g).tolist()
        for s, t in zip(active, new):
            said[s].append(t)
        logits = m.extend(active, [[t] for t in new])
        if step == 1:  # the prompts end, and what is left moves together
            m.end([0, 1])
            m.compact()
            held = int((m.refs > 0).sum())
            assert bool((m.refs[:held] > 0).all())
    for i, s in enumerate(active):
        near(logits[i], plain(m, said[s]), type)
        assert int(m.lengths[s]) == m.held[s] == len(said[s])
    m.end(active)
    assert not m.refs.any() and bool((m.tables == -1).all())


def test_pages_that_do_not_suffice(gpu):
    m = model(torch.float16, slots=2, pages=3, capacity=128)
    m.extend([0], [[1] * 30])
    with pytest.raises(praghip.PraghipError, match="E_PAGES_EXHAUSTED"):
        m.extend([1], [[1] * 17])
    with pytest.raises(praghip.PraghipError, match="E_PAGES_CAPACITY"):
        m.extend([0], [[1] * 99])
    assert m.held == [30, 0] == m.lengths.tolist()
    near(m.extend([1], [[5, 6, 7]])[0], plain(m, [5, 6, 7]), torch.float16)


def test_the_last_position_and_what_is_refused(gpu):
    """A capacity that is no whole number of pages is rounded up, and its last position used."""
    m = model(torch.float16, slots=2, pages=8, capacity=20)
    tokens = [(7 * i) % VOCAB for i in range(32)]
    m.extend([0], [tokens[:31]])
    near(m.extend([0], [tokens[31:]])[0], plain(m, tokens), torch.float16)
    with pytest.raises(praghip.PraghipError, match="E_PAGES_CAPACITY"):
        m.extend([0], [[1]])
    for bad in ([[]], [[VOCAB]], [[-1]], [[1], [2]]):
        with pytest.raises(ValueError):
            m.extend([1], bad)
    for sequences in ([1, 1], [2], [-1]):
        with pytest.raises(praghip.PraghipError, match="E_PAGES_SEQUENCE"):
            m.extend(sequences, [[1]] * len(sequences))
    with pytest.raises(praghip.PraghipError, match="E_PAGES_SEQUENCE"):
        m.fork(0, [0])
    assert m.held == [32, 0] == m.lengths.tolist()


@pytest.mark.parametrize("window,sinks", [(0, 0), (24, 2)])
def test_steps_of_a_captured_graph(gpu, window, sinks):
    """Every replay against an eager model with the same tokens, with forks, ends, compactions
    and eager extensions between them, and the last against 64 bits."""
    print("[answers] steps", window, sinks, flush=True)
    both = [model(torch.float16, slots=4, pages=30, capacity=128, window=window, sinks=sinks) for _ in range(2)]
    g = torch.Generator().manual_seed(6)
    said = {0: torch.randint(0, VOCAB, (45,), generator=g).tolist()}
    for m in both:
        m.extend([0], [said[0]])
        m.fork(0, [1, 2])
    said |= {1: list(said[0]), 2: list(said[0])}
    m, eager = both
    step = m.steps([2, 1])
    assert m.lengths.tolist() == eager.lengths.tolist() and torch.equal(m.pool, eager.pool)
    for i in range(20):
        new = torch.randint(0, VOCAB, (2,), generator=g).tolist()
        got = step(new if i % 2 else torch.tensor(new, device="cuda"))
        want = eager.extend([2, 1], [[t] for t in new])
        said[2].append(new[0]), said[1].append(new[1])
        # (the launch's size may differ, and with it the order of a sum)
        near(got, want.cpu().double(), torch.float16)
        if i == 5:
            for x in both:
                x.end([0])
                x.compact()
        if i == 9:
            for x in both:
                x.extend([1], [[3, 4, 5]])
            said[1] += [3, 4, 5]
    for i, s in enumerate((2, 1)):
        near(got[i], plain(m, said[s]), torch.float16)
    for bad in ([], [4], [-1]):
        with pytest.raises(ValueError):
            m.steps(bad)
    with pytest.raises(ValueError):
        step([1])
    with pytest.raises(ValueError):
        step([1, VOCAB])
    assert m.lengths.tolist() == eager.lengths.tolist() == m.held
