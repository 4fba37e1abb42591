"""Qwen3Answers where answers share prefixes: which it finds, and the logits of reading them once
against a forward in 64 bits, call by call and as a captured graph."""
import pytest
import torch

import praghip
from praghip import answers
from test_gpu_answers import SHAPE, VOCAB, model, near, plain

pytestmark = pytest.mark.gpu


@pytest.fixture
def always(monkeypatch):
    """Any shared token is enough, and how often the call is made."""
    monkeypatch.setattr(answers, "_ENOUGH", 1)
    calls = []
    shared = answers.paged_shared

    def counted(*a, **k):
        calls.append(1)
        return shared(*a, **k)

    monkeypatch.setattr(answers, "paged_shared", counted)
    return calls


def prompt(n, seed):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def test_which_prefixes(gpu):
    m = model(torch.float16, slots=9, pages=60, capacity=128)
    m.extend([0, 1], [prompt(40, 1), prompt(20, 2)])
    assert m._groups([0, 1]) == ([0, 1, 2], [0, 0], 0)
    m.fork(0, [2, 3])
    m.fork(1, [4])
    assert m._groups([2, 3, 4]) == ([0, 2, 3], [40, 20], 40)
    assert m._groups([0, 2, 4, 3, 1]) == ([0, 2, 3, 4, 5], [40, 20, 40, 20], 40)
    m.extend([2], [[5, 6, 7]])
    m.fork(2, [5, 6])  # 2, 5 and 6 have 43 in common, and 40 with 0 and 3
    assert m._groups([2, 5, 6]) == ([0, 3], [43], 86)
    assert m._groups([2, 5, 3, 6]) == ([0, 4], [40], 120)
    m.fork(2, [7])     # from the same state
    assert m._groups([6, 7]) == ([0, 2], [43], 43) and len(m.marks[2]) == 2
    m.end([0, 2])
    assert m._groups([5, 6, 3]) == ([0, 3], [40], 80) and m._groups([0, 5]) == ([0, 1, 2], [0, 43], 0)
    m.extend([0], [prompt(30, 3)])
    assert m._groups([0, 3]) == ([0, 1, 2], [0, 40], 0)


@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
def test_answers_of_shared_prompts(gpu, always, type):
    print("[answers] shared", type, flush=True)
    m = model(type, slots=8, pages=70, capacity=192)
    said = {0: prompt(90, 4), 1: prompt(33, 5)}
    m.extend([0, 1], [said[0], said[1]])
    assert not always
    m.fork(0, [2, 3, 4])
    m.fork(1, [5])
    said |= {2: list(said[0]), 3: list(said[0]), 4: list(said[0]), 5: list(said[1])}
    active = [2, 3, 4, 5, 1]
    for step in range(5):
        new = prompt(5, 10 + step)
        for s, t in zip(active, new):
            said[s].append(t)
        logits = m.extend(active, [[t] for t in new])
        assert len(always) == SHAPE.layers * (step + 1)
        if step == 2:
            m.end([0])
            m.compact()
    for i, s in enumerate(active):
        near(logits[i], plain(m, said[s]), type)
    m.fork(3, [6])
    said[6] = list(said[3])
    new = prompt(3, 20)
    for s, t in zip([6, 3, 2], new):
        said[s].append(t)
    logits = m.extend([6, 3, 2], [[t] for t in new])
    for i, s in enumerate([6, 3, 2]):
        near(logits[i], plain(m, said[s]), type)


def test_steps_that_share(gpu, always):
    """Replays against an eager model that shares nothing, with ends, forks and other prompts
    between them."""
    print("[answers] steps that share", flush=True)
    both = [model(torch.float16, slots=6, pages=60, capacity=160) for _ in range(2)]
    said = {0: prompt(45, 6)}
    for m in both:
        m.extend([0], [said[0]])
        m.fork(0, [1, 2, 3])
    m, eager = both
    said |= {s: list(said[0]) for s in (1, 2, 3)}
    order = [3, 1, 2]
    step = m.steps(order)
    assert len(always) == 2 * SHAPE.layers  # the first time and the capture
    assert m.lengths.tolist() == eager.lengths.tolist() and torch.equal(m.pool, eager.pool)

    def alone(sequences, new):
        return torch.cat([eager.extend([s], [[t]]) for s, t in zip(sequences, new)])

    for i in range(16):
        new = prompt(3, 30 + i)
        got = step(torch.tensor(new, device="cuda")).clone()
        want = alone(order, new)
        for s, t in zip(order, new):
            said[s].append(t)
        near(got, want.cpu().double(), torch.float16)
        if i == 3:    # one ends, and another prompt takes its place
            for x in both:
                x.end([1])
                x.extend([1], [prompt(30, 7)])
            said[1] = prompt(30, 7)
        if i == 7:    # it branches off an answer that has gone on
            for x in both:
                x.end([1])
                x.fork(3, [1])
            said[1] = list(said[3])
        if i == 11:   # nothing is shared any more
            for x in both:
                x.end([0, 1, 2])
                x.extend([1, 2], [[3], [4, 5]])
            said |= {1: [3], 2: [4, 5]}
    for i, s in enumerate(order):
        near(got[i], plain(m, said[s]), torch.float16)


def test_a_window_shares_nothing(gpu, always):
    m = model(torch.float16, slots=3, pages=40, capacity=128, window=24, sinks=2)
    m.extend([0], [prompt(50, 8)])
    m.fork(0, [1, 2])
    m.extend([1, 2], [[3], [4]])
    m.steps([1, 2])([5, 6])
    assert not always


def test_norms_of_other_types_and_places(gpu):
    """Norm weights in 32 bits, and at an odd address."""
    weights = answers.random_weights(SHAPE, VOCAB, seed=3, type=torch.float16)
    want = answers.Qwen3Answers(weights, SHAPE, group=32, slots=1, pages=8, capacity=64).extend([0], [[1, 2, 3]])
    for layer in weights["layers"]:
        layer["q_norm"] = layer["q_norm"].float()
        layer["k_norm"] = torch.cat((layer["k_norm"][:1], layer["k_norm"]))[1:]
    got = answers.Qwen3Answers(weights, SHAPE, group=32, slots=1, pages=8, capacity=64).extend([0], [[1, 2, 3]])
    assert torch.equal(got, want)


def test_far_contexts(gpu):
    """Angles of a longer context, against 64 bits with the same ones."""
    m = model(torch.float16, slots=1, pages=8, capacity=128, rotary={"factor": 4.0})
    tokens = prompt(60, 9)
    got = m.extend([0], [tokens])
    cos, _ = praghip.rotary_table(128, SHAPE.head_dim, factor=4.0)
    assert torch.equal(m.cos, cos)
    same = model(torch.float16, slots=1, pages=8, capacity=128)
    assert not torch.allclose(same.extend([0], [tokens]).float(), got.float(), atol=1e-2)


@pytest.mark.parametrize("more", [[], ["--temperature", "0.8", "--top-k", "50", "--top-p", "0.9", "--min-p", "0.02"]])
def test_the_command(gpu, monkeypatch, capsys, more):
    monkeypatch.setattr("sys.argv", ["answers", "--prompt", "700", "--answers", "8", "--tokens", "4", *more])
    monkeypatch.setattr(answers, "random_weights", lambda: random_small())
    monkeypatch.setattr(answers, "Qwen3Answers", small)
    answers.main()
    out = capsys.readouterr().out
    assert "token" in out and "answers begin" in out


def random_small():
    return random_weights(praghip.Qwen3Shape(layers=2, hidden=64, q_heads=4, kv_heads=2, head_dim=32, intermediate=96), 32768)


random_weights, Model = answers.random_weights, answers.Qwen3Answers


def small(weights, **kw):
    return Model(weights, praghip.Qwen3Shape(layers=2, hidden=64, q_heads=4, kv_heads=2, head_dim=32, intermediate=96), group=32, **kw)
