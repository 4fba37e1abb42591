"""Answers to several questions over one system prompt: each question's are read together, call by
call and as a captured graph, against a forward in 64 bits."""
import pytest
import torch

from praghip import answers
from test_gpu_answers import SHAPE, VOCAB, model, near, plain

pytestmark = pytest.mark.gpu


def prompt(n, seed):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
def test_two_questions(gpu, monkeypatch, type):
    print("[trees]", type, flush=True)
    # (as one group of six they would save 5 x 20 keys, as two of three 2 x 2 x 90)
    monkeypatch.setattr(answers, "_ENOUGH", 300)
    calls, shared = [], answers.paged_shared
    monkeypatch.setattr(answers, "paged_shared", lambda *a, **k: (calls.append(1), shared(*a, **k))[1])
    m = model(type, slots=9, pages=80, capacity=128)
    said = {0: prompt(20, 1)}
    m.extend([0], [said[0]])
    m.fork(0, [1, 2])
    for s in (1, 2):
        said[s] = said[0] + prompt(70, 1 + s)
    m.extend([1, 2], [said[1][20:], said[2][20:]])
    m.fork(1, [3, 4, 5])
    m.fork(2, [6, 7, 8])
    order = [3, 4, 5, 6, 7, 8]
    said |= {s: list(said[1 if s < 6 else 2]) for s in order}
    assert m._groups(order) == ([0, 3, 6], [90, 90], 360) and not calls
    for turn in range(2):
        new = prompt(6, 10 + turn)
        for s, t in zip(order, new):
            said[s].append(t)
        logits = m.extend(order, [[t] for t in new])
        assert len(calls) == SHAPE.layers * (turn + 1)
    for row, s in zip(logits, order):
        near(row, plain(m, said[s]), type)
    step = m.steps(order)
    for turn in range(4):
        new = prompt(6, 20 + turn)
        for s, t in zip(order, new):
            said[s].append(t)
        got = step(new).clone()
        torch.cuda.synchronize()
        for row, s in zip(got, order):
            near(row, plain(m, said[s]), type)
        if turn == 1:  # an answer to the other question in a place among the first's
            m.end([4])
            m.fork(2, [4])
            said[4] = list(said[2])
            assert m._groups(order) == ([0, 3, 6], [20, 90], 220)
