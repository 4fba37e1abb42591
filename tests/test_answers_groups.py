"""Which neighbours of a list of answers read a prefix together (praghip.answers), without a GPU: the
runs that save the most keys, against all ways to cut the list, and forks of forks."""
import itertools
import random

import pytest

from praghip import answers


def best(common):
    """(keys saved, cut points) of the best of all cuts."""
    n, found = len(common) + 1, []
    for cuts in itertools.product((False, True), repeat=n - 1):
        at = [0] + [i + 1 for i in range(n - 1) if cuts[i]] + [n]
        found.append(sum((b - a - 1) * min(common[a: b - 1], default=0) for a, b in zip(at, at[1:])))
    return max(found)


@pytest.mark.parametrize("seed", range(60))
def test_runs_save_the_most(seed):
    r = random.Random(seed)
    common = [r.choice([0, 1, 2, 5, 40, 100, 101, 8000]) for _ in range(r.randint(0, 9))]
    at = answers._runs(common)
    assert at[0] == 0 and at[-1] == len(common) + 1 and all(a < b for a, b in zip(at, at[1:]))
    saved = [(b - a - 1) * min(common[a: b - 1], default=0) for a, b in zip(at, at[1:])]
    assert sum(saved) == best(common)
    assert all(s or b == a + 1 for s, a, b in zip(saved, at, at[1:]))  # neighbours that share nothing stay apart


class Tree(answers.Qwen3Answers):
    """What it keeps of forks and ends, with no model."""

    def __init__(self, slots):
        self.held, self.marks, self.states, self.changes = [0] * slots, [[] for _ in range(slots)], 0, 0

    def _said(self, sequence, n):
        self.held[sequence] += n

    fork = answers.Qwen3Answers._forked
    end = answers.Qwen3Answers._ended


def test_questions_over_one_system_prompt():
    """A prompt of 100 tokens for two questions of 8000, each with four answers."""
    m = Tree(11)
    m._said(0, 100)
    m.fork(0, [1, 2])
    m._said(1, 7900), m._said(2, 7900)
    m.fork(1, [3, 4, 5, 6])
    m.fork(2, [7, 8, 9, 10])
    assert m._groups([3, 4, 5, 6]) == ([0, 4], [8000], 24000)
    assert m._groups(range(3, 11)) == ([0, 4, 8], [8000, 8000], 48000)
    assert m._groups([0, 1, 2]) == ([0, 3], [100], 200)          # each of the three is another
    assert m._groups([3, 7, 4, 8]) == ([0, 4], [100], 300)       # no neighbours share more
    assert m._groups([0, 3, 4, 7]) == ([0, 1, 3, 4], [100, 8000, 8000], 8000)
    m.end([3])
    assert m._groups([4, 5, 6, 3, 7]) == ([0, 3, 4, 5], [8000, 0, 8000], 16000)


def test_answers_of_answers():
    """Shares fall along the list; what a run reads together is what its members all have."""
    m = Tree(8)
    m._said(0, 1000)
    m.fork(0, [1])
    m._said(1, 1000)
    m.fork(1, [2])
    m._said(2, 1000)
    m.fork(2, [3, 4])
    assert m._groups([4, 3, 2, 1, 0]) == ([0, 3, 5], [3000, 1000], 7000)
    assert m._groups([4, 3, 2, 1]) == ([0, 3, 4], [3000, 2000], 6000)  # (as many as all four over 2000)
    m.fork(0, [5, 6, 7])
    assert m._groups([5, 6, 7, 0, 4]) == ([0, 5], [1000], 4000)


def random_tree(seed):
    r, m, tokens = random.Random(seed), Tree(12), {s: [] for s in range(12)}
    count = 0
    for _ in range(60):
        s, empty = r.randrange(12), [x for x in range(12) if not m.held[x]]
        what = r.random()
        if what < 0.45:
            n = r.randint(1, 30)
            m._said(s, n)
            tokens[s] += range(count, count + n)
            count += n
        elif what < 0.85 and m.held[s] and empty:
            children = r.sample(empty, r.randint(1, min(3, len(empty))))
            m.fork(s, children)
            for c in children:
                tokens[c] = list(tokens[s])
        elif what < 0.95 and m.held[s]:
            m.end([s])
            tokens[s] = []
    return r, m, tokens


@pytest.mark.parametrize("seed", range(40))
def test_groups_share_what_they_say(seed):
    """After forks, ends and prompts at random: every group's shared tokens are the same tokens."""
    r, m, tokens = random_tree(seed)
    for _ in range(5):
        order = r.sample([s for s in range(12) if m.held[s]] or [0], r.randint(1, max(1, sum(map(bool, m.held)))))
        at, shared, saved = m._groups(order)
        assert at[0] == 0 and at[-1] == len(order) and saved == sum((b - a - 1) * n for a, b, n in zip(at, at[1:], shared))
        for a, b, n in zip(at, at[1:], shared):
            assert all(tokens[s][:n] == tokens[order[a]][:n] and len(tokens[s]) >= n for s in order[a: b])


def test_the_same_list_after_a_change():
    m = Tree(4)
    m._said(0, 500)
    m.fork(0, [1, 2])
    order = [1, 2]
    assert m._groups(order)[2] == 500 and m._groups(order) == m._groups(tuple(order))
    m.end([2])
    assert m._groups(order)[2] == 0
    m.fork(1, [2])
    assert m._groups(order)[2] == 500
