"""What Qwen3Answers.steps and its calls do with what does not fit: nothing is changed."""
import pytest
import torch

import praghip
from praghip.answers import Qwen3Answers, random_weights

pytestmark = pytest.mark.gpu

SHAPE = praghip.Qwen3Shape(layers=2, hidden=64, q_heads=4, kv_heads=2, head_dim=32, intermediate=96)
VOCAB = 211


def model():
    m = Qwen3Answers(random_weights(SHAPE, VOCAB, seed=3, type=torch.float16), SHAPE, group=32, slots=4, pages=30, capacity=64)
    m.extend([0, 1], [[5, 6, 7, 8], [9] * 16])
    return m


def state(m):
    torch.cuda.synchronize()
    return [t.clone() for t in (m.tables, m.lengths, m.refs, m.status, m.pool)] + [list(m.held)]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a[:-1], b[:-1])) and a[-1] == b[-1]


@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_a_step_takes_one_whole_number_for_each_sequence(gpu, device):
    print("[steps] shapes", device, flush=True)
    m = model()
    step = m.steps([1, 0])
    before = state(m)
    for new in (torch.tensor(3), torch.tensor([3]), torch.tensor([3, 4, 5]), torch.tensor([[3, 4]]), torch.tensor([[3], [4]]),
                torch.tensor([], dtype=torch.int64), torch.tensor([3.0, 4.0]), torch.tensor([True, False])):
        with pytest.raises(ValueError):
            step(new.to(device))
    for new in ([3], [3, 4, 5], [], [3, -1], [VOCAB, 3], [3.5, 4.0], [[3], [4]]):
        with pytest.raises((ValueError, TypeError)):
            step(new)
    assert same(state(m), before)
    # and takes what it took
    want = m.extend([1, 0], [[3], [4]]).clone()
    m = model()
    step = m.steps([1, 0])
    for dtype in (torch.int64, torch.int32, torch.uint8):
        got = step(torch.tensor([3, 4], dtype=dtype, device=device)).clone()
        if dtype is torch.int64:
            assert (got.float() - want.float()).norm() <= 4 * 31 ** 0.5 * 2.0 ** -11 * want.float().norm()
    assert m.held == [7, 19, 0, 0] == m.lengths.tolist()


def test_a_first_time_that_fails_leaves_the_lengths(gpu, monkeypatch):
    """Memory that does not suffice for the graph's first run, say."""
    print("[steps] a first time that fails", flush=True)
    m = model()
    before = state(m)

    def fails(*a, **k):
        raise RuntimeError("out of memory")

    monkeypatch.setattr(m, "_logits", fails)
    with pytest.raises(RuntimeError, match="out of memory"):
        m.steps([0, 1])
    monkeypatch.undo()
    assert same(state(m), before)
    m.extend([0], [[3]])
    assert m.held == [5, 16, 0, 0] == m.lengths.tolist()
