"""Where the memory of a step's calls on another stream comes from, without a GPU, as in
test_serving_streams.py, whose stand-ins for torch and its tensors these are."""
import pytest
import torch

import test_serving_streams as stand
from praghip import append, attention, norm, sample
from test_serving_streams import BF16, I32, SIDE, Library, Tensor

F32 = torch.float32


@pytest.fixture(autouse=True)
def without_a_gpu(monkeypatch):
    attention._load()
    sample._load()
    monkeypatch.setattr(stand, "fake", stand.Fake())
    stand.fake.int64 = torch.int64
    monkeypatch.setattr(attention, "_torch", stand.fake)
    monkeypatch.setattr(attention, "_current", lambda index: 3)
    monkeypatch.setattr(Tensor, "new_empty", lambda t, shape, dtype=None: stand.fake.empty(tuple(shape), dtype=dtype or t.dtype))
    for module in (append, attention, norm, sample):
        monkeypatch.setattr(module, "lib", Library)


def calls():
    q, kv, new = Tensor((2, 4, 64), BF16), Tensor((9, 2, 16, 64), BF16), Tensor((2, 2, 64), BF16)
    tables, lengths, starts = Tensor((2, 4), I32), Tensor((2,), I32), Tensor((3,), I32)
    turns, one, two = Tensor((64, 32), F32), Tensor((1,), I32), Tensor((2,), I32)
    x, w, rows, u = Tensor((2, 64), BF16), Tensor((64,), BF16), Tensor((2, 100), F32), Tensor((2,), F32)
    return {
        "shared": lambda **k: attention.paged_shared(q, kv, kv, tables, lengths, two, one, lse=True, **k),
        "append": lambda **k: append.page_append(q, new, new, kv, kv, tables, lengths, starts, turns, turns, **k),
        "norm": lambda **k: norm.add_norm(x, w, x, **k),
        "norm alone": lambda **k: norm.add_norm(x, w, **k),
        "sample": lambda **k: sample.sample_tokens(rows, u, **k),
    }


MADE = {"shared": 3, "append": 1, "norm": 2, "norm alone": 1, "sample": 2}  # results and workspaces


@pytest.mark.parametrize("name", MADE)
def test_memory_is_the_streams_own(name):
    got = calls()[name](stream=SIDE)
    assert len(stand.fake.made) == MADE[name] and all(t.made is SIDE for t in stand.fake.made)
    for t in got if isinstance(got, tuple) else (got,):
        assert t.recorded == ["current"]


@pytest.mark.parametrize("name", MADE)
def test_the_current_stream_takes_its_own(name):
    calls()[name]()
    assert len(stand.fake.made) == MADE[name]
    assert all(t.made == "current" and not t.recorded for t in stand.fake.made)
