"""Where the memory of a serving call on another stream comes from, without a GPU: what the
call writes is made under its stream, and what it returns is kept for the current one."""
import contextlib
import types

import pytest
import torch

from praghip import attention, matvec, pages


class Tensor:
    """What the calls ask of a tensor on the GPU, and which streams it was made under and
    recorded on."""

    def __init__(self, shape, dtype, strides=None, made=None):
        self.shape, self.dtype, self.device, self.made, self.recorded = torch.Size(shape), dtype, "cuda:0", made, []
        self._strides = strides or [int(torch.Size(shape[i + 1:]).numel()) for i in range(len(shape))]

    requires_grad = False

    def stride(self, i=None):
        return tuple(self._strides) if i is None else self._strides[i]

    def get_device(self):
        return 0

    def data_ptr(self):
        return 1 << 40

    def is_contiguous(self):
        return True

    def element_size(self):
        return 2

    def record_stream(self, stream):
        self.recorded.append(stream)

    def new_empty(self, shape):
        return fake.empty(shape, dtype=self.dtype)


class Fake:
    """torch, as far as the calls use it: the streams' contexts and every tensor made."""

    def __init__(self):
        self.now, self.made = "current", []
        self.cuda = types.SimpleNamespace(stream=self.under, current_stream=lambda index=None: self.now)
        self.float32 = torch.float32

    @contextlib.contextmanager
    def under(self, stream):
        before, self.now = self.now, stream
        yield
        self.now = before

    def empty(self, shape, dtype=None, device=None):
        t = Tensor((shape,) if isinstance(shape, int) else tuple(shape), dtype, made=self.now)
        self.made.append(t)
        return t

    def empty_like(self, t):
        return self.empty(t.shape, dtype=t.dtype)

    def is_grad_enabled(self):
        return True


fake = None
SIDE = types.SimpleNamespace(cuda_stream=5)
BF16, I32, U8 = torch.bfloat16, torch.int32, torch.uint8


class Library:
    """Every call is done, and every workspace has a size."""

    def __getattr__(self, name):
        return (lambda *a: 4096) if name.endswith("_workspace") else (lambda *a: 0)


@pytest.fixture(autouse=True)
def without_a_gpu(monkeypatch):
    global fake
    attention._load()
    fake = Fake()
    monkeypatch.setattr(attention, "_torch", fake)
    monkeypatch.setattr(attention, "_current", lambda index: 3)
    for module in (attention, matvec, pages):
        monkeypatch.setattr(module, "lib", Library)


def calls():
    q, kv = Tensor((2, 4, 64), BF16), Tensor((9, 2, 16, 64), BF16)
    tables, lengths, starts = Tensor((2, 4), I32), Tensor((2,), I32), Tensor((3,), I32)
    pool, refs, two = Tensor((1, 2, 9, 2, 16, 64), BF16), Tensor((9,), I32), Tensor((2,), I32)
    x, w, s = Tensor((2, 64), BF16), Tensor((32, 32), U8), Tensor((32, 1), BF16)
    return {
        "decode": lambda **k: attention.paged_decode(q, kv, kv, tables, lengths, lse=True, **k),
        "prompt": lambda **k: attention.paged_prompt(q, kv, kv, tables, lengths, starts, 1, lse=True, **k),
        "fork": lambda **k: pages.page_fork(pool, tables, lengths, refs, two, two, **k),
        "compact": lambda **k: pages.page_compact(pool, tables, refs, **k),
        "w4": lambda **k: matvec.matvec_w4(x, w, s, **k),
    }


MADE = {"decode": 3, "prompt": 3, "fork": 1, "compact": 1, "w4": 1}  # results and workspaces


@pytest.mark.parametrize("name", MADE)
def test_memory_is_the_streams_own(name):
    got = calls()[name](stream=SIDE)
    assert len(fake.made) == MADE[name] and all(t.made is SIDE for t in fake.made)
    # what comes back may be read on the current stream, and let go with that under way
    for t in got if isinstance(got, tuple) else () if got is None else (got,):
        assert t.recorded == ["current"]


@pytest.mark.parametrize("name", MADE)
def test_the_current_stream_takes_its_own(name):
    calls()[name]()
    assert len(fake.made) == MADE[name]
    assert all(t.made == "current" and not t.recorded for t in fake.made)
