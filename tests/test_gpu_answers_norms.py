"""Qwen3Answers with norm weights of 32 bits that its 16-bit type does not hold: they stay as they
are, in every norm, call by call and in a captured graph."""
import pytest
import torch

import praghip
from praghip.answers import Qwen3Answers, random_weights
from test_gpu_answers import GROUP, SHAPE, VOCAB, near, plain, wide as wide_weights

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def model(type, change, shape=SHAPE, **more):
    """A model whose norm weights `change` has made of ones."""
    weights = random_weights(shape, VOCAB, seed=3, type=type)
    g = torch.Generator(device="cuda").manual_seed(4)
    weights["norm"] = change(weights["norm"], g)
    for layer in weights["layers"]:
        for name in ("attention_norm", "mlp_norm", "q_norm", "k_norm"):
            layer[name] = change(layer[name], g)
    return weights, Qwen3Answers(weights, shape, group=GROUP, **more)


def wide(w, g):
    return 1 + 0.2 * torch.randn(w.shape, generator=g, device="cuda")


@pytest.mark.parametrize("type", [F16, BF16])
def test_they_are_kept(gpu, type):
    weights, m = model(type, wide, slots=1, pages=8, capacity=64)
    for name in ("attention_norm", "mlp_norm", "q_norm", "k_norm"):
        for layer, given in zip(m.layers, weights["layers"]):
            assert torch.equal(layer[name].float(), given[name])
    assert torch.equal(m.norm.float(), weights["norm"])


def test_weights_beyond_the_type(gpu):
    """Last weights above float16's largest number, of values whose products with them are below it."""
    shape = praghip.Qwen3Shape(layers=0, hidden=64, q_heads=4, kv_heads=2, head_dim=32, intermediate=96)
    weights = random_weights(shape, VOCAB, seed=3, type=F16)
    weights["embed"][:, 0] = 40  # (the others are about 1/8: the norm divides by 5)
    weights["norm"] = torch.full((64,), 7e4, device="cuda")
    weights["norm"][0] = 1
    m = Qwen3Answers(weights, shape, group=GROUP, slots=1, pages=8, capacity=64)
    for token in (1, 2, 100):
        near(m.extend([0], [[token]])[0], last_logits(m, token), F16)


def last_logits(m, token):
    x = m.embed[token].cpu().double()
    h = x * (x.square().mean() + m.eps).rsqrt() * m.norm.cpu().double()
    assert h.abs().max() < 65504 and m.norm.max() > 65504
    return h @ wide_weights(m.head)[:, :64].T


@pytest.mark.parametrize("type", [F16, BF16])
def test_answers(gpu, type):
    """A prompt, a token beside it, and a graph's tokens, against 64 bits."""
    print("[answers] wide norms", type, flush=True)
    _, m = model(type, wide, slots=3, pages=24, capacity=96)
    g = torch.Generator().manual_seed(5)
    said = {s: torch.randint(0, VOCAB, (40,), generator=g).tolist() for s in (0, 1)}
    logits = m.extend([0, 1], [said[0], said[1]])
    for s in (0, 1):
        near(logits[s], plain(m, said[s]), type)
    m.fork(0, [2])
    said[2] = list(said[0])
    step = m.steps([2, 1, 0])
    for i in range(4):
        new = torch.randint(0, VOCAB, (3,), generator=g).tolist()
        got = step(new).clone()
        for s, t in zip((2, 1, 0), new):
            said[s].append(t)
        torch.cuda.synchronize()
        for row, s in zip(got, (2, 1, 0)):
            near(row, plain(m, said[s]), type)


@pytest.mark.parametrize("type", [F16, BF16])
def test_each_norm_alone(gpu, type):
    """One norm of 32 bits among those that the type holds: the same calls on both sides of it."""
    for one in ("attention_norm", "mlp_norm", "q_norm", "k_norm", "norm"):
        weights = random_weights(SHAPE, VOCAB, seed=3, type=type)
        g = torch.Generator(device="cuda").manual_seed(6)
        if one == "norm":
            weights["norm"] = wide(weights["norm"], g)
        else:
            weights["layers"][1][one] = wide(weights["layers"][1][one], g)
        m = Qwen3Answers(weights, SHAPE, group=GROUP, slots=1, pages=8, capacity=64)
        tokens = list(range(20, 50))
        near(m.extend([0], [tokens])[0], plain(m, tokens), type)
