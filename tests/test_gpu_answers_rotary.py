"""Qwen3Answers for contexts beyond those of the training, against a forward in 64 bits with the
angles that the interpolation is defined by."""
import math

import pytest
import torch

from test_gpu_answers import SHAPE, VOCAB, model, near, wide

pytestmark = pytest.mark.gpu
DIM = SHAPE.head_dim


def plain(m, tokens, frequencies, magnitude=1.0):
    """Logits after the last of the tokens."""
    def normed(x, weight):
        return x * (x.square().mean(-1, keepdim=True) + m.eps).rsqrt() * weight.cpu().double()

    def product(x, w):
        return x @ wide(w)[:, : x.shape[-1]].T

    angle = torch.arange(len(tokens)).double()[:, None, None] * torch.tensor(frequencies, dtype=torch.float64)

    def turned(x):
        a, b = x.chunk(2, -1)
        return magnitude * torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()), -1)

    i = torch.arange(len(tokens))
    x = m.embed.cpu().double()[tokens]
    for layer in m.layers:
        qkv = product(normed(x, layer["attention_norm"]), layer["qkv"]).unflatten(1, (-1, DIM))
        q, k, v = qkv.split((SHAPE.q_heads, SHAPE.kv_heads, SHAPE.kv_heads), 1)
        q, k = turned(normed(q, layer["q_norm"])), turned(normed(k, layer["k_norm"]))
        k, v = (t.repeat_interleave(SHAPE.q_heads // SHAPE.kv_heads, 1) for t in (k, v))
        s = (q.transpose(0, 1) @ k.permute(1, 2, 0).contiguous() * DIM ** -0.5).masked_fill(i[None] > i[:, None], -math.inf)
        o = s.softmax(-1) @ v.transpose(0, 1).contiguous()
        x = x + product(o.transpose(0, 1).flatten(1), layer["o"])
        gate, up = product(normed(x, layer["mlp_norm"]), layer["gate_up"]).chunk(2, 1)
        x = x + product(torch.nn.functional.silu(gate) * up, layer["down"])
    return product(normed(x[-1:], m.norm), m.head)[0]


def linear(factor):
    return [1e6 ** (-2 * i / DIM) / factor for i in range(DIM // 2)]


def by_parts(factor, original, fast, slow):
    """Each frequency by how often it turns within the training's tokens, between the whole pairs on both sides."""
    pair = {n: DIM * math.log(original / (2 * math.pi * n)) / (2 * math.log(1e6)) for n in (fast, slow)}
    low, high = max(math.floor(pair[fast]), 0), min(math.ceil(pair[slow]), DIM - 1)
    made = []
    for i in range(DIM // 2):
        share = min(max((i - low) / (high - low), 0), 1)
        made.append(1e6 ** (-2 * i / DIM) * (1 - share + share / factor))
    return made


CASES = {"as trained": ({}, linear(1), 1.0),
         "linear": ({"factor": 4.0}, linear(4), 1.0),
         "by parts": ({"factor": 4.0, "original": 32}, by_parts(4, 32, 32, 1), 1.0),
         "by parts, scaled": ({"factor": 8.0, "original": 64, "fast": 8.0, "slow": 0.5, "magnitude": 0.1 * math.log(8) + 1},
                              by_parts(8, 64, 8, 0.5), 0.1 * math.log(8) + 1)}


@pytest.mark.parametrize("type", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", CASES)
def test_far_contexts(gpu, case, type):
    """A prompt, and tokens after it one by one."""
    print("[rotary]", case, type, flush=True)
    given, frequencies, magnitude = CASES[case]
    m = model(type, slots=1, pages=8, capacity=128, rotary=given)
    tokens = torch.randint(0, VOCAB, (90,), generator=torch.Generator().manual_seed(9)).tolist()
    near(m.extend([0], [tokens[:80]])[0], plain(m, tokens[:80], frequencies, magnitude), type)
    for n in range(81, 91):
        logits = m.extend([0], [tokens[n - 1: n]])
    want = plain(m, tokens, frequencies, magnitude)
    near(logits[0], want, type)
    # and the angles count: other ones' logits are far outside
    for other in CASES:
        if CASES[other][1:] != (frequencies, magnitude):
            with pytest.raises(AssertionError):
                near(logits[0], plain(m, tokens, *CASES[other][1:]), type)
