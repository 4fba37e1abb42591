"""The serving calls have no backward pass, and say so where one would be asked for."""
import pytest
import torch

import attention_plain as plain
import praghip
from praghip.answers import Qwen3Answers, random_weights

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def calls():
    c = plain.make([40, 20], 4, 2, 64, 16, BF16, seed=51, fill=0.0)
    k, v, tables, lengths = (c[x].to("cuda") for x in ("k", "v", "tables", "lengths"))
    q, new = (torch.randn((2, n, 64), generator=c["g"]).to(BF16).to("cuda") for n in (4, 2))
    starts = torch.arange(3, dtype=torch.int32, device="cuda")
    x = torch.randn((2, 64), generator=c["g"]).to(BF16).to("cuda")
    w, s, z = praghip.quantize_w4(torch.randn((32, 64), generator=c["g"]).to(BF16).to("cuda"), 32, zeros=True)
    return {
        "decode": ((q, k, v), lambda q, k, v: praghip.paged_decode(q, k, v, tables, lengths), "E_ATTENTION_GRADIENT"),
        "prompt": ((q, k, v), lambda q, k, v: praghip.paged_prompt(q, k, v, tables, lengths, starts, 1), "E_ATTENTION_GRADIENT"),
        "write": ((new, new.clone(), k, v), lambda a, b, k, v: praghip.page_write(a, b, k, v, tables, lengths, starts),
                  "E_ATTENTION_GRADIENT"),
        "w4": ((x, s), lambda x, s: praghip.matvec_w4(x, w, s, z, group=32), "E_W4_GRADIENT"),
    }


@pytest.mark.parametrize("name", ["decode", "prompt", "write", "w4"])
def test_inputs_that_require_gradients(gpu, name):
    inputs, call, text = calls()[name]
    want = call(*inputs)
    for i in range(len(inputs)):
        some = [t.clone().requires_grad_() if i == j else t for j, t in enumerate(inputs)]
        with pytest.raises(praghip.PraghipError) as e:
            call(*some)
        assert e.value.text == text
        for off in (torch.no_grad, torch.inference_mode):
            with off():
                got = call(*some)
            assert want is None or (torch.equal(got, want) and not got.requires_grad)


def test_a_model_of_parameters(gpu):
    """Weights that a training program holds: served as they are, without gradients."""
    shape = praghip.Qwen3Shape(layers=1, hidden=64, q_heads=4, kv_heads=2, head_dim=32, intermediate=96)
    weights = random_weights(shape, 211, seed=3, type=torch.float16)
    want = Qwen3Answers(weights, shape, group=32, slots=2, pages=8, capacity=64).extend([0], [[1, 2, 3]])
    for t in [weights["embed"], weights["norm"]] + [w for layer in weights["layers"] for w in layer.values()]:
        t.requires_grad_()
    m = Qwen3Answers(weights, shape, group=32, slots=2, pages=8, capacity=64)
    got = m.extend([0], [[1, 2, 3]])
    assert torch.equal(got, want) and not got.requires_grad
    assert not any(t.requires_grad for t in praghip.quantize_w4(weights["embed"], 32, zeros=True))
    assert torch.equal(m.steps([0])([4]).isfinite(), torch.ones_like(want, dtype=torch.bool))
