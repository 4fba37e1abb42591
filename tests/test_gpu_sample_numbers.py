"""sample_tokens' filters as numbers: what is refused, in the call's own words, and what counts as
what, beside the same values as lists."""
import math

import numpy as np
import pytest
import torch

import praghip

pytestmark = pytest.mark.gpu


def given(rows=6, vocab=300):
    g = torch.Generator().manual_seed(1)
    return (torch.randn((rows, vocab), generator=g) * 2).cuda(), torch.rand(rows, generator=g).cuda()


@pytest.mark.parametrize("top_k", [5.0, 5.5, math.nan, math.inf, "5", np.float32(3)])
def test_counts_that_are_not_whole(gpu, top_k):
    with pytest.raises(praghip.PraghipError) as e:
        praghip.sample_tokens(*given(), top_k=top_k)
    assert e.value.text == "E_SAMPLE_FILTER"


@pytest.mark.parametrize("top_k", [np.int64(5), np.int32(5), 5])
def test_whole_numbers_of_any_kind(gpu, top_k):
    logits, u = given()
    want = praghip.sample_tokens(logits, u, top_k=torch.full((6,), 5, dtype=torch.int32, device="cuda"))
    assert torch.equal(praghip.sample_tokens(logits, u, top_k=top_k), want)


@pytest.mark.parametrize("name,number,other", [("top_p", 1e39, 1.0), ("top_p", 7.0, 1.0), ("temperature", 1e39, math.inf),
                                               ("temperature", 1e-50, 0.0), ("top_k", 2 ** 31 - 1, 0)])
def test_numbers_beyond_the_range(gpu, name, number, other):
    """Of 32 bits, and those that filter nothing."""
    logits, u = given()
    assert torch.equal(praghip.sample_tokens(logits, u, **{name: number}), praghip.sample_tokens(logits, u, **{name: other}))


def test_a_least_weight_above_one(gpu):
    """Refused as a number; of a list it counts as 1, as the largest weight is."""
    logits, u = given()
    with pytest.raises(praghip.PraghipError) as e:
        praghip.sample_tokens(logits, u, min_p=1.5)
    assert e.value.text == "E_SAMPLE_FILTER"
    got = praghip.sample_tokens(logits, u, min_p=torch.full((6,), 1.5, device="cuda"))
    assert torch.equal(got, praghip.sample_tokens(logits, u, min_p=1.0)) and torch.equal(got, logits.argmax(-1))
