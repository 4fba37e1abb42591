"""page_reserve where its counts are largest: more new pages than 32 bits count."""
import pytest
import torch

import praghip

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("seqs,each", [
    (8192, 1 << 18),        # 2^31 - 1 pages (a sequence has one already)
    (8192, 1 << 19),        # 2^32 - 1
    (4096, 1 << 20),
    (8191, (1 << 20) - 1),
])
def test_more_pages_than_32_bits_count(gpu, seqs, each):
    print("[reserve]", seqs, each, flush=True)
    page = 16
    tables = torch.full((1, each), -1, dtype=torch.int32, device="cuda").expand(seqs, each)  # (a refused call writes none)
    lengths, refs = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (seqs, 1000))
    lengths[3] = 5
    rows, counts, status = torch.arange(seqs, dtype=torch.int32, device="cuda"), torch.full_like(lengths, each * page - 5), ints([0])
    held = lengths.clone()
    praghip.page_reserve(tables, lengths, refs, page, rows, counts, status)
    with pytest.raises(praghip.PraghipError) as e:
        praghip.page_check(status)
    assert e.value.text == "E_PAGES_EXHAUSTED"
    assert torch.equal(lengths, held) and not refs.any() and bool((tables[0] == -1).all())
