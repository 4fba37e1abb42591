"""page_reserve where its counts are largest: more new pages than 32 bits count, and lengths
that 32 bits hold no more."""
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


def test_a_length_of_32_bits(gpu):
    """A row of the tables with room for more than 2^31 - 1 tokens: so many are given, and no more."""
    print("[reserve] a length of 32 bits", flush=True)
    page, width, most = 32768, 65600, 2 ** 31 - 1
    tables = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
    lengths, refs, status = ints([0, 0]), torch.zeros(70000, dtype=torch.int32, device="cuda"), ints([0])

    def reserve(rows, counts):
        praghip.page_reserve(tables, lengths, refs, page, ints(rows), ints(counts), status)
        praghip.page_check(status)

    reserve([0], [most - 40000])
    assert lengths.tolist() == [most - 40000, 0]
    for rows, counts in (([0], [40001]), ([1, 0], [1, 40001]), ([0], [most])):
        before = tables.clone(), lengths.clone(), refs.clone()
        with pytest.raises(praghip.PraghipError) as e:
            reserve(rows, counts)
        assert e.value.text == "E_PAGES_CAPACITY"
        assert all(torch.equal(a, b) for a, b in zip((tables, lengths, refs), before))
    reserve([1, 0], [1, 40000])
    assert lengths.tolist() == [most, 1] and int(refs.sum()) == 65537
    assert torch.equal(tables[0, :65535].cpu(), torch.arange(65535, dtype=torch.int32))  # (as many were given first)
    with pytest.raises(praghip.PraghipError) as e:
        reserve([0], [1])
    assert e.value.text == "E_PAGES_CAPACITY"
    assert lengths.tolist() == [most, 1]
