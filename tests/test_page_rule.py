"""The count of a reservation's new pages (csrc/page_rule.hpp), on the host."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def summed(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("page_rule") / "check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "privacy-rag_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "page_rule_check.cpp"), "-o", exe], check=True)

    def run(rows):
        text = "".join("%d %d %d %d\n" % r for r in rows)
        got = subprocess.run([exe], input=text, capture_output=True, text=True, check=True).stdout.strip()
        return got if got == "refused" else int(got)

    return run


def test_sums_beyond_32_bits(summed):
    for seqs, each in ((8192, 1 << 18), (4096, 1 << 20), (8192, 1 << 19), (8192, (1 << 27) - 1)):
        assert summed([(0, 16 * each, 1 << 27, 4)] * seqs) == seqs * each


@pytest.mark.parametrize("shift", [0, 4, 7, 15])
def test_pages_of_one_sequence(summed, shift):
    page, width = 1 << shift, 9
    most = page * width
    for old in sorted({0, 1, page - 1, page, page + 1, most - 1, most}):
        for more in sorted({0, 1, page - 1, page, page + 1, most - old}):
            want = -(-(old + more) // page) - -(-old // page) if old + more <= most else "refused"
            assert summed([(old, more, width, shift)]) == want, (old, more)


def test_what_may_not_be(summed):
    for row in ((-1, 2, 9, 4), (5, -1, 9, 4), (144, 1, 9, 4), (0, 2 ** 31 - 1, 9, 4)):
        assert summed([(0, 1, 9, 4), row, (0, 1, 9, 4)]) == "refused"


def test_a_length_has_32_bits(summed):
    most, width = 2 ** 31 - 1, 65600  # pages of 32768: room for more tokens than a length counts
    assert summed([(0, most, width, 15)]) == 65536
    assert summed([(most - 40000, 40000, width, 15)]) == 1
    for old, more in ((most, 1), (1, most), (most - 40000, 40001), (most, most)):
        assert summed([(old, more, width, 15)]) == "refused"
