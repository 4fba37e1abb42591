"""Which entry of a table the shared prefixes' attention looks up (csrc/shared_rule.hpp), on the host:
the next blocks of a wave may lie beyond the table, and beyond 2^31 positions."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def looked_up(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("shared_rule") / "check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "privacy-rag_amd", "csrc"),
                    os.path.join(ROOT, "tests", "cpp", "shared_rule_check.cpp"), "-o", exe], check=True)

    def run(rows):
        text = "".join("%d %d %d %d\n" % r for r in rows)
        got = subprocess.run([exe], input=text, capture_output=True, text=True, check=True).stdout
        return [int(x) for x in got.split()]

    return run


@pytest.mark.parametrize("shift", [4, 5, 7, 10, 15])
@pytest.mark.parametrize("positions", [1, 500, 2 ** 20, 2 ** 30, 2 ** 31 - 1 - 64])
def test_entries_of_the_table(looked_up, shift, positions):
    """As whole numbers of any size have them, eight blocks beyond the table's last position too."""
    width = max(1, positions >> shift)  # whole pages, as the kernels count a table's positions
    blocks = -(-(width << shift) // 32)
    rows = [(b, half, shift, width - 1) for b in range(max(0, blocks - 40), blocks + 9) for half in (0, 1)]
    assert looked_up(rows) == [min(32 * b + 16 * half >> shift, width - 1) for b, half, _, _ in rows]
