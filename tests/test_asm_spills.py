"""Registers that the compiler keeps in accumulator registers or scratch memory, in the gfx950
machine code of the built library: none is put there by some of a wave's lanes alone.

Where a kernel has more values than registers, the compiler copies some away and back.  It may place
the copy at the start of the block in which the lanes of a condition come together again, before
the instruction that makes all of them active: lanes that did not take the condition then read
back whatever the accumulator register held.  An unlucky allocation of the shared prefixes' attention in
heads of 136 to 248 values took addresses from such lanes.  A straight run from where lanes leave (or
where they meet: the target of a branch on no active lanes) to where they are active again therefore
holds no such copy.
"""
import re

from test_asm_hazards import machine_code, pytestmark  # noqa: F401

RESTORED = re.compile(r"s_or_b64 exec, exec, ")
PUT = re.compile(r"v_accvgpr_write_b32 a\d+, v\d+|v_accvgpr_mov_b32|scratch_store_")


def at(line):
    """(address, first word) of an instruction."""
    m = re.search(r"// ([0-9A-F]+): ([0-9A-F]{8})", line)
    return int(m.group(1), 16), int(m.group(2), 16)


def put_by_some(code):
    found, regions = [], 0
    start = 0
    for end in range(1, len(code) + 1):  # a kernel's (an object's) instructions at a time
        if end < len(code) and code[end][0] != "FUNC":
            continue
        part = code[start + 1: end]
        name, start = code[start][2], end
        meet = set()
        for op, _, line in part:
            if op == "s_cbranch_execz":
                address, word = at(line)
                meet.add(address + 4 + 4 * ((word & 0xffff) - ((word & 0x8000) << 1)))
        puts = None  # in the run so far, where some lanes are active
        for op, _, line in part:
            if at(line)[0] in meet:
                puts = []
            if "saveexec" in op:
                puts = []
            elif puts is not None and RESTORED.match(line):
                regions += 1
                found += [(name, x) for x in puts]
                puts = None
            elif op.startswith("s_cbranch") or op in ("s_branch", "s_endpgm", "s_setpc_b64") or re.match(r"s_\w+ exec\b", line):
                puts = None
            elif puts is not None and PUT.match(line):
                puts.append(line)
    return found, regions


def test_nothing_is_put_away_by_some_lanes(machine_code):
    found, regions = put_by_some(machine_code)
    assert regions > 1000
    assert not found, found[:5]
