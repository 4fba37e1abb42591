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


def functions(code):
    """(name, instructions, addresses that branches on no active lanes go to) of each function."""
    start = 0
    for end in range(1, len(code) + 1):
        if end < len(code) and code[end][0] != "FUNC":
            continue
        part, name = code[start + 1: end], code[start][2]
        meet, start = set(), end
        for op, _, line in part:
            if op == "s_cbranch_execz":
                address, word = at(line)
                meet.add(address + 4 + 4 * ((word & 0xffff) - ((word & 0x8000) << 1)))
        yield name, part, meet


def leaves(op, line):
    return op.startswith("s_cbranch") or op in ("s_branch", "s_endpgm", "s_setpc_b64") or re.match(r"s_\w+ exec\b", line)


def put_by_some(code):
    found, regions = [], 0
    for name, part, meet in functions(code):
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
            elif leaves(op, line):
                puts = None
            elif puts is not None and PUT.match(line):
                puts.append(line)
    return found, regions


def test_nothing_is_put_away_by_some_lanes(machine_code):
    found, regions = put_by_some(machine_code)
    assert regions > 1000
    assert not found, found[:5]


def test_nothing_is_done_by_some_where_lanes_meet(machine_code):
    """From the target of a branch on no active lanes to where they are active again there is no
    vector instruction at all (but writes of a lane that is named, which need none active)."""
    found, met = [], 0
    for name, part, meet in functions(machine_code):
        run = None
        for op, _, line in part:
            if at(line)[0] in meet:
                run = []
            if run is None:
                continue
            if RESTORED.match(line):
                met += 1
                found += [(name, x) for x in run]
                run = None
            elif leaves(op, line) or "saveexec" in op:
                run = None
            elif re.match(r"(v|ds|global|flat|scratch|buffer)_", op) and op not in ("v_writelane_b32", "v_readlane_b32"):
                run.append(line)
    assert met > 1000
    assert not found, found[:5]
