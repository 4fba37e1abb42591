"""Wait states between a VALU write of an SGPR and a memory instruction that takes its
address from it, in the gfx950 machine code of the built library.

The prompt attention's DMA (attention_prompt.hip) is inline asm whose base address comes
out of v_readlane.  The hardware needs five wait states there, and the compiler, which
adds them before its own loads, does not see the dependency into the asm: without them
the load goes to an address of whatever the register held before.
"""
import re

import pytest

from test_asm_hazards import block_start, last_writer, machine_code, pytestmark, sgpr_defs, sgprs, wait_states  # noqa: F401

MEMORY = re.compile(r"(global|buffer|flat|scratch)_")


def addresses(op, ops, line):
    """SGPRs that a memory instruction reads (its operands may carry modifiers)."""
    found = set()
    for tok in ops:
        found |= sgprs(tok.split()[0]) if tok else set()
    return found - {"vcc_lo", "vcc_hi", "m0"}


def test_memory_reads_five_wait_states_after_a_valu_write(machine_code):
    reads = bad = 0
    worst = []
    for i, (op, ops, line) in enumerate(machine_code):
        if not MEMORY.match(op):
            continue
        for reg in addresses(op, ops, line):
            w = last_writer(machine_code, i, {reg})
            if w and w[1]:
                reads += 1
                if w[0] < 5:
                    bad += 1
                    worst.append((machine_code[w[2]][2], line))
    assert reads > 0  # the prompt attention's DMA
    assert bad == 0, (bad, worst[:5])


def test_m0_before_the_prompt_attention_dma(machine_code):
    """A write of M0, scalar or by a VALU, at least one wait state before an LDS DMA."""
    dmas = bad = 0
    for i, (op, ops, line) in enumerate(machine_code):
        if not op.startswith("global_load_lds"):
            continue
        w = last_writer(machine_code, i, {"m0"})
        if w:
            dmas += 1
            bad += w[0] < 1
    assert dmas > 0 and bad == 0


def test_addresses_come_from_lanes_that_are_on(machine_code):
    """The prompt attention keeps 64 addresses across a wave's lanes.  Loaded where some lanes
    are off (as when a compiler moves them to memory and back inside a branch), the others'
    would be taken from whatever the register held before."""
    taken = 0
    bad = []
    for i, (op, ops, line) in enumerate(machine_code):
        if not op.startswith("v_readlane"):
            continue
        taken += 1
        source, load = ops[1], None
        for k in range(i - 1, max(0, i - 200), -1):
            o, p, text = machine_code[k]
            if o == "FUNC":
                break
            if load is None:
                if p and p[0].split()[0] == source:
                    if not (MEMORY.match(o) and "load" in o):
                        break
                    load = text
            elif "saveexec" in o or (p and p[0] == "exec"):
                if o.startswith(("s_and_saveexec", "s_andn2_saveexec")):
                    bad.append((load, line))
                break
    assert taken > 0 and not bad, bad[:5]
