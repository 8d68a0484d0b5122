"""The generated gfx950 code of the attention kernels over packed sequences once more (tests/test_isa_attention_seq_cpu.py), where that
reads straight on or leaves long loops out:

 * no scratch memory at all, in a loop or outside;
 * the wait states behind a matrix instruction whose result is in vector registers, and in front of one whose source a vector
   instruction wrote, along every branch: from the end of a loop to its first instructions, out of it and into it;
 * every wide kernel has its pipelined loops: innermost ones with the matrix instructions of a step or two."""
import re

import pytest

from test_isa_attention_seq_cpu import kernels, operands, registers, states  # noqa: F401 (a fixture)
from test_isa_hazards_cpu import HIPCC

pytestmark = pytest.mark.skipif(HIPCC is None, reason="no hipcc to generate the assembly with")


def test_no_scratch(kernels):  # noqa: F811
    for name, lines in kernels.items():
        assert not [x for x in lines if x.startswith("scratch_")], name


def paths(lines, n=14):
    """the instructions around every branch that is taken: up to n before it, and n from its target on"""
    at, code = {}, []
    for x in lines:
        if x.endswith(":"):
            at[x[:-1]] = len(code)
        else:
            code.append(x)
    for i, x in enumerate(code):
        m = re.match(r"s_c?branch\w*\s+(\.LBB\w+)", x)
        if m and m.group(1) in at:
            yield code[max(0, i - n):i + 1], code[at[m.group(1)]:at[m.group(1)] + n]


def test_wait_states_along_branches(kernels):  # noqa: F811
    for name, lines in kernels.items():
        if "wide" not in name:
            continue  # (compiler builtins only: it counts for itself)
        for before, behind in paths(lines):
            code = before + behind
            for i, line in enumerate(before):
                if not line.startswith("v_mfma"):
                    continue
                result, waited = registers(operands(line)[0]), 0
                for after in code[i + 1:]:
                    if waited >= 8 or after.startswith(("s_branch", "s_endpgm")) and after is not before[-1]:
                        break
                    if after.startswith("v_mfma"):
                        o = operands(after)
                        assert not (registers(o[1]) | registers(o[2])) & result, (name, line, after)
                    elif not after.startswith("s_"):
                        assert not registers(after) & result, (name, line, after)
                    waited += states(after)
            for i, line in enumerate(behind):
                if not line.startswith("v_mfma"):
                    continue
                ops, waited = operands(line), 0
                sources = registers(ops[1]) | registers(ops[2]) | registers(ops[3])
                for earlier in reversed(code[:len(before) + i]):
                    if waited >= 2:
                        break
                    if earlier.startswith("v_") and not earlier.startswith(("v_mfma", "v_cmp")):
                        assert not registers(operands(earlier)[0]) & sources, (name, earlier, line)
                    waited += states(earlier)


def loops(lines):
    """(first, last) of every loop, by its branch back"""
    at = {x[:-1]: i for i, x in enumerate(lines) if x.endswith(":")}
    return [(at[m.group(1)], i) for i, x in enumerate(lines) for m in [re.match(r"s_c?branch\w*\s+(\.LBB\w+)", x)] if m and at.get(m.group(1), i) < i]


def test_every_wide_kernel_has_pipelined_loops(kernels):  # noqa: F811
    for name, lines in kernels.items():
        m = re.search(r"wide_kernelILi\d+ELi(\d+)ELb\dELb\dELi(\d)E", name)
        if not m:
            continue
        d, rt = int(m.group(1)), int(m.group(2))
        step = rt * (2 * d // 32 + d // 16 + 1)  # scores, P V, the row sums
        counts = [sum(x.startswith("v_mfma") for x in lines[a:b]) for a, b in loops(lines)]
        assert any(n >= 2 * step for n in counts), (name, step, counts)
