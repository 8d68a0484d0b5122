"""The generated gfx950 code of the attention kernels over packed sequences, for what neither the hardware nor the compiler
sees to (cross-compiled here, no GPU).  Their scores come out of matrix instructions in assembly with vector registers as the
result: the compiler's hazard recogniser does not know when such a result is there, and its allocator may place a copy right
behind.  Held to, for every kernel of the file:

 * no instruction but another matrix instruction's accumulation names a matrix instruction's result within 8 wait states of it (a
   16x16x32 instruction runs 16 cycles, 4 states; its result is there 7 states after issue at the latest);
 * two wait states between a vector instruction and a matrix instruction that takes its result;
 * the value of an exponential is not used by the very next instruction;
 * no scratch memory inside a loop that holds a matrix instruction, and few registers spilled outside."""
import os
import re
import subprocess

import pytest

from hodu_amd.build import FLAGS as BUILD_FLAGS
from test_isa_hazards_cpu import CSRC, HIPCC

pytestmark = pytest.mark.skipif(HIPCC is None, reason="no hipcc to generate the assembly with")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{symbol: [instruction or label]}"""
    out = tmp_path_factory.mktemp("isa") / "seq.s"
    r = subprocess.run([HIPCC, *BUILD_FLAGS, "--cuda-device-only", "-S", os.path.join(CSRC, "attention_seq.hip"), "-o", str(out)], capture_output=True,
                       text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    found, now = {}, None
    for line in out.read_text().split("\n"):
        line = line.split(";")[0].strip()
        m = re.fullmatch(r"(_ZN\w*seq_attention\w*):", line)
        if m:
            now = found.setdefault(m.group(1), [])
        elif line.startswith(".Lfunc_end"):
            now = None
        elif now is not None and line and (not line.startswith(".") or line.endswith(":")):
            now.append(line)
    assert len(found) == 36, sorted(found)  # (16 rows, two wide heights) x (packed, paged, paged 8-bit) x 2 types x 2 head dims
    return found


def registers(text):
    out = set()
    for m in re.finditer(r"\b([va])(\d+)\b|\b([va])\[(\d+):(\d+)\]", text):
        out |= {m.group(1) + m.group(2)} if m.group(1) else {m.group(3) + str(i) for i in range(int(m.group(4)), int(m.group(5)) + 1)}
    return out


def operands(line):
    return [o.strip() for o in line.split(None, 1)[1].split(",")] if " " in line else []


def states(line):
    return int(line.split()[1], 0) + 1 if line.startswith("s_nop") else 4 if line.startswith("v_mfma") else 1


def test_matrix_results_and_sources_have_their_wait_states(kernels):
    for name, lines in kernels.items():
        lines = [x for x in lines if not x.endswith(":")]
        if "wide" not in name:
            continue  # (compiler builtins only: it counts for itself)
        for i, line in enumerate(lines):
            if not line.startswith("v_mfma"):
                continue
            ops, waited = operands(line), 0
            result = registers(ops[0])
            for after in lines[i + 1:i + 12]:
                if waited >= 8:
                    break
                if after.startswith("v_mfma"):
                    o = operands(after)
                    assert not (registers(o[1]) | registers(o[2])) & result, (name, line, after)
                elif not after.startswith("s_"):
                    assert not registers(after) & result, (name, line, after)
                waited += states(after)
            sources, waited = registers(ops[1]) | registers(ops[2]) | registers(ops[3]), 0
            for before in reversed(lines[max(i - 6, 0):i]):
                if waited >= 2:
                    break
                if before.startswith("v_") and not before.startswith(("v_mfma", "v_cmp")):
                    assert not registers(operands(before)[0]) & sources, (name, before, line)
                waited += states(before)


def test_exponentials_are_not_used_at_once(kernels):
    for name, lines in kernels.items():
        for line, after in zip(lines, lines[1:]):
            if line.startswith("v_exp_f32") and after.startswith("v_") and not after.startswith("v_exp"):
                assert not registers(operands(line)[0]) & registers(",".join(operands(after)[1:])), (name, line, after)


def test_no_scratch_in_the_loops(kernels):
    for name, lines in kernels.items():
        at = {x[:-1]: i for i, x in enumerate(lines) if x.endswith(":")}
        for i, line in enumerate(lines):
            m = re.match(r"s_c?branch\w*\s+(\.LBB\w+)", line)
            if m and at.get(m.group(1), i) < i:  # a branch back: the loop's own blocks
                body = lines[at[m.group(1)]:i]
                if sum(x.startswith("v_mfma") for x in body) and len(body) < 1400:
                    assert not any(x.startswith("scratch_") for x in body), (name, m.group(1))
