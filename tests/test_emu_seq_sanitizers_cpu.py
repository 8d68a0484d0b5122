"""The serving operators' tests of the CPU build under the race detector and under AddressSanitizer (opt-in, as in
tests/test_emu_races_cpu.py and tests/test_emu_address_cpu.py, whose lists they are not on): HODU_EMU_ALL=1 runs their default
cases under ThreadSanitizer, HODU_EMU_ALL=2 under AddressSanitizer too."""
import glob
import os
import subprocess
import sys

import pytest

import emu_util
from test_emu_races_cpu import OPTIONS, run

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FILES = ["test_emu_seq_cpu.py", "test_emu_seq_extremes_cpu.py", "test_emu_seq_search_cpu.py", "test_emu_paged_limits_cpu.py", "test_emu_graph_memory_cpu.py",
         "test_emu_stream_cpu.py", "test_emu_operand_checks_cpu.py"]
PYTEST = [*[os.path.join("tests", f) for f in FILES], "-q", "-x", "-p", "no:cacheprovider"]
pytestmark = pytest.mark.skipif(emu_util.compiler() is None, reason="no host clang for the CPU build")


@pytest.mark.skipif(os.environ.get("HODU_EMU_ALL", "") in ("", "0"), reason="a quarter of an hour; set HODU_EMU_ALL=1")
def test_under_the_race_detector(tmp_path):
    python = emu_util.build_race_checked_python()
    if python is None:
        pytest.skip("no Python headers or library to link the sanitizer-carrying interpreter")
    log = str(tmp_path / "report")
    # (one thread for torch's own loops, which are not instrumented)
    r = run([python, "-m", "pytest", *PYTEST], TSAN_OPTIONS=OPTIONS + f" exitcode=0 log_path={log}", HODU_EMU_SANITIZE="thread", HODU_EMU_ALL="0", OMP_NUM_THREADS="1",
            PYTHONPATH=os.pathsep.join(p for p in sys.path if p))
    reports = "".join(open(p).read() for p in glob.glob(log + ".*"))
    assert "ThreadSanitizer" not in reports, reports[:4000]
    assert " passed" in r.stdout and " failed" not in r.stdout, r.stdout[-3000:]


@pytest.mark.skipif(os.environ.get("HODU_EMU_ALL", "") != "2", reason="most of an hour; set HODU_EMU_ALL=2")
def test_under_the_address_sanitizer():
    python = emu_util.build_race_checked_python("address")
    if python is None:
        pytest.skip("no Python headers or library to link the sanitizer-carrying interpreter")
    env = {**os.environ, "HODU_EMU_SANITIZE": "address", "HODU_EMU_ALL": "0", "PYTHONPATH": os.pathsep.join(p for p in sys.path if p),
           "ASAN_OPTIONS": "detect_stack_use_after_return=0:detect_leaks=0:verify_asan_link_order=0"}
    r = subprocess.run([python, "-m", "pytest", *PYTEST], capture_output=True, text=True, cwd=ROOT, env=env)
    assert "AddressSanitizer" not in r.stderr and "AddressSanitizer" not in r.stdout, r.stdout[-3000:] + r.stderr[-3000:]
    assert r.returncode == 0 and " passed" in r.stdout, r.stdout[-3000:] + r.stderr[-3000:]
