"""The library's calls on torch's streams: tests/stream_checks.py, run once in a process that imports torch before the library."""
import os
import subprocess
import sys

import pytest

import stream_checks

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def output():
    r = subprocess.run([sys.executable, "-u", os.path.abspath(stream_checks.__file__)], capture_output=True, text=True, timeout=100)
    return r.stdout + r.stderr


@pytest.mark.parametrize("check", [c.__name__ for c in stream_checks.CHECKS])
def test_on_torchs_streams(output, check):
    assert f"ok {check}\n" in output, output[-3000:]
