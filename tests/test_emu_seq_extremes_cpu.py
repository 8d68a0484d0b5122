"""tests/test_gpu_seq_extremes.py, run unmodified against the CPU build of the kernels (tests/emu_util.EmuContext); the taller one of the
two wide tiles, which share their source, with HODU_EMU_ALL=1 only."""
import os

import pytest

import emu_util
import test_emu_gpu_suites_cpu as suites
import test_gpu_seq_extremes

pytestmark = pytest.mark.skipif(emu_util.compiler() is None, reason="no host clang++ for the CPU build")


ALL = os.environ.get("HODU_EMU_ALL", "0") not in ("", "0")


def _cases():
    for name, fn in sorted(vars(test_gpu_seq_extremes).items()):
        if name.startswith("test_") and getattr(fn, "__module__", "") == test_gpu_seq_extremes.__name__:
            for kwargs in suites._expansions(fn):
                if not ALL and kwargs.get("tile") == 52:
                    continue
                yield pytest.param(fn, kwargs, id=name[5:] + "[" + "-".join(str(v) for v in kwargs.values()) + "]")


@pytest.mark.parametrize("fn,kwargs", list(_cases()))
def test_gpu_test_passes_in_the_cpu_build(fn, kwargs):
    ctx = emu_util.EmuContext()
    ctx.lds_fill(0xFF)
    try:
        fn(ctx=ctx, **kwargs)
    finally:
        ctx.close()
