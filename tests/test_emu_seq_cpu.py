"""tests/test_gpu_paged.py and tests/test_gpu_attention_seq.py, run unmodified against the CPU build of the kernels
(tests/emu_util.EmuContext): operands between inaccessible pages, tight against either one, LDS-DMA bytes arriving at issue
or as late as their wait allows."""
import pytest

import emu_util
import test_emu_gpu_suites_cpu as suites
import test_gpu_attention_seq
import test_gpu_paged

pytestmark = pytest.mark.skipif(emu_util.compiler() is None, reason="no host clang++ for the CPU build")


def _cases():
    for mod in (test_gpu_paged, test_gpu_attention_seq):
        for name, fn in sorted(vars(mod).items()):
            if name.startswith("test_") and getattr(fn, "__module__", "") == mod.__name__:
                for kwargs in suites._expansions(fn):
                    yield pytest.param(fn, kwargs, id=name[5:] + ("[" + "-".join(str(v) for v in kwargs.values()) + "]" if kwargs else ""))


@pytest.mark.parametrize("tight,late", [("end", 1), ("start", 0)])
@pytest.mark.parametrize("fn,kwargs", list(_cases()))
def test_gpu_test_passes_in_the_cpu_build(fn, kwargs, tight, late):
    ctx = emu_util.EmuContext(tight=tight)
    ctx.dma_lazy(late)
    ctx.lds_fill(0xFF)
    try:
        fn(ctx=ctx, **kwargs)
    finally:
        ctx.dma_lazy(0)
        ctx.close()
