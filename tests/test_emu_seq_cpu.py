"""tests/test_gpu_paged.py and tests/test_gpu_attention_seq.py, run unmodified against the CPU build of the kernels
(tests/emu_util.EmuContext): operands between inaccessible pages, tight against either one, LDS-DMA bytes arriving at issue
or as late as their wait allows.  By default the cases of a few seconds, each once; HODU_EMU_ALL=1 runs all of them, both ways (7 minutes
with seven workers)."""
import os

import pytest

import emu_util
import test_emu_gpu_suites_cpu as suites
import test_gpu_attention_seq
import test_gpu_paged

pytestmark = pytest.mark.skipif(emu_util.compiler() is None, reason="no host clang++ for the CPU build")


ALL = os.environ.get("HODU_EMU_ALL", "0") not in ("", "0")
# {test: the parameters of the cases that run by default}
HEAVY = {"many_sequences": [], "every_tile": [], "tables_longer_than_what_a_workgroup_holds_of_them": [], "chunks_over_the_cache": [], "longer_prompts": [],
         "scores_that_grow_along_the_keys": [], "prompt_layouts": [], "cache_layouts": [], "calls_in_a_row_give_the_same_bits": [],
         "keys_cut_across_workgroups": [["bf16", "f8e4m3", 64, 51]], "single_tokens_over_the_cache": [[64, "bf16", "bf16"]],
         "packed_prompts": [[True, 128, "f16"], [False, 64, "bf16"]]}


def _cases():
    for mod in (test_gpu_paged, test_gpu_attention_seq):
        for name, fn in sorted(vars(mod).items()):
            if name.startswith("test_") and getattr(fn, "__module__", "") == mod.__name__:
                for kwargs in suites._expansions(fn):
                    if ALL or name[5:] not in HEAVY or list(kwargs.values()) in HEAVY[name[5:]]:
                        yield pytest.param(fn, kwargs, id=name[5:] + ("[" + "-".join(str(v) for v in kwargs.values()) + "]" if kwargs else ""))


@pytest.mark.parametrize("tight,late", [("end", 1), ("start", 0)] if ALL else [("end", 1)])
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
