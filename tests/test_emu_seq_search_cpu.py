"""tests/test_gpu_seq_search.py and tests/test_gpu_seq_exactness.py, run unmodified against the CPU build of the kernels
(tests/emu_util.EmuContext), by default the cases of a few seconds (HODU_EMU_ALL=1: all); and that the latter's bound would see
P rounded once."""
import os

import numpy as np
import pytest

import emu_util
import seq_util as S
import test_emu_gpu_suites_cpu as suites
import test_gpu_seq_exactness as exactness
import test_gpu_seq_search

needs_clang = pytest.mark.skipif(emu_util.compiler() is None, reason="no host clang++ for the CPU build")
ALL = os.environ.get("HODU_EMU_ALL", "0") not in ("", "0")
QUICK = {"long_sequences_among_many": [[0, 50], [0, 51], [0, 52]], "both_searches_give_the_same": [], "single_tokens_and_short_chunks": [[0, "bf16"], [2, "f16"]]}


def _cases():
    for mod in (test_gpu_seq_search, exactness):
        for name, fn in sorted(vars(mod).items()):
            if name.startswith("test_") and getattr(fn, "__module__", "") == mod.__name__:
                for kwargs in suites._expansions(fn):
                    if ALL or sorted(map(str, kwargs.values())) in [sorted(map(str, q)) for q in QUICK[name[5:]]]:
                        yield pytest.param(fn, kwargs, id=name[5:] + "[" + "-".join(str(v) for v in kwargs.values()) + "]")


@needs_clang
@pytest.mark.parametrize("fn,kwargs", list(_cases()))
def test_gpu_test_passes_in_the_cpu_build(fn, kwargs):
    ctx = emu_util.EmuContext()
    ctx.lds_fill(0xFF)
    try:
        fn(ctx=ctx, **kwargs)
    finally:
        ctx.close()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("size", range(4))
def test_the_bound_sees_p_rounded_once(dt, size):
    """the definition with P rounded to dt, and the row sum over it, as a kernel without the remainders' product would have it"""
    d, n, m = exactness.SIZES[size]
    q, k, v = (x.values for x in exactness.operands(dt, d, n, m, size))
    scale = S.scalar(d, dt)[1]
    got = np.zeros((n, 4, d))
    exact = np.zeros((n, 4, d))
    for h in range(4):
        for i in range(n):
            s = k[:, h // 2] @ q[i, h] * scale
            s[i + m - n + 1:] = -np.inf
            p = np.exp2(np.log2(np.e) * s - np.ceil(np.log2(np.e) * s.max()))
            rounded = S.widen(S.to_bits(p, dt), dt).reshape(p.shape)
            got[i, h] = rounded @ v[:, h // 2] / rounded.sum()
            exact[i, h] = p @ v[:, h // 2] / p.sum()
    got, exact = (S.widen(S.to_bits(x, dt), dt).reshape(x.shape) for x in (got, exact))
    assert exactness.outside(exact, q, k, v, dt, d, scale) == 0
    if dt == "bf16":  # (in f16 the bound's term for a P below its normal range covers a rounding as well)
        assert exactness.outside(got, q, k, v, dt, d, scale) > 0
