"""What a captured graph holds stays allocated while its context lives, in the CPU build (tests/emu_util.EmuContext): the workspace
that a recorded call took is not freed when a later call outgrows it, and the sizes that the attention launcher asks
for, which do not grow with the rows."""
import numpy as np
import pytest

import emu_util
import seq_util as S
from hodu_amd import ffi

pytestmark = pytest.mark.skipif(emu_util.compiler() is None, reason="no host clang++ for the CPU build")


@pytest.fixture()
def ctx():
    c = emu_util.EmuContext()
    yield c
    if c.handle is not None:
        c.close()


def workspace_bytes(ctx):
    n, a, f = (ffi.ctypes.c_size_t(), ffi.ctypes.c_int(), ffi.ctypes.c_int())
    ctx._check(ctx.debug.hodu_rocm_debug_scratch_state(ctx.handle, *(ffi.ctypes.byref(x) for x in (n, a, f))))
    return n.value


class Call:
    """attention of `added` tokens of each request over the cache, every page of it the same one; `cached` is what the
    table has room for, `lens` what there is"""

    def __init__(self, ctx, batch, added, cached, lens, hq=4, hk=1, d=64, page=64):
        self.ctx, t, width = ctx, batch * added, cached // page
        g = np.random.default_rng(added)
        self.q, self.kc, self.vc = (ctx.upload(S.to_bits(g.standard_normal(n), "bf16")) for n in (t * hq * d, page * hk * d, page * hk * d))
        self.out, self.n = ctx.alloc(t * hq * d * 2), t * hq * d
        self.offsets = ctx.upload(np.arange(0, t + 1, added, dtype=np.int32))
        self.table, self.lens = ctx.upload(np.zeros((batch, width), np.int32)), ctx.upload(np.full(batch, lens, np.int32))
        self.md, self.bits = ffi.paged_attention_md(batch, t, hq, hk, d, 1, page, width), S.scalar(d, "bf16")[0]

    def __call__(self):
        self.ctx.attention_paged("bf16", self.q, self.kc, self.vc, self.out, self.offsets, self.table, self.lens, self.md, self.bits)

    def result(self):
        return self.ctx.download(self.out, np.uint16).copy()


def allocations(ctx):
    return ctx.lib.emu_live_allocations()


def test_a_recorded_workspace_outlives_its_growth(ctx):
    before = allocations(ctx)
    one, large = Call(ctx, 1, 1, 4096, 4000), Call(ctx, 4, 448, 8192, 0, hq=32, hk=8, d=128)
    operands = allocations(ctx) - before
    one()
    want = one.result()
    graph = ctx.record(one)
    small = workspace_bytes(ctx)
    assert small > 0
    large()  # (no key, so nothing but the launch; the launcher cannot know)
    assert workspace_bytes(ctx) > small
    # operands, the counters, two workspaces: the recorded one is still there
    assert allocations(ctx) - before == operands + 3
    ctx.fill(one.out, 0xFF)
    graph.replay()
    assert np.array_equal(one.result(), want)
    large()
    one()
    assert np.array_equal(one.result(), want)
    graph.free()
    for x in (one, large):
        for b in (x.q, x.kc, x.vc, x.out, x.offsets, x.table, x.lens):
            b.free()
    ctx.close()
    assert allocations(ctx) == before


def test_a_workspace_that_no_graph_holds_is_freed(ctx):
    before = allocations(ctx)
    one, large = Call(ctx, 1, 1, 4096, 100), Call(ctx, 4, 448, 8192, 0, hq=32, hk=8, d=128)
    operands = allocations(ctx) - before
    one()
    small = workspace_bytes(ctx)
    large()
    assert workspace_bytes(ctx) > small and allocations(ctx) - before == operands + 2


def test_a_call_that_would_grow_it_is_refused_while_recording(ctx):
    one, large = Call(ctx, 1, 1, 4096, 100), Call(ctx, 4, 448, 8192, 0, hq=32, hk=8, d=128)
    one()
    with pytest.raises(ffi.HoduRocmError) as e:
        ctx.record(large)
    assert e.value.status == 5 and "captured" in str(e.value)  # HODU_ROCM_SCRATCH


def test_fewer_rows_may_need_more_workspace(ctx):
    """the reason that no order of calls makes the workspace large enough once and for all"""
    few, many = Call(ctx, 4, 448, 8192, 0, hq=32, hk=8, d=128), Call(ctx, 4, 512, 8192, 0, hq=32, hk=8, d=128)
    many()
    after_many = workspace_bytes(ctx)
    few()
    assert workspace_bytes(ctx) > after_many
