"""A serving step -- paged plan, store, attention over the cache -- recorded into graphs and replayed with other inputs, two
graphs of one context in turn and eager work between them; and many launches in a row of the kernels whose workgroups meet
through the workspace."""
import numpy as np
import pytest

from hodu_amd import ffi
import seq_util as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = ffi.Context(0)
    yield c
    c.close()


class Step:
    """one decode or chunk step of `added` tokens per request behind `cached` ones, everything on the device"""

    def __init__(self, ctx, cached, added, hq, hk, d, page, cache_dt, tile, seed):
        self.ctx, self.g, self.tile, b, t = ctx, np.random.default_rng(seed), tile, len(cached), sum(added)
        self.added, width = np.array(added, np.int32), -(-max(c + 3 * a for c, a in zip(cached, added)) // page)
        pool, f8 = b * width, cache_dt == "f8e4m3"
        table = self.g.permutation(pool).reshape(b, width).astype(np.int32)
        held = [-(-c // page) for c in cached]
        free = np.concatenate([table[r, h:] for r, h in enumerate(held)])
        words = np.uint8 if f8 else np.uint16
        cache = [S.to_bits(self.g.standard_normal((pool, page, hk, d)), cache_dt) for _ in range(2)]
        self.kc, self.vc = (ctx.upload(c.astype(words)) for c in cache)
        self.cached, self.dadded, self.free, self.table = (ctx.upload(np.ascontiguousarray(x, np.int32)) for x in (cached, added, free, table))
        self.lens, self.offsets, self.slots, self.used = (ctx.alloc(4 * n) for n in (b, b + 1, t, 2))
        self.qkv, self.out = ctx.alloc(t * (hq + 2 * hk) * d * 2), ctx.alloc(t * hq * d * 2)
        self.dt, self.shape, self.row = "bf16", (t, hq, d), (hq + 2 * hk) * d
        scales = dict(k_scale=ctx.upload(np.full(hk, 0.02, np.float32)), v_scale=ctx.upload(np.full(hk, 0.03, np.float32))) if f8 else {}
        self.plan_md = ffi.paged_plan_md(b, page, width, len(free), t)
        self.store_md = ffi.paged_store_md(t, hk, d, pool, page, (self.row, d), (self.row, d), k_offset=hq * d, v_offset=(hq + hk) * d)
        self.md = ffi.paged_attention_md(b, t, hq, hk, d, pool, page, width, q_strides=(self.row, d))
        self.bits, self.kw = S.scalar(d, "bf16")[0], dict(cache_dt=cache_dt, **scales)

    def inputs(self):
        self.ctx.upload_into(self.qkv, S.to_bits(self.g.standard_normal((self.shape[0], self.row)), "bf16"))

    def calls(self):
        c = self.ctx
        c.force_tile(self.tile)
        c.paged_plan(self.cached, self.dadded, self.free, self.table, self.lens, self.offsets, self.slots, self.used, self.plan_md)
        c.paged_store(self.dt, self.qkv, self.qkv, self.kc, self.vc, self.slots, self.store_md, **self.kw)
        c.attention_paged(self.dt, self.qkv, self.kc, self.vc, self.out, self.offsets, self.table, self.lens, self.md, self.bits, **self.kw)
        c.force_tile(-1)

    def result(self):
        return self.ctx.download(self.out, np.uint16).copy()


@pytest.mark.parametrize("cache_dt", ["bf16", "f8e4m3"])
def test_steps_recorded_and_replayed(ctx, cache_dt):
    steps = [Step(ctx, [1500, 3000, 40], [1, 1, 1], 8, 2, 128, 16, cache_dt, 50, 1), Step(ctx, [1500, 2100], [20, 33], 4, 1, 64, 16, cache_dt, 51, 2)]
    graphs = []
    for s in steps:
        s.inputs()
        s.calls()  # (what grows grows outside the recording)
    for s in steps:
        graphs.append(ctx.record(s.calls))
    try:
        for _ in range(4):
            for s, graph in zip(steps, graphs):
                s.inputs()
                ctx.fill(s.out, 0xFF)
                graph.replay()
                got = s.result()
                s.calls()
                assert np.array_equal(got, s.result())
                assert np.isfinite(S.widen(got, "bf16")).all()
            for s, graph in zip(steps, graphs):  # the two back to back, through the one workspace
                ctx.fill(s.out, 0xFF)
                graph.replay()
            assert np.array_equal(steps[0].result(), run_again(steps[0])) and np.array_equal(steps[1].result(), run_again(steps[1]))
    finally:
        for graph in graphs:
            graph.free()


def run_again(step):
    step.calls()
    return step.result()


@pytest.mark.parametrize("tile", [50, 51, 52])
def test_many_launches_in_a_row(ctx, tile):
    """the counters that workgroups meet through are back at zero after each launch, and the ranges are added in their order"""
    step = Step(ctx, [2000, 1100, 3900], [1, 7, 12], 8, 1, 64, 16, "bf16", tile, 3)
    step.inputs()
    step.calls()
    want = step.result()
    for i in range(300):
        step.calls()
        if i % 50 == 0:
            assert np.array_equal(step.result(), want), i
    assert np.array_equal(step.result(), want)
