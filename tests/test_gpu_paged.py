"""Block tables, slot maps and the stores into the paged cache against their definitions written out in numpy
(tests/seq_util.py): whole numbers and copied words equal, 8-bit values equal to the f32 quotient rounded by torch."""
import numpy as np
import pytest
import torch

from hodu_amd import ffi
import seq_util as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = ffi.Context(0)
    yield c
    c.close()


def check_plan(ctx, cached, added, page, width, n_free, capacity, seed=0):
    g = np.random.default_rng(seed)
    cached, added = np.array(cached, np.int32), np.array(added, np.int32)
    b = len(cached)
    table = g.integers(0, 1 << 20, (b, width)).astype(np.int32)
    free = g.permutation(n_free + 7)[:n_free].astype(np.int32)
    want = S.plan_reference(cached, added, free, table, page, capacity)
    dev = [ctx.upload(np.concatenate([x.ravel(), np.array([-77], np.int32)])) for x in
           (cached, added, free, table, np.zeros(b, np.int32), np.zeros(b + 1, np.int32), np.zeros(capacity, np.int32), np.zeros(2, np.int32))]
    for _ in range(2):  # (taking the same pages again gives the same: the inputs are left as they were)
        ctx.paged_plan(*dev, ffi.paged_plan_md(b, page, width, n_free, capacity))
        got = [ctx.download(d, np.int32) for d in dev]
        for name, x, w in zip(("table", "lens", "offsets", "slots", "used"), got[3:], want):
            assert np.array_equal(x[:-1], w.ravel()), (name, x[:-1][:40], w.ravel()[:40])
        assert all(x[-1] == -77 for x in got)  # nothing behind an output
        for x, w in zip(got[:3], (cached, added, free)):
            assert np.array_equal(x[:-1], w)


@pytest.mark.parametrize("page", [1, 3, 16, 24, 64, 256])
def test_plan_of_mixed_requests(ctx, page):
    g = np.random.default_rng(page)
    for b in (1, 2, 63, 64, 65, 257, 300):
        cached = g.integers(0, 200, b) * g.integers(0, 2, b)
        added = np.where(g.random(b) < 0.5, 1, g.integers(0, 90, b))
        width = -(-int((cached + added).max()) // page) + 1
        check_plan(ctx, cached, added, page, width, int(sum(-(-(c + n) // page) for c, n in zip(cached, added))), int(added.sum()) + 5, seed=b)


def test_plan_at_the_ends_of_pages(ctx):
    for page in (1, 16, 24):
        cached = [0, 0, page - 1, page, page + 1, 2 * page, 2 * page - 1, 5]
        added = [0, page, 1, 1, page - 1, 0, 2, 0]
        check_plan(ctx, cached, added, page, 8, 40, sum(added))
    check_plan(ctx, [], [], 16, 4, 3, 6)  # no request: every slot is -1
    check_plan(ctx, [0, 0], [0, 0], 16, 4, 0, 0)
    check_plan(ctx, [0], [0], 16, 0, 0, 0)


def test_plan_refuses_what_does_not_fit(ctx):
    check_plan(ctx, [3, -1, 5, 6], [4, 2, -3, 1], 4, 4, 10, 30)          # negative lengths
    check_plan(ctx, [0, 0, 0], [40, 17, 16], 4, 4, 100, 100)              # rows of the table too short
    check_plan(ctx, [0, 0, 3, 0, 3], [8, 8, 1, 4, 1], 4, 4, 3, 100)       # the list runs out; who needs no page still goes on
    check_plan(ctx, [0, 0, 0, 0], [8, 8, 1, 0], 4, 4, 100, 9)             # the slots run out
    check_plan(ctx, [0, 0, 2, 0, 1], [8, 9, 1, 4, 2], 4, 4, 4, 12)        # both
    check_plan(ctx, [2 ** 31 - 1, 0], [2 ** 31 - 1, 3], 4, 4, 9, 9)       # a sum beyond 32 bits
    check_plan(ctx, [0] * 600, [2 ** 31 - 1] * 600, 1 << 20, 2047, 9, 9)  # running sums beyond 32 bits


def test_plan_argument_checks(ctx):
    b = ctx.alloc(4096)
    bufs = [ctx.alloc(4096) for _ in range(8)]
    ok = ffi.paged_plan_md(4, 16, 4, 8, 8)
    for md, status in (((4, 0, 4, 8, 8), ffi.INVALID_ARG), ((4, 16, 4, 8), ffi.INVALID_ARG), ((4, 1 << 30, 4, 8, 8), ffi.UNSUPPORTED),
                       ((4, 16, 4, 8, 1 << 40), None), ((400, 16, 4, 8, 8), None)):
        with pytest.raises(ffi.HoduRocmError) as e:
            ctx.paged_plan(*bufs, md)
        assert status is None or e.value.status == status
    with pytest.raises(ffi.HoduRocmError):  # two outputs in one place
        ctx.paged_plan(bufs[0], bufs[1], bufs[2], bufs[3], b, bufs[5], b, bufs[7], ok)
    with pytest.raises(ffi.HoduRocmError):  # an output over an input
        ctx.paged_plan(b, bufs[1], bufs[2], bufs[3], b, bufs[5], bufs[6], bufs[7], ok)
    big = ctx.alloc(1 << 20)
    with pytest.raises(ffi.HoduRocmError) as e:
        ctx.paged_plan(big, ctx.alloc(1 << 20), bufs[2], ctx.alloc(1 << 20), ctx.alloc(1 << 20), ctx.alloc(1 << 20), bufs[6], bufs[7],
                       ffi.paged_plan_md(20000, 16, 4, 8, 8))
    assert e.value.status == ffi.UNSUPPORTED


def check_store(ctx, dt, cache_dt, tokens, hk, d, page, seed=0, k_order=None, c_order=None, gap=0, offset=0, extra_heads=0, skip=(), special=False):
    g = np.random.default_rng(seed)
    pages = -(-tokens // page) + 3
    joint = g.standard_normal((tokens, 2 * hk + extra_heads, d)) * 30.0
    if special:
        flat = joint.reshape(-1)
        flat[::17], flat[5::19], flat[7::23], flat[9::29] = np.inf, np.nan, 0.0, -1e30 if dt == "bf16" else -6e4
        flat[11::31] = 1e-7
    rows = S.Side(joint, dt, k_order, gap, offset)
    kc, vc = S.make_cache(g, cache_dt, pages, page, hk, d, c_order, gap, offset), S.make_cache(g, cache_dt, pages, page, hk, d, c_order, gap, 2 * offset)
    slots = g.permutation(pages * page)[:tokens].astype(np.int32)
    for i, bad in enumerate(skip):
        if i < tokens:
            slots[i] = bad
    ks, vs = g.uniform(0.01, 0.3, hk).astype(np.float32), g.uniform(0.01, 0.3, hk).astype(np.float32)
    scales = dict(k_scale=ctx.upload(ks), v_scale=ctx.upload(vs)) if cache_dt == "f8e4m3" else {}
    drows, dk, dv = ctx.upload(rows.flat), ctx.upload(kc.flat), ctx.upload(vc.flat)
    head = rows.strides[1]
    md = ffi.paged_store_md(tokens, hk, d, pages, page, rows.strides[:2], rows.strides[:2], kc.strides[:3], vc.strides[:3],
                            rows.offset + extra_heads * head, rows.offset + (extra_heads + hk) * head, kc.offset, vc.offset)
    ctx.paged_store(dt, drows, drows, dk, dv, ctx.upload(slots), md, cache_dt=cache_dt, **scales)
    words = rows.view(rows.flat)
    for cache, dev, sc, at in ((kc, dk, ks, extra_heads), (vc, dv, vs, extra_heads + hk)):
        want = cache.flat.copy()
        w = cache.view(want)
        for t, s in enumerate(slots):
            if 0 <= s < pages * page:
                if cache_dt != "f8e4m3":
                    w[s // page, s % page] = words[t, at:at + hk]
                else:
                    x = torch.from_numpy(words[t, at:at + hk].view(np.int16).copy()).view(S.TORCH[dt]).float() / torch.from_numpy(sc)[:, None]
                    w[s // page, s % page] = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        got = ctx.download(dev, want.dtype)
        if cache_dt == "f8e4m3":  # (a NaN may keep its sign)
            nan = (want & 0x7F) == 0x7F
            assert np.array_equal((got & 0x7F) == 0x7F, nan)
            got, want = np.where(nan, 0, got), np.where(nan, 0, want)
        assert np.array_equal(got, want), np.argwhere(got != want)[:5]


@pytest.mark.parametrize("dt,cache_dt", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8e4m3"), ("f16", "f8e4m3")])
def test_store_into_slots(ctx, dt, cache_dt):
    for n, (tokens, hk, d, page) in enumerate([(1, 1, 64, 16), (1, 8, 128, 1), (7, 2, 128, 24), (33, 3, 64, 16), (130, 8, 128, 64), (65, 5, 8, 3), (9, 1, 72, 256)]):
        check_store(ctx, dt, cache_dt, tokens, hk, d, page, seed=n)
    check_store(ctx, dt, cache_dt, 21, 2, 64, 16, seed=20, skip=(-1, -2 ** 31, 2 ** 31 - 1, 5 * 16))  # skipped slots
    check_store(ctx, dt, cache_dt, 21, 2, 64, 16, seed=21, extra_heads=4)                        # rows of a joint projection
    check_store(ctx, dt, cache_dt, 18, 3, 64, 8, seed=22, k_order=(1, 0), c_order=(0, 2, 1), gap=16, offset=32)  # heads first, gaps, offsets
    check_store(ctx, dt, cache_dt, 18, 3, 64, 8, seed=23, c_order=(2, 0, 1), gap=8, offset=8)
    check_store(ctx, dt, cache_dt, 40, 2, 128, 16, seed=24, special=True)                        # infinities, NaN, zeros, tiny and huge values


def test_store_of_nothing_and_refusals(ctx):
    x, c, s = ctx.alloc(1 << 16), ctx.alloc(1 << 16), ctx.upload(np.zeros(64, np.int32))
    c2, f = ctx.alloc(1 << 16), ctx.upload(np.ones(8, np.float32))
    ctx.fill(c, 0x5A)
    ctx.paged_store("bf16", x, x, c, c2, s, ffi.paged_store_md(0, 2, 64, 4, 16))
    ctx.sync()
    assert np.all(ctx.download(c, np.uint8) == 0x5A)
    md = ffi.paged_store_md(4, 2, 64, 4, 16)
    for args, kw, status in (
            (("bf16", x, x, c, c2, s, md), dict(cache_dt="f16"), ffi.UNSUPPORTED), (("f32", x, x, c, c2, s, md), {}, ffi.UNSUPPORTED),
            (("bf16", x, x, c, c2, s, md), dict(cache_dt="f8e4m3"), ffi.INVALID_ARG), (("bf16", x, x, c, c2, s, md), dict(k_scale=f, v_scale=f), ffi.INVALID_ARG),
            (("bf16", x, x, x, c2, s, md), {}, ffi.INVALID_ARG),
            (("bf16", x, x, c, c2, s, ffi.paged_store_md(4, 2, 64, 4, 16, k_offset=4)), {}, ffi.UNSUPPORTED),
            (("bf16", x, x, c, c2, s, ffi.paged_store_md(4, 2, 60, 4, 16)), {}, ffi.UNSUPPORTED),
            (("bf16", x, x, c, c2, s, ffi.paged_store_md(4, 2, 64, 4, 0)), {}, ffi.INVALID_ARG),
            (("bf16", x, x, c, c2, s, ffi.paged_store_md(4, 2, 64, 400, 16)), {}, ffi.INVALID_ARG),
            (("bf16", x, x, c, c2, s, md[:-1]), {}, ffi.INVALID_ARG)):
        with pytest.raises(ffi.HoduRocmError) as e:
            ctx.paged_store(*args, **kw)
        assert e.value.status == status, e.value
