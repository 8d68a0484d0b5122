"""Attention over packed sequences and over the paged cache against the definition in float64 (tests/seq_util.py, which
derives the bound), and a serving loop's run of all four operators together."""
import numpy as np
import pytest

from hodu_amd import ffi
import seq_util as S

pytestmark = pytest.mark.gpu

HEADS = [(1, 1), (4, 2), (5, 1), (8, 1), (6, 6), (34, 2)]  # (query heads, key / value heads)


TILES = [50, 51, 52]  # the kernels for tiles of 16, 128 and 192 or 256 rows


@pytest.fixture(scope="module")
def ctx():
    c = ffi.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_prompts(ctx, dt, d, causal):
    for n, (hq, hk) in enumerate(HEADS):
        lens = [[1], [1, 1, 1], [5, 0, 33, 64], [31, 32, 33], [63, 2, 65], [0, 0, 7, 0]][n]
        S.run_varlen(ctx, dt, lens, lens, hq, hk, d, causal, seed=n, shared_offsets=True)


@pytest.mark.parametrize("dt,d", [("bf16", 128), ("f16", 64)])
def test_longer_prompts(ctx, dt, d):
    S.run_varlen(ctx, dt, [300, 129, 257], [300, 129, 257], 4, 2, d, True, seed=30)
    S.run_varlen(ctx, dt, [200, 70], [200, 70], 2, 2, d, False, seed=31)
    S.run_varlen(ctx, dt, [513], [513], 2, 1, d, True, seed=32)


@pytest.mark.parametrize("dt,d", [("bf16", 64), ("f16", 128)])
def test_rows_and_keys_of_different_lengths(ctx, dt, d):
    for causal in (True, False):
        S.run_varlen(ctx, dt, [3, 10, 1, 40], [50, 10, 33, 7], 4, 2, d, causal, seed=40)  # the last: rows that attend nothing
        S.run_varlen(ctx, dt, [4, 3, 2], [0, 9, 0], 4, 4, d, causal, seed=41)              # sequences without keys
        S.run_varlen(ctx, dt, [0, 3], [20, 9], 2, 1, d, causal, seed=42)
        S.run_varlen(ctx, dt, [9], [200], 8, 1, d, causal, seed=43)
        S.run_varlen(ctx, dt, [150], [40], 2, 1, d, causal, seed=44)


def test_prompt_layouts(ctx):
    for n, kw in enumerate((dict(q_order=(1, 0)), dict(k_order=(1, 0)), dict(q_order=(1, 0), k_order=(1, 0), gap=8, offset=24), dict(gap=64, offset=8))):
        S.run_varlen(ctx, "bf16", [37, 12], [37, 12], 4, 2, 64, True, seed=50 + n, **kw)
        S.run_varlen(ctx, "f16", [37, 140], [37, 140], 4, 2, 128, True, seed=60 + n, **kw)
    S.run_varlen(ctx, "bf16", [20, 3], [20, 3], 4, 2, 64, True, seed=70, spare=9)  # rows behind the last sequence


def test_scores_that_grow_along_the_keys(ctx):
    """maxima that move at every step, in both directions, and scores far apart"""
    def ramp(sign):
        def edit(q, k, v):
            q[...] = np.abs(q)
            k[...] = 0.3 * k + sign * np.linspace(0, 4, k.shape[0])[:, None, None]
        return edit
    for n, sign in enumerate((1, -1)):
        for dt in ("bf16", "f16"):
            S.run_varlen(ctx, dt, [300], [300], 2, 1, 64, False, seed=80 + n, edit=ramp(sign))
            S.run_varlen(ctx, dt, [290], [290], 2, 1, 128, True, seed=82 + n, edit=ramp(sign))
    S.run_varlen(ctx, "bf16", [100], [100], 2, 2, 128, True, seed=84, qscale=30.0)


@pytest.mark.parametrize("dt,cache_dt", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8e4m3"), ("f16", "f8e4m3")])
@pytest.mark.parametrize("d", [64, 128])
def test_single_tokens_over_the_cache(ctx, dt, cache_dt, d):
    for n, page in enumerate((1, 3, 16, 24, 64, 128)):
        hq, hk = HEADS[n]
        S.run_paged(ctx, dt, [1, 1, 1, 1], [1, page, 2 * page + 1, 77], hq, hk, d, page, cache_dt, seed=100 + n)
    S.run_paged(ctx, dt, [1], [700], 8, 2, d, 16, cache_dt, seed=110)
    S.run_paged(ctx, dt, [1, 0, 1], [33, 40, 0], 4, 2, d, 16, cache_dt, seed=111)  # a request without new tokens, one without keys


@pytest.mark.parametrize("dt,cache_dt", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8e4m3"), ("f16", "f8e4m3")])
@pytest.mark.parametrize("d", [64, 128])
def test_chunks_over_the_cache(ctx, dt, cache_dt, d):
    for n, page in enumerate((1, 3, 16, 24, 64, 128)):
        hq, hk = HEADS[n]
        S.run_paged(ctx, dt, [5, 1, 17, 40], [5, 90, 64, 103], hq, hk, d, page, cache_dt, seed=120 + n)
    S.run_paged(ctx, dt, [130, 1, 1], [390, 300, 5], 4, 1, d, 16, cache_dt, seed=130)
    S.run_paged(ctx, dt, [12, 3], [7, 3], 4, 2, d, 16, cache_dt, seed=131)  # more new tokens than tokens: rows that attend nothing


@pytest.mark.parametrize("cache_dt,garbage", [("bf16", 0x7FC0), ("bf16", 0x7F80), ("f8e4m3", 0x7F)])
def test_what_unused_slots_hold_does_not_matter(ctx, cache_dt, garbage):
    """NaN and infinities in every slot that no request's tokens are in: behind the last token of a page, in free pages"""
    for d in (64, 128):
        S.run_paged(ctx, "bf16", [1, 3, 1], [17, 50, 95], 4, 2, d, 16, cache_dt, seed=140, garbage=garbage)
        S.run_paged(ctx, "bf16", [40, 20], [141, 20], 4, 2, d, 64, cache_dt, seed=141, garbage=garbage)
        S.run_paged(ctx, "bf16", [200], [333], 4, 2, d, 24, cache_dt, seed=142, garbage=garbage)


def test_cache_layouts(ctx):
    for n, kw in enumerate((dict(order=(0, 2, 1)), dict(order=(2, 0, 1), gap=16, offset=32), dict(gap=64, offset=16), dict(q_order=(1, 0), spare=5))):
        for cache_dt in ("bf16", "f8e4m3"):
            S.run_paged(ctx, "bf16", [1, 20, 1], [90, 61, 33], 4, 2, 128, 16, cache_dt, seed=150 + n, **kw)
            S.run_paged(ctx, "bf16", [150, 2], [170, 61], 4, 2, 64, 24, cache_dt, seed=160 + n, **kw)


def seq_buffers(ctx, dt="bf16", tokens=8, hq=4, hk=2, d=64, pages=4, page=16, batch=2, width=4):
    q, kc, vc = ctx.alloc(tokens * hq * d * 2), ctx.alloc(pages * page * hk * d * 2), ctx.alloc(pages * page * hk * d * 2)
    for b in (q, kc, vc):
        ctx.fill(b, 0)
    return q, kc, vc, ctx.alloc(tokens * hq * d * 2)


def test_pages_and_offsets_that_make_no_sense_stay_in_bounds(ctx):
    """(results are unspecified: the call returns, and reads and writes nothing outside its operands, which the CPU build's
    guard pages hold it to)"""
    q, kc, vc, out = seq_buffers(ctx)
    bits, _ = S.scalar(64, "bf16")
    md = ffi.paged_attention_md(2, 8, 4, 2, 64, 4, 16, 4)
    for table in ([[-5, 10 ** 9, 2 ** 31 - 1, -2 ** 31], [0, 4, 5, 6]], [[0, 1, 2, 3], [-1, -1, -1, -1]]):
        for offsets in ([0, 1, 2], [0, 4, 8], [-7, 3, 100], [8, 2, 5], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], [5, 5, 5]):
            for lens in ([64, 20], [10 ** 9, -3], [2 ** 31 - 1, 2 ** 31 - 1], [0, 0]):
                ctx.attention_paged("bf16", q, kc, vc, out, ctx.upload(np.array(offsets, np.int32)), ctx.upload(np.array(table, np.int32)),
                                    ctx.upload(np.array(lens, np.int32)), md, bits)
    ctx.sync()
    vmd = ffi.varlen_md(2, 8, 8, 4, 2, 64)
    for a in ([0, 4, 8], [-7, 3, 100], [8, 2, 5], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1]):
        for b in ([0, 4, 8], [-7, 3, 100], [9, 9, 9], [-2 ** 31, 2 ** 31 - 1, -4]):
            for causal in (False, True):
                ctx.attention_varlen("bf16", q, kc, vc, out, ctx.upload(np.array(a, np.int32)), ctx.upload(np.array(b, np.int32)), vmd, bits, causal)
    ctx.sync()


def test_refusals(ctx):
    q, kc, vc, out = seq_buffers(ctx)
    f = ctx.upload(np.ones(8, np.float32))
    off, table, lens = ctx.upload(np.array([0, 1, 2], np.int32)), ctx.upload(np.zeros((2, 4), np.int32)), ctx.upload(np.array([3, 4], np.int32))
    bits, _ = S.scalar(64, "bf16")
    neg, inf = S.to_bits(np.array([-0.125]), "bf16"), np.array([0x7F80], np.uint16)
    vmd, pmd = ffi.varlen_md(2, 8, 8, 4, 2, 64), ffi.paged_attention_md(2, 8, 4, 2, 64, 4, 16, 4)

    def varlen(md=vmd, dt="bf16", scale=bits, o=out):
        ctx.attention_varlen(dt, q, kc, vc, o, off, off, md, scale)

    def paged(md=pmd, dt="bf16", scale=bits, o=out, **kw):
        ctx.attention_paged(dt, q, kc, vc, o, off, table, lens, md, scale, **kw)

    varlen()
    paged()
    for call, kw, status in (
            (varlen, dict(md=ffi.varlen_md(2, 8, 8, 4, 3, 64)), ffi.INVALID_ARG), (varlen, dict(md=ffi.varlen_md(2, 8, 8, 4, 0, 64)), ffi.INVALID_ARG),
            (varlen, dict(md=ffi.varlen_md(2, 8, 8, 4, 2, 32)), ffi.UNSUPPORTED), (varlen, dict(md=ffi.varlen_md(2, 7, 8, 4, 2, 64, q_offset=4)), ffi.UNSUPPORTED),
            (varlen, dict(md=ffi.varlen_md(2, 4, 8, 4, 2, 64, q_strides=(260, 64))), ffi.UNSUPPORTED), (varlen, dict(md=vmd[:-1]), ffi.INVALID_ARG),
            (varlen, dict(dt="f32"), ffi.INVALID_ARG), (varlen, dict(scale=neg), ffi.UNSUPPORTED), (varlen, dict(scale=inf), ffi.UNSUPPORTED),
            (varlen, dict(o=q), ffi.INVALID_ARG), (varlen, dict(md=ffi.varlen_md(2, 9, 8, 4, 2, 64)), ffi.INVALID_ARG),
            (varlen, dict(md=ffi.varlen_md(3, 8, 8, 4, 2, 64)), ffi.INVALID_ARG),
            (paged, dict(md=ffi.paged_attention_md(2, 8, 4, 2, 96, 2, 16, 4)), ffi.INVALID_ARG), (paged, dict(md=ffi.paged_attention_md(2, 8, 4, 2, 64, 5, 16, 4)), ffi.INVALID_ARG),
            (paged, dict(md=ffi.paged_attention_md(2, 4, 4, 2, 96, 2, 16, 4)), ffi.UNSUPPORTED), (paged, dict(md=ffi.paged_attention_md(2, 8, 4, 2, 64, 4, 0, 4)), ffi.INVALID_ARG),
            (paged, dict(md=ffi.paged_attention_md(2, 8, 4, 2, 64, 4, 16, 5)), ffi.INVALID_ARG), (paged, dict(cache_dt="f8e4m3"), ffi.INVALID_ARG),
            (paged, dict(cache_dt="f16"), ffi.UNSUPPORTED), (paged, dict(k_scale=f, v_scale=f), ffi.INVALID_ARG),
            (paged, dict(cache_dt="f8e4m3", k_scale=f, v_scale=f, md=ffi.paged_attention_md(2, 8, 4, 2, 64, 4, 16, 4, k_cache_offset=8)), ffi.UNSUPPORTED)):
        with pytest.raises(ffi.HoduRocmError) as e:
            call(**kw)
        assert e.value.status == status, (kw, e.value)
    ctx.attention_varlen("bf16", q, kc, vc, out, off, off, ffi.varlen_md(0, 8, 8, 4, 2, 64), bits)  # nothing to do
    ctx.attention_varlen("bf16", q, kc, vc, out, off, off, ffi.varlen_md(2, 0, 8, 4, 2, 64), bits)
    ctx.attention_varlen("bf16", q, kc, vc, out, off, off, ffi.varlen_md(2, 8, 0, 4, 2, 64), bits)
    ctx.attention_paged("bf16", q, kc, vc, out, off, table, lens, ffi.paged_attention_md(2, 8, 4, 2, 64, 0, 16, 4), bits)
    ctx.sync()
    assert not ctx.download(out, np.uint16)[:2 * 4 * 64].any()  # no page, no key: zeros


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dt,cache_dt", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f8e4m3"), ("f16", "f8e4m3")])
@pytest.mark.parametrize("d", [64, 128])
def test_every_tile(ctx, tile, dt, cache_dt, d):
    """each kernel on what the choice would not hand it: few rows, many short sequences, ragged ends of every stage"""
    ctx.force_tile(tile)
    try:
        for n, (new, lens, hq, hk, page) in enumerate([([1, 1, 3], [1, 30, 70], 4, 2, 16), ([1, 9], [200, 129], 7, 1, 3), ([70, 2], [290, 64], 2, 2, 24),
                                                       ([66], [391], 5, 1, 1), ([5, 0, 2], [3, 0, 257], 2, 1, 64)]):
            S.run_paged(ctx, dt, new, lens, hq, hk, d, page, cache_dt, seed=200 + n)
        S.run_paged(ctx, dt, [40, 3], [333, 95], 4, 2, d, 16, cache_dt, seed=210, garbage=0x7F if cache_dt == "f8e4m3" else 0x7F80)
        if cache_dt == dt:
            for causal in (True, False):
                for n, (lens, hq, hk) in enumerate([([1, 2], 4, 2), ([65, 31, 100], 3, 1), ([0, 193, 1], 2, 2), ([330], 2, 1)]):
                    S.run_varlen(ctx, dt, lens, lens, hq, hk, d, causal, seed=220 + n)
                S.run_varlen(ctx, dt, [3, 40, 70], [260, 7, 65], 4, 2, d, causal, seed=230)

            def ramp(q, k, v):
                q[...] = np.abs(q)
                k[...] = 0.3 * k + np.linspace(-3, 3, k.shape[0])[:, None, None]
            S.run_varlen(ctx, dt, [420], [420], 2, 1, d, True, seed=231, edit=ramp)
            S.run_varlen(ctx, dt, [3], [420], 2, 1, d, False, seed=232, edit=ramp)
    finally:
        ctx.force_tile(-1)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("cache_dt", ["bf16", "f8e4m3"])
def test_tables_longer_than_what_a_workgroup_holds_of_them(ctx, tile, cache_dt):
    """pages of one and of three tokens: the windows of table entries in LDS are filled again and again"""
    ctx.force_tile(tile)
    try:
        S.run_paged(ctx, "bf16", [9, 1], [2500, 1300], 2, 1, 64, 1, cache_dt, seed=240)
        S.run_paged(ctx, "bf16", [3], [7000], 1, 1, 128, 3, cache_dt, seed=241)
    finally:
        ctx.force_tile(-1)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dt,cache_dt,d", [("bf16", "bf16", 128), ("f16", "f16", 64), ("bf16", "f8e4m3", 64), ("f16", "f8e4m3", 128)])
def test_keys_cut_across_workgroups(ctx, tile, dt, cache_dt, d):
    """few tiles over long caches: a sequence that is cut often, one that is not, one whose first rows attend nothing of the last range"""
    ctx.force_tile(tile)
    try:
        for _ in range(2):  # (the second finds the counters as the first left them)
            S.run_paged(ctx, dt, [20, 0, 7, 1], [2900, 600, 1100, 40], 4, 1, d, 16, cache_dt, seed=260)
        S.run_paged(ctx, dt, [520], [1300], 1, 1, d, 64, cache_dt, seed=261, garbage=0x7F if cache_dt == "f8e4m3" else 0x7F80)
        S.run_paged(ctx, dt, [30, 3], [1100, 1500], 2, 2, d, 3, cache_dt, seed=262)
    finally:
        ctx.force_tile(-1)


def test_pages_further_apart_than_32_bits(ctx):
    """a page stride that the wide kernels' offsets do not hold: the rows go to the other kernel"""
    q, kc, vc, out, off, table, lens = (ctx.alloc(n) for n in (40 * 4 * 64 * 2, 48 * 2 * 64 * 2, 48 * 2 * 64 * 2, 40 * 4 * 64 * 2, 8, 4, 4))
    for b in (q, kc, vc):
        ctx.upload_into(b, np.full(b.nbytes // 2, 0x3F80, np.uint16))
    ctx.upload_into(off, np.array([0, 40], np.int32))
    ctx.upload_into(table, np.array([0], np.int32))
    ctx.upload_into(lens, np.array([48], np.int32))
    for page, kernel in ((1 << 31, "r16"), (48 * 2 * 64, "wide")):
        ctx.fill(out, 0xFF)
        ctx.attention_paged("bf16", q, kc, vc, out, off, table, lens, ffi.paged_attention_md(1, 40, 4, 2, 64, 1, 48, 1, k_cache_strides=(page, 128, 64), v_cache_strides=(page, 128, 64)),
                            S.scalar(64, "bf16")[0])
        assert kernel in ctx.last_kernel()
        assert np.all(ctx.download(out, np.uint16) == 0x3F80)  # the mean of ones


def test_many_sequences(ctx):
    """more than a workgroup looks at in one step of its search"""
    g = np.random.default_rng(3)
    for n in (255, 256, 257, 600):
        lens = (g.integers(0, 3, n) * g.integers(0, 2, n)).tolist()
        lens[-1] = 2
        S.run_varlen(ctx, "bf16", lens, lens, 2, 1, 64, True, seed=250, expect="r16")
        S.run_paged(ctx, "f16", [min(1, x) for x in lens], [x + 3 for x in lens], 2, 2, 64, 4, seed=251)


def test_calls_in_a_row_give_the_same_bits(ctx):
    a = S.run_paged(ctx, "bf16", [1, 1, 30], [400, 77, 130], 8, 2, 128, 16, seed=170)
    S.run_paged(ctx, "bf16", [60], [160], 4, 1, 64, 16, seed=171)
    assert np.array_equal(a, S.run_paged(ctx, "bf16", [1, 1, 30], [400, 77, 130], 8, 2, 128, 16, seed=170))


@pytest.mark.parametrize("cache_dt", ["bf16", "f8e4m3"])
def test_a_serving_loop(ctx, cache_dt):
    """prompts admitted, a chunk and single tokens added, step by step: lengths in, plan -> store -> attention, nothing read
    back in between; every step's outputs against attention over all of the requests' tokens so far as the cache holds them"""
    dt, hq, hk, d, page, width, pool = "bf16", 8, 2, 64, 16, 12, 40
    g = np.random.default_rng(7)
    b = 3
    bits, scale = S.scalar(d, dt)
    kc, vc = ctx.alloc(pool * page * hk * d * 2), ctx.alloc(pool * page * hk * d * 2)
    ctx.fill(kc, 0xFF)  # every slot a NaN until something is stored there
    ctx.fill(vc, 0xFF)
    ks, vs = np.array([0.02, 0.03], np.float32), np.array([0.04, 0.025], np.float32)
    f8 = cache_dt == "f8e4m3"
    scales = dict(k_scale=ctx.upload(ks), v_scale=ctx.upload(vs)) if f8 else {}
    table, lens = ctx.upload(np.full((b, width), -1, np.int32)), ctx.upload(np.zeros(b, np.int32))
    free, all_k, all_v = g.permutation(pool).astype(np.int32), [np.zeros((0, hk, d))] * b, [np.zeros((0, hk, d))] * b
    for added in ([37, 16, 0], [1, 1, 70], [1, 20, 1], [1, 1, 1], [1, 0, 1]):
        t, spare = sum(added), 3
        rows = S.Side(g.standard_normal((t + spare, hq + 2 * hk, d)), dt)
        drows = ctx.upload(rows.flat)
        offsets, slots, used, new_lens = ctx.alloc(4 * b + 4), ctx.alloc(4 * (t + spare)), ctx.alloc(8), ctx.alloc(4 * b)
        out = ctx.upload(np.full((t + spare) * hq * d, S.POISON, np.uint16))
        ctx.paged_plan(lens, ctx.upload(np.array(added, np.int32)), ctx.upload(free), table, new_lens, offsets, slots, used,
                       ffi.paged_plan_md(b, page, width, len(free), t + spare))
        lens = new_lens
        row = (hq + 2 * hk) * d
        ctx.paged_store(dt, drows, drows, kc, vc, slots, ffi.paged_store_md(t + spare, hk, d, pool, page, (row, d), (row, d), k_offset=hq * d, v_offset=(hq + hk) * d),
                        cache_dt=cache_dt, **scales)
        ctx.attention_paged(dt, drows, kc, vc, out, offsets, table, lens, ffi.paged_attention_md(b, t + spare, hq, hk, d, pool, page, width, q_strides=(row, d)),
                            bits, cache_dt=cache_dt, **scales)
        got = S.widen(ctx.download(out, np.uint16), dt).reshape(t + spare, hq, d)
        taken, refused = ctx.download(used, np.int32)
        assert refused == 0
        free, at = free[taken:], 0
        for r, n in enumerate(added):
            x = rows.values[at:at + n]
            k, v = x[:, hq:hq + hk], x[:, hq + hk:]
            if f8:
                k = S.widen(S.to_bits(k.astype(np.float32) / ks[:, None], "f8e4m3"), "f8e4m3").reshape(k.shape) * ks.astype(np.float64)[:, None]
                v = S.widen(S.to_bits(v.astype(np.float32) / vs[:, None], "f8e4m3"), "f8e4m3").reshape(v.shape) * vs.astype(np.float64)[:, None]
            all_k[r], all_v[r] = np.concatenate([all_k[r], k]), np.concatenate([all_v[r], v])
            S.assert_attention(got[at:at + n], S.attend(x[:, :hq], all_k[r], all_v[r], scale, True), dt, len(all_k[r]),
                               np.abs(all_v[r]).max() if len(all_v[r]) else 0.0, d, f"request {r}")
            at += n
        assert np.all(ctx.download(out, np.uint16).reshape(t + spare, hq, d)[t:] == S.POISON)
