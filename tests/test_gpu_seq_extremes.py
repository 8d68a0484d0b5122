"""Attention over packed sequences and over the cache where values or scores are far from ordinary: values up to the largest that
sums over the keys leave finite, scores far apart, and results that are known without a sum.  The wanted outputs come from
the definition in float64 (tests/seq_util.attend)."""
import numpy as np
import pytest

from hodu_amd import ffi
import seq_util as S

pytestmark = pytest.mark.gpu

TILES = [50, 51, 52]  # the kernels for tiles of 16, 128 and 192 or 256 rows


@pytest.fixture(scope="module")
def ctx():
    c = ffi.Context(0)
    yield c
    c.close()


def varlen(ctx, tile, dt, q, k, v, causal):
    """(bits, values) of one sequence's outputs; q [n, Hq, D], k and v [m, Hk, D] float64, values of dt"""
    n, hq, d = q.shape
    m, hk, _ = k.shape
    operands = [ctx.upload(S.to_bits(x, dt)) for x in (q, k, v)]
    for x, buf in zip((q, k, v), operands):
        assert np.array_equal(S.widen(S.to_bits(x, dt), dt).reshape(x.shape), x)
    out = ctx.alloc(n * hq * d * 2)
    qo, ko = ctx.upload(np.array([0, n], np.int32)), ctx.upload(np.array([0, m], np.int32))
    ctx.force_tile(tile)
    try:
        ctx.attention_varlen(dt, *operands, out, qo, ko, ffi.varlen_md(1, n, m, hq, hk, d), S.scalar(d, dt)[0], causal)
    finally:
        ctx.force_tile(-1)
    bits = ctx.download(out, np.uint16).reshape(n, hq, d)
    return bits, S.widen(bits, dt).reshape(n, hq, d)


def paged(ctx, tile, dt, q, k, v, page=16, cut=None):
    """the same over a cache, its pages in reverse; the q rows are the last of the keys' tokens.  cut: table columns beyond the
    keys, which let the launcher cut the keys into ranges"""
    n, hq, d = q.shape
    m, hk, _ = k.shape
    pages = -(-m // page)
    width = pages + (cut or 0)
    caches = []
    for x in (k, v):
        flat = np.full((pages * page, hk, d), np.nan)
        flat[:m] = x
        caches.append(ctx.upload(S.to_bits(flat.reshape(pages, page, hk, d)[::-1], dt)))
    table = np.full((1, width), -1, np.int32)
    table[0, :pages] = np.arange(pages)[::-1]
    out = ctx.alloc(n * hq * d * 2)
    ctx.force_tile(tile)
    try:
        ctx.attention_paged(dt, ctx.upload(S.to_bits(q, dt)), *caches, out, ctx.upload(np.array([0, n], np.int32)), ctx.upload(table),
                            ctx.upload(np.array([m], np.int32)), ffi.paged_attention_md(1, n, hq, hk, d, pages, page, width), S.scalar(d, dt)[0])
    finally:
        ctx.force_tile(-1)
    bits = ctx.download(out, np.uint16).reshape(n, hq, d)
    return bits, S.widen(bits, dt).reshape(n, hq, d)


def rounded(x, dt):
    return S.widen(S.to_bits(x, dt), dt).reshape(np.shape(x))


def check(got, q, k, v, dt, causal, what, d):
    scale = S.scalar(d, dt)[1]
    parts = S.attend(q, k, v, scale, causal)
    S.assert_attention(got, parts, dt, k.shape[0], np.abs(v).max(), d, what)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("d", [64, 128])
def test_large_values_behind_scores_that_grow(ctx, tile, d):
    """bf16 reaches to 2^127, and so do the values: keys whose scores rise by 2^60 and more behind the first ones must not take the
    sums beyond f32.  (|v| up to 2^118: 400 of them sum to less than 2^127)"""
    for m, grown, size in ((128, 100, 2.0 ** 73), (100, 40, 2.0 ** 90), (400, 350, 2.0 ** 90), (400, 64, 2.0 ** 118), (130, 129, -2.0 ** 118)):
        g = np.random.default_rng(m)
        q, k = np.ones((3, 2, d)), np.zeros((m, 1, d))
        # 40 nats (58 powers of two) above the first ones, some 43 for head dim 128
        k[grown:] = 5.0 if d == 64 else 3.75
        v = rounded(g.uniform(0.5, 1.0, (m, 1, d)) * size, "bf16")
        for causal in (False, True):
            _, got = varlen(ctx, tile, "bf16", q, k, v, causal)
            assert np.isfinite(got).all()
            check(got, q, k, v, "bf16", causal, f"{m} keys", d)
        _, got = paged(ctx, tile, "bf16", q, k, v, cut=200)
        check(got, q, k, v, "bf16", True, f"{m} cached keys", d)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_scores_that_rise_step_by_step(ctx, tile, dt):
    """the reference moves again and again, by less and by more than its slack, in stages whose keys are all open and in masked ones"""
    d = 64
    for step in (0.05, 0.4, 2.0):
        g = np.random.default_rng(int(step * 100))
        m = 330
        q = rounded(np.ones((m, 1, d)) * 0.5, dt)
        k = rounded(np.repeat((np.arange(m) // 8 * step)[:, None, None], d, 2) + g.standard_normal((m, 1, d)) * 0.1, dt)
        v = rounded(g.standard_normal((m, 1, d)) * (1e3 if dt == "f16" else 2.0 ** 60), dt)
        for causal in (True, False):
            _, got = varlen(ctx, tile, dt, q, k, v, causal)
            check(got, q, k, v, dt, causal, f"steps of {step}", d)
