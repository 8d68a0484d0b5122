"""Tiles of 16 rows multiply what P's rounding left too: their outputs are held to what that owes, which is less than
seq_util.allowed grants the other tiles."""
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


def allowed16(dt, o, a, size, inv, m, vmax, d):
    """As seq_util.allowed (u half a step of dt, e = 2^-24), but for P and the row sum: P is two numbers of dt, the second one what
    the first one's rounding left, so it is off by u^2 of itself: u^2 a in the product and u^2 |o| in the row sum.  In f16 the
    second is below the normal range for most, off by 2^-25 of the largest P as before.  The result is rounded once."""
    u, e = S.HALF_STEP[dt], 2.0 ** -24
    rel = u * u + 2 * ((d + 2) * e * size + 8 * e + 2 * size * e) + (m + 8) * e
    tol = a * rel[..., None] + np.abs(o) * (u + u * u)
    if dt == "f16":
        tol = tol + (m * 2.0 ** -25 * inv * vmax)[..., None] + 2.0 ** -25
    return tol * (1 + 2 * u) + 1e-30


SIZES = [(64, 1, 40), (128, 1, 75), (64, 3, 130), (128, 2, 700), (128, 1, 2500)]  # head dim, rows, keys


def operands(dt, d, n, m, seed):
    g = np.random.default_rng(seed)
    return [S.Side(g.standard_normal(s), dt) for s in ((n, 4, d), (m, 2, d), (m, 2, d))]


def outside(got, q, k, v, dt, d, scale):
    o, a, size, inv = S.attend(q, k, v, scale, True)
    tol = allowed16(dt, o, a, size, inv, k.shape[0], np.abs(v).max(), d)
    return int((~(np.abs(got - o) <= tol)).sum())


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("size", range(len(SIZES)))
def test_single_tokens_and_short_chunks(ctx, dt, size):
    d, n, m = SIZES[size]
    q, k, v = operands(dt, d, n, m, size)
    bits, scale = S.scalar(d, dt)
    out, qo, ko = ctx.alloc(n * 4 * d * 2), ctx.upload(np.array([0, n], np.int32)), ctx.upload(np.array([0, m], np.int32))
    ctx.attention_varlen(dt, ctx.upload(q.flat), ctx.upload(k.flat), ctx.upload(v.flat), out, qo, ko, ffi.varlen_md(1, n, m, 4, 2, d), bits, True)
    assert "r16" in ctx.last_kernel()
    got = S.widen(ctx.download(out, np.uint16), dt).reshape(n, 4, d)
    assert outside(got, q.values, k.values, v.values, dt, d, scale) == 0
    # the same keys in pages, cut across workgroups where there are many
    page = 16
    pages = -(-m // page)
    caches = []
    for x in (k, v):
        c = np.zeros((pages * page, 2, d), np.uint16)
        c[:m] = S.to_bits(x.values, dt).reshape(m, 2, d)
        caches.append(ctx.upload(c))
    ctx.attention_paged(dt, ctx.upload(q.flat), *caches, out, qo, ctx.upload(np.arange(pages, dtype=np.int32)), ctx.upload(np.array([m], np.int32)),
                        ffi.paged_attention_md(1, n, 4, 2, d, pages, page, pages), bits)
    assert "r16" in ctx.last_kernel()
    got = S.widen(ctx.download(out, np.uint16), dt).reshape(n, 4, d)
    assert outside(got, q.values, k.values, v.values, dt, d, scale) == 0
