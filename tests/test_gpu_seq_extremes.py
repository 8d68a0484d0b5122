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


def varlen(ctx, tile, dt, q, k, v, causal, scale=None):
    """(bits, values) of one sequence's outputs; q [n, Hq, D], k and v [m, Hk, D] float64, values of dt"""
    n, hq, d = q.shape
    m, hk, _ = k.shape
    operands = [ctx.upload(S.to_bits(x, dt)) for x in (q, k, v)]
    for x, buf in zip((q, k, v), operands):
        assert np.array_equal(S.widen(S.to_bits(x, dt), dt).reshape(x.shape), x, equal_nan=True)
    out = ctx.alloc(n * hq * d * 2)
    qo, ko = ctx.upload(np.array([0, n], np.int32)), ctx.upload(np.array([0, m], np.int32))
    ctx.force_tile(tile)
    try:
        ctx.attention_varlen(dt, *operands, out, qo, ko, ffi.varlen_md(1, n, m, hq, hk, d),
                             S.scalar(d, dt)[0] if scale is None else S.to_bits(np.array([scale]), dt), causal)
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


def check_exact_scores(got, q, k, v, dt, causal, what, scale=None):
    """For scores that are exact in f32 (one product, or a power of two and a small whole number), where what they are does not enter the
    bound, only what they differ by.  With u half a step of dt and e = 2^-24: P is rounded to dt, and once more where
    a reference moves before it is multiplied: 2 u a (a = sum of p |v|); a P whose exponent is below -64 is nothing,
    the argument of the others is off by three roundings of up to 64 e each, the exponential by 8 e, the same again in the
    row sum; sums over m keys (m + 8) e a; the rounded row sum and the result u |o| each; an f16 P below its normal
    range, and an f16 result, by 2^-25 as in seq_util.allowed."""
    n, hq, d = q.shape
    scale = S.scalar(d, dt)[1] if scale is None else scale
    o, a, _, inv = S.attend(q, k, v, scale, causal)
    u, e, m = S.HALF_STEP[dt], 2.0 ** -24, k.shape[0]
    tol = a * (2 * u + 2 * (8 * e + 3 * 64 * e) + (m + 8) * e) + 2 * np.abs(o) * u
    if dt == "f16":
        tol = tol + (m * 2.0 ** -25 * inv * np.abs(v).max())[..., None] + 2.0 ** -25
    off = np.abs(got - o)
    bad = ~(off <= tol * (1 + 2 * u))
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} wrong, first at {np.argwhere(bad)[0].tolist()}: got {got[tuple(np.argwhere(bad)[0])]}, " \
                          f"want {o[tuple(np.argwhere(bad)[0])]}"


def one_product(m, n, d, dt, q0, scores, seed):
    """q and k whose product is q0 * scores, one element of the head dim each (key by key; the same for all rows but every third,
    which is zero: an ordinary row among them), and values"""
    g = np.random.default_rng(seed)
    q, k = np.zeros((n, 1, d)), np.zeros((m, 1, d))
    q[:, 0, 5] = q0
    q[2::3] = 0
    k[:, 0, 5] = scores
    return q, rounded(k, dt), rounded(g.standard_normal((m, 1, d)), dt)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dt,d", [("bf16", 64), ("f16", 128)])
def test_scores_larger_than_their_differences_can_be(ctx, tile, dt, d):
    """scores so large that a step of f32 between them is a factor of more than 2^100: equal ones share the row, the larger one of two takes it"""
    n, m = 7, 150
    big, unit = (1e30, 1.0) if dt == "bf16" else (4.9e4, 5e4)
    for name, scores in (("equal", np.full(m, big)), ("equal, negative", np.full(m, -big)), ("all but the first", np.r_[0, np.full(m - 1, -big)]),
                         ("one in the middle", np.r_[np.full(m // 2, -big), big, np.full(m - m // 2 - 1, -big)]),
                         ("the last ones", np.r_[np.full(m - 3, big / 2), np.full(3, big)]), ("from negative to zero", np.r_[np.full(100, -big), np.zeros(m - 100)]),
                         ("falling", -big * np.arange(1, m + 1) / m), ("rising", big * np.arange(1, m + 1) / m), ("in pairs", big * (np.arange(m) // 2) / m),
                         ("ordinary, then large", np.r_[np.linspace(-1, 1, 70) / unit, np.full(m - 70, big)])):
        q, k, v = one_product(m, n, d, dt, unit, scores, len(name))
        q = rounded(q, dt)
        for causal in (False, True):
            _, got = varlen(ctx, tile, dt, q, k, v, causal)
            check_exact_scores(got, q, k, v, dt, causal, f"{name}, causal {causal}")
        _, got = paged(ctx, tile, dt, q, k, v, cut=400)
        check_exact_scores(got, q, k, v, dt, True, f"{name}, cached")


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_small_differences_of_large_scores(ctx, tile, dt):
    """scores of 2^24 to 2^28 that differ by a few steps of f32: exact, and so are their differences"""
    d, n, m = 64, 4, 200
    for size, step in ((13, 8.0), (14, 32.0), (12, 2.0), (-13, 8.0)):
        g = np.random.default_rng(abs(size))
        q, k = np.zeros((n, 1, d)), np.zeros((m, 1, d))
        q[:, 0, 0], q[:, 0, 1] = 2.0 ** abs(size), 1
        k[:, 0, 0] = np.sign(size) * 2.0 ** abs(size)
        k[:, 0, 1] = step * g.integers(0, 12, m)
        v = rounded(g.standard_normal((m, 1, d)), dt)
        for causal in (False, True):
            _, got = varlen(ctx, tile, dt, q, k, v, causal)
            check_exact_scores(got, q, k, v, dt, causal, f"2^{2 * abs(size)}")
        _, got = paged(ctx, tile, dt, q, k, v, cut=400)
        check_exact_scores(got, q, k, v, dt, True, f"2^{2 * abs(size)}, cached")


@pytest.mark.parametrize("tile", TILES)
def test_scores_beyond_f32_once_they_are_scaled(ctx, tile):
    for q0, scores, scale in ((1.0, np.full(90, -2.0 ** 127), 8.0), (1.0, np.r_[np.full(60, -2.0 ** 127), np.full(30, -2.0 ** 126)], 4.0), (1.0, np.full(90, 2.0 ** 127), 8.0),
                              (2.0 ** -100, np.full(90, 2.0 ** 10), 2.0 ** -130)):
        q, k, v = one_product(90, 7, 64, "bf16", q0, scores, 3)
        _, got = varlen(ctx, tile, "bf16", q, k, v, True, scale)
        check_exact_scores(got, q, k, v, "bf16", True, f"{scores[0]} scaled by {scale}", scale)


@pytest.mark.parametrize("tile", TILES)
def test_ranges_of_keys_with_scores_far_apart_are_added(ctx, tile):
    """keys cut across workgroups: each range's reference is of its own size"""
    for dt, big in (("bf16", 1e30), ("f16", 6e4)):
        m, d = 1500, 64
        for name, scores in (("the first range", np.r_[np.full(300, big), np.zeros(m - 300)]), ("the last range", np.r_[np.zeros(m - 10), np.full(10, big)]),
                             ("negative but for the middle", np.r_[np.full(700, -big), np.linspace(-1, 1, 100) / big, np.full(m - 800, -big)]),
                             ("all negative", np.full(m, -big)), ("rising", big * (np.arange(m) // 4) / m)):
            q, k, v = one_product(m, 9, d, dt, 1.0 if dt == "bf16" else 6e4, scores, 4)
            q = rounded(q, dt)
            _, got = paged(ctx, tile, dt, q, k, v, cut=100)
            check_exact_scores(got, q, k, v, dt, True, f"{dt}: {name}")


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_infinite_values_that_are_attended(ctx, tile, dt):
    """an infinity among a row's values is the row's result in its column, infinities of both signs or a NaN make it NaN, and the other
    columns are what they would be"""
    n, d = 9, 64
    for m, at in ((40, 0), (300, 0), (300, 37), (300, 299), (1500, 700)):
        g = np.random.default_rng(m + at)
        q, k = rounded(g.standard_normal((n, 2, d)), dt), rounded(g.standard_normal((m, 1, d)) * 0.3, dt)
        k[3::5] = k[2::5][:len(k[3::5])]  # (equal scores among them: probabilities that have no remainder, or the same one)
        v = rounded(g.standard_normal((m, 1, d)), dt)
        finite = v.copy()
        for col, word in ((1, np.inf), (6, -np.inf), (17, np.nan), (40, np.inf), (63, -np.inf)):
            v[at, 0, col], finite[at, 0, col] = word, 0.0
        v[(at + 1) % n, 0, 40], finite[(at + 1) % n, 0, 40] = -np.inf, 0.0
        if at < n:  # every row attends the key
            calls = [varlen(ctx, tile, dt, q, k, v, False)]
        else:
            calls = [varlen(ctx, tile, dt, q, k, v, False)] + ([paged(ctx, tile, dt, q, k, v, cut=100)] if at < m - n else [])
        others = [c for c in range(d) if c not in (1, 6, 17, 40, 63)]
        for _, got in calls:
            assert np.all(np.isposinf(got[:, :, 1])) and np.all(np.isneginf(got[:, :, 6])) and np.all(np.isneginf(got[:, :, 63]))
            assert np.all(np.isnan(got[:, :, 17])) and np.all(np.isnan(got[:, :, 40]))
            o, a, size, inv = S.attend(q, k, finite, S.scalar(d, dt)[1], False)
            if len(calls) > 1 and got is calls[1][1]:
                o, a, size, inv = S.attend(q, k, finite, S.scalar(d, dt)[1], True)
            S.assert_attention(got[:, :, others], (o[:, :, others], a[:, :, others], size, inv), dt, m, np.abs(finite).max(), d, f"{m} keys, one at {at}")
