"""Which sequence a tile belongs to, for more than 64 sequences: sequences of several tiles between short and empty ones, in
every part of the search (four sequences a lane, 256 at a step), under each tile height."""
import numpy as np
import pytest

from hodu_amd import ffi
import seq_util as S

pytestmark = pytest.mark.gpu

KERNELS = {50: "r16", 51: "wide128", 52: "wide"}


@pytest.fixture(scope="module")
def ctx():
    c = ffi.Context(0)
    yield c
    c.close()


def lengths(batch, long_ones, seed):
    g = np.random.default_rng(seed)
    lens = (g.integers(0, 4, batch) * g.integers(0, 2, batch)).tolist()
    for at, n in long_ones.items():
        lens[at % batch] = n
    return lens


CASES = [(66, {0: 150, 5: 290, 6: 17, 65: 131}), (130, {1: 260, 63: 33, 64: 200, 127: 16, 129: 65}), (300, {2: 130, 255: 257, 256: 300, 259: 129, 299: 40}),
         (600, {254: 64, 257: 385, 511: 16, 513: 260, 599: 193})]


@pytest.mark.parametrize("tile", sorted(KERNELS))
@pytest.mark.parametrize("case", range(len(CASES)))
def test_long_sequences_among_many(ctx, tile, case):
    batch, long_ones = CASES[case]
    ctx.force_tile(tile)
    try:
        lens = lengths(batch, long_ones, case)
        S.run_varlen(ctx, "bf16", lens, lens, 2, 1, 64, True, seed=300 + case)
        assert KERNELS[tile] in ctx.last_kernel() and ("wide128" in ctx.last_kernel()) == (tile == 51)
        # chunks behind what is cached: other lengths of the keys than of the rows, some requests without new tokens
        S.run_paged(ctx, "f16", [min(n, 40) if n > 200 else n for n in lens], [n + 5 * (i % 3) for i, n in enumerate(lens)], 3, 1, 64, 16, seed=310 + case)
        assert KERNELS[tile] in ctx.last_kernel() and ("wide128" in ctx.last_kernel()) == (tile == 51)
    finally:
        ctx.force_tile(-1)


@pytest.mark.parametrize("batch", [64, 65])
def test_both_searches_give_the_same(ctx, batch):
    """64 sequences are searched longest first, 65 in their order: the same sequences give the same bits"""
    lens = lengths(64, {0: 100, 31: 1, 32: 0, 40: 213, 63: 77}, 7)
    raw = S.run_varlen(ctx, "bf16", lens + [0] * (batch - 64), lens + [0] * (batch - 64), 4, 2, 128, True, seed=320)
    ctx.force_tile(52)
    try:
        a = S.run_varlen(ctx, "bf16", lens, lens, 4, 2, 128, True, seed=320)
        b = S.run_varlen(ctx, "bf16", lens + [0] * (batch - 64), lens + [0] * (batch - 64), 4, 2, 128, True, seed=320)
    finally:
        ctx.force_tile(-1)
    assert np.array_equal(a, b) and raw.shape == a.shape
