"""What the operators around the paged cache do with numbers at the ends of their ranges: page numbers that are none, sizes next to
2^31."""
import numpy as np
import pytest

from hodu_amd import ffi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = ffi.Context(0)
    yield c
    c.close()


def test_a_page_whose_slots_are_beyond_32_bits_gives_no_slot(ctx):
    """(page * page_size wrapped around would be the slot of somebody else's token)"""
    page, width = 16, 4
    cached, added = np.array([5, 0, 20, 3], np.int32), np.array([3, 20, 2, 4], np.int32)
    table = np.array([[1 << 28, 0, 0, 0], [0] * 4, [7, -1, 0, 0], [-(1 << 28), 0, 0, 0]], np.int32)
    free = np.array([(1 << 27) - 1, 2 ** 31 - 1, 9], np.int32)
    want_table = table.copy()
    want_table[1, :2] = free[:2]
    last = (1 << 27) - 1
    want = [-1] * 3 + [last * page + i for i in range(16)] + [-1] * 4 + [-1] * 2 + [-1] * 4
    assert want[18] == 2 ** 31 - 1
    capacity = len(want) + 3
    dev = [ctx.upload(x) for x in (cached, added, free, table, np.zeros(4, np.int32), np.zeros(5, np.int32), np.zeros(capacity, np.int32), np.zeros(2, np.int32))]
    ctx.paged_plan(*dev, ffi.paged_plan_md(4, page, width, len(free), capacity))
    assert ctx.download(dev[6], np.int32).tolist() == want + [-1] * 3
    assert np.array_equal(ctx.download(dev[3], np.int32).reshape(4, width), want_table)
    assert ctx.download(dev[4], np.int32).tolist() == [8, 20, 22, 7] and ctx.download(dev[7], np.int32).tolist() == [2, 0]
