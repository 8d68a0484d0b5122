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


def test_sizes_next_to_the_end_of_32_bits_are_refused(ctx):
    """(calls of no sequence, which do nothing where the sizes are taken)"""
    b, bits = ctx.alloc(4096), np.array([0x3E00], np.uint16)
    out = ctx.alloc(4096)

    def words(md):
        return (ffi.ctypes.c_size_t * len(md))(*md), len(md)

    def varlen(q_tokens, k_tokens, heads=1, batch=0):
        md, n = words(ffi.varlen_md(batch, q_tokens, k_tokens, heads, 1, 64))
        return ctx.lib.hodu_rocm_attention_varlen(ctx.handle, ffi.DTYPE_ID["bf16"], b.ptr, b.ptr, b.ptr, out.ptr, b.ptr, b.ptr, md, n, bits.ctypes.data, 1)

    def paged(q_tokens, page, width, heads=1):
        md, n = words(ffi.paged_attention_md(0, q_tokens, heads, 1, 64, 1, page, width))
        t = ffi.DTYPE_ID["bf16"]
        return ctx.lib.hodu_rocm_attention_paged(ctx.handle, t, t, b.ptr, b.ptr, b.ptr, out.ptr, b.ptr, b.ptr, b.ptr, None, None, md, n, bits.ctypes.data)

    most = 2 ** 31 - 4096
    assert varlen(1, most) == ffi.OK and varlen(most, 1) == ffi.OK and varlen(most // 8, 1, 8) == ffi.OK
    assert paged(1, 4096, most // 4096) == ffi.OK and paged(most // 8, 16, 4, 8) == ffi.OK
    for call in (lambda: varlen(1, most + 1), lambda: varlen(most + 1, 1), lambda: varlen(most // 8 + 1, 1, 8), lambda: paged(1, 4096, most // 4096 + 1),
                 lambda: paged(1, 1, 2 ** 31 - 1), lambda: paged(most // 8 + 1, 16, 4, 8)):
        assert call() == ffi.UNSUPPORTED
