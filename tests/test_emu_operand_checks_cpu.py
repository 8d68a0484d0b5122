"""What the Python binding refuses before a call reaches the library (CPU build of the kernels, tests/emu_util.EmuContext): a scale
that is not in the operands' storage, operands on another device than the context's."""
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
    c.close()


def attentions(ctx, view=lambda b: b):
    """{name: call(scale)} of the attention entry points on small operands; view: wraps the first operand"""
    d, n = 64, 4
    q, k, v, out = (ctx.upload(np.zeros(n * d, np.uint16)) for _ in range(4))
    off, table, lens = ctx.upload(np.array([0, n], np.int32)), ctx.upload(np.zeros((1, 1), np.int32)), ctx.upload(np.array([n], np.int32))
    dense = (1, 1, n, n, d, n * d, d, 1, n * d, d, 1, n * d, d, 1, 0, 0, 0)
    return {"attention": lambda scale: ctx.attention("bf16", view(q), k, v, out, dense, scale),
            "attention_varlen": lambda scale: ctx.attention_varlen("bf16", view(q), k, v, out, off, off, ffi.varlen_md(1, n, n, 1, 1, d), scale),
            "attention_paged": lambda scale: ctx.attention_paged("bf16", view(q), k, v, out, off, table, lens, ffi.paged_attention_md(1, n, 1, 1, d, 1, n, 1), scale)}


@pytest.mark.parametrize("name", ["attention", "attention_varlen", "attention_paged"])
def test_a_scale_of_another_storage_is_refused(ctx, name):
    call = attentions(ctx)[name]
    call(S.scalar(64, "bf16")[0])
    for scale in (0.125, np.float32(0.125), np.array([0.125]), np.zeros(1, np.uint8), np.zeros(2, np.uint16)):
        with pytest.raises((ffi.HoduRocmError, ValueError)):
            call(scale)


class Tensor:
    """what DeviceView.of reads of a torch tensor"""

    def __init__(self, buf, index):
        self.nbytes, self.buf, self.index = buf.nbytes, buf, index

    def get_device(self):
        return self.index

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return self.buf.ptr


@pytest.mark.parametrize("name", ["attention_varlen", "attention_paged"])
def test_an_operand_of_another_device_is_refused(ctx, name):
    bits = S.scalar(64, "bf16")[0]
    attentions(ctx, lambda b: ffi.DeviceView.of(Tensor(b, 0)))[name](bits)
    attentions(ctx, lambda b: ffi.DeviceView(b.ptr, b.nbytes))[name](bits)  # (memory of an unnamed device is the caller's word)
    with pytest.raises(ffi.HoduRocmError) as e:
        attentions(ctx, lambda b: ffi.DeviceView.of(Tensor(b, 1)))[name](bits)
    assert e.value.status == ffi.INVALID_ARG and "device 1" in str(e.value)


def test_plan_and_store_refuse_it_too(ctx):
    b = [ctx.alloc(4096) for _ in range(8)]
    other = ffi.DeviceView.of(Tensor(b[2], 3))
    for call in (lambda: ctx.paged_plan(b[0], b[1], other, b[3], b[4], b[5], b[6], b[7], ffi.paged_plan_md(1, 16, 1, 1, 1)),
                 lambda: ctx.paged_store("bf16", b[0], b[1], b[3], b[4], other, ffi.paged_store_md(1, 1, 64, 1, 16))):
        with pytest.raises(ffi.HoduRocmError) as e:
            call()
        assert e.value.status == ffi.INVALID_ARG and "device 3" in str(e.value)
