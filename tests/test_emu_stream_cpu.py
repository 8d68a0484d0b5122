"""The stream that a context's calls are issued on, in the CPU build (tests/emu_util.EmuContext): handed over and back, what a
new stream waits for, and the hand-overs that are refused."""
import ctypes

import numpy as np
import pytest

import emu_util
from hodu_amd import ffi

pytestmark = pytest.mark.skipif(emu_util.compiler() is None, reason="no host clang++ for the CPU build")


@pytest.fixture()
def ctx():
    c = emu_util.EmuContext()
    yield c
    c.close()


def last_wait(ctx):
    a, b = ctypes.c_void_p(), ctypes.c_void_p()
    ctx.lib.emu_last_wait(ctypes.byref(a), ctypes.byref(b))
    return a.value or 0, b.value or 0


def test_a_stream_is_handed_over_and_back(ctx):
    class Theirs:
        cuda_stream = 0x1230

    own = ctx.stream
    assert own != 0
    ctx.set_stream(Theirs())
    assert ctx.stream == 0x1230 and last_wait(ctx) == (0x1230, own)  # behind what was issued on the stream before
    ctx.set_stream(0)  # the default stream
    assert ctx.stream == 0 and last_wait(ctx) == (0, 0x1230)
    ctx.set_stream(own)
    assert ctx.stream == own and last_wait(ctx) == (own, 0)
    assert ctx.lib.hodu_rocm_ctx_set_stream(ctx.handle, own) == ffi.OK
    assert last_wait(ctx) == (own, 0)  # the same one again: nothing to wait for
    b = ctx.upload(np.arange(4, dtype=np.int32))
    assert ctx.download(b, np.int32).tolist() == [0, 1, 2, 3]


def test_a_context_that_holds_a_callers_stream_closes():
    c = emu_util.EmuContext()
    c.set_stream(0x4560)
    c.close()


def test_no_hand_over_during_a_capture(ctx):
    own = ctx.stream

    def calls():
        with pytest.raises(ffi.HoduRocmError) as e:
            ctx.set_stream(0x1230)
        assert e.value.status == ffi.INVALID_ARG and "captured" in str(e.value)
        ctx.set_stream(own)  # (the one it has)
    ctx.record(calls).free()
    assert ctx.stream == own
    ctx.set_stream(0x1230)
    assert ctx.stream == 0x1230


def test_null_arguments():
    lib = ffi.load()
    assert lib.hodu_rocm_ctx_set_stream(None, None) == ffi.INVALID_ARG
    assert lib.hodu_rocm_ctx_stream(None, None) == ffi.INVALID_ARG
