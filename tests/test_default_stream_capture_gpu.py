"""A synchronous launch beside another party's stream capture."""
import ctypes as C

import pytest

import t0_gpu_b200 as t
from t0_gpu_b200._lib import lib

pytestmark = pytest.mark.gpu

RELAXED = 2      # CU_STREAM_CAPTURE_MODE_RELAXED


def test_a_capture_of_a_blocking_stream_survives_a_synchronous_launch():
    """While a blocking stream is captured the default stream may not be used at all: a launch that touched it would lose
    the capture."""
    import torch as th

    rt, L = t.GpuRuntime(), lib()
    x = th.randn(1000, device="cuda")
    y = th.zeros(1000, device="cuda", dtype=th.bfloat16)
    th.cuda.synchronize()

    def call():
        rt._check(L.t0b_cast_f32_to_bf16(rt.handle, x.data_ptr(), y.data_ptr(), x.numel(), 0))

    call()      # the kernel is loaded
    y.zero_()
    th.cuda.synchronize()
    cu = C.CDLL("libcuda.so.1")
    stream, graph, state = C.c_void_p(), C.c_void_p(), C.c_int(-1)
    assert cu.cuStreamCreate(C.byref(stream), 0) == 0          # CU_STREAM_DEFAULT: a blocking stream
    assert cu.cuStreamBeginCapture_v2(stream, RELAXED) == 0
    call()
    call()
    assert cu.cuStreamIsCapturing(stream, C.byref(state)) == 0 and state.value == 1
    assert cu.cuStreamEndCapture(stream, C.byref(graph)) == 0
    assert cu.cuGraphDestroy(graph) == 0 and cu.cuStreamDestroy_v2(stream) == 0
    assert th.equal(y, x.bfloat16())
    rt.close()


def test_the_order_can_be_switched_off(monkeypatch):
    """T0B_DEFAULT_STREAM_ORDER=0: a synchronous launch returns while the default stream is busy."""
    import torch as th

    monkeypatch.setenv("T0B_DEFAULT_STREAM_ORDER", "0")
    rt, L = t.GpuRuntime(), lib()
    x = th.randn(1000, device="cuda")
    y = th.zeros(1000, device="cuda", dtype=th.bfloat16)
    a, out = th.ones((8192, 8192), device="cuda", dtype=th.bfloat16), th.empty((8192, 8192), device="cuda", dtype=th.bfloat16)
    done = th.cuda.Event()

    def call():
        rt._check(L.t0b_cast_f32_to_bf16(rt.handle, x.data_ptr(), y.data_ptr(), x.numel(), 0))

    th.mm(a, a, out=out)
    th.cuda.synchronize()
    call()      # the kernel is loaded
    for _ in range(100):
        th.mm(a, a, out=out)
    done.record()
    call()
    assert not done.query()      # about 80 ms of products were queued
    th.cuda.synchronize()
    assert th.equal(y, x.bfloat16())
    rt.close()
