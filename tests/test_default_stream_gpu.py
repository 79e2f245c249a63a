"""A synchronous launch on the runtime's own stream starts behind the work of the device's default stream."""
import pytest

import t0_gpu_b200 as t
from t0_gpu_b200._lib import lib

pytestmark = pytest.mark.gpu


def busy(th):
    """About 30 ms of work on the default stream, all of it queued at once."""
    a, out = th.ones((8192, 8192), device="cuda", dtype=th.bfloat16), th.empty((8192, 8192), device="cuda", dtype=th.bfloat16)
    th.mm(a, a, out=out)
    th.cuda.synchronize()
    for _ in range(40):
        th.mm(a, a, out=out)


def test_synchronous_gemm_waits_for_the_default_stream():
    import torch as th

    rt, L = t.GpuRuntime(), lib()
    m, n, k = 256, 512, 128
    a0 = th.randint(-4, 5, (m, k), device="cuda").bfloat16()
    b0 = th.randint(-4, 5, (k, n), device="cuda").bfloat16()
    a, b, c = th.zeros_like(a0), th.zeros_like(b0), th.zeros((m, n), device="cuda")

    def call():
        rt._check(L.t0b_gemm(rt.handle, None, 0, 0, a.data_ptr(), b.data_ptr(), c.data_ptr(), m, n, k, k, n, n, 0, 0, 0, 1.0, 0, 0, 0))

    call()      # the kernel is loaded
    busy(th)
    a.copy_(a0)
    b.copy_(b0)
    call()
    assert th.equal(c, a0.float() @ b0.float())      # whole numbers below 2^24: exact
    rt.close()


def test_synchronous_row_kernel_waits_for_the_default_stream():
    import torch as th

    rt, L = t.GpuRuntime(), lib()
    x0 = th.randn(100_000, device="cuda")
    x, y = th.zeros_like(x0), th.zeros(100_000, device="cuda", dtype=th.bfloat16)

    def call():
        rt._check(L.t0b_cast_f32_to_bf16(rt.handle, x.data_ptr(), y.data_ptr(), x0.numel(), 0))

    call()
    busy(th)
    x.copy_(x0)
    call()
    assert th.equal(y, x0.bfloat16())
    rt.close()
