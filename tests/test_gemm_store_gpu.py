"""bf16 stores of tiles whose last chunks lie behind column N, many short tiles after one another."""
import pytest

import t0_gpu_b200 as t
from t0_gpu_b200 import OUT_BF16, GemmConfig

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("preset", ["b200_128x64", "b200_128x128", "b200_128x256", "b200_256x128", "b200_256x256", "b200_512x256", "b200_256x512"])
@pytest.mark.parametrize("m,n", [(76416, 208), (20000, 3784), (30000, 40), (30000, 104)])
def test_short_tiles_with_an_odd_number_of_chunks(preset, m, n):
    import torch as th

    rt, k = t.GpuRuntime(), 64
    g = th.Generator(device="cuda")
    g.manual_seed(m + n)
    a = th.randint(-2, 3, (m, k), device="cuda", generator=g).bfloat16()
    b = th.randint(-2, 3, (k, n), device="cuda", generator=g).bfloat16()
    want = (a.float() @ b.float()).bfloat16()       # whole numbers up to 256: exact in f32 and in bf16
    s = th.cuda.Stream()
    s.wait_stream(th.cuda.current_stream())
    rt.set_stream(s.cuda_stream)
    with th.cuda.stream(s):
        for _ in range(10):
            c = th.zeros((m, n), device="cuda", dtype=th.bfloat16)
            rt.gemm(a.data_ptr(), b.data_ptr(), c.data_ptr(), m, n, k, cfg=GemmConfig.preset(preset), trans_b=False, out_dtype=OUT_BF16)
            rt.synchronize()
            assert th.equal(c, want)
    rt.close()
