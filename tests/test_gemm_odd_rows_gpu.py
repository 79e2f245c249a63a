"""Products whose rows start off 16-byte boundaries: every tile, type, split and destination offset, exact in whole numbers, and
no slower than their aligned neighbours by more than their stores."""
import pytest

import t0_gpu_b200 as t
from t0_gpu_b200 import OUT_BF16, OUT_F32, GemmConfig

pytestmark = pytest.mark.gpu

PRESETS = ["b200_128x64", "b200_128x128", "b200_128x256", "b200_256x128", "b200_256x256", "b200_512x256", "b200_256x512"]


@pytest.fixture(scope="module")
def th():
    import torch

    return torch


@pytest.fixture(scope="module")
def art(th):
    r = t.GpuRuntime()
    s = th.cuda.Stream()
    with th.cuda.stream(s):
        r.set_stream(s.cuda_stream)
        yield r
        r.synchronize()
    r.close()


@pytest.mark.parametrize("preset", PRESETS)
@pytest.mark.parametrize("out_dtype", [OUT_F32, OUT_BF16])
def test_any_pitch_and_offset(th, art, preset, out_dtype):
    dt = th.float32 if out_dtype == OUT_F32 else th.bfloat16
    g = th.Generator(device="cuda")
    g.manual_seed(len(preset) + out_dtype)
    for m, n, k, pad, offset, split in [(1, 1, 8, 0, 0, 0), (33, 1001, 512, 0, 0, 0), (700, 33, 64, 1, 0, 0), (129, 95, 200, 3, 1, 0), (300, 513, 96, 0, 5, 0),
                                        (64, 257, 1024, 2, 3, 4), (257, 31, 2048, 0, 7, 2), (600, 1030, 64, 1, 2, 0)]:
        a = th.randint(-2, 3, (m, k), device="cuda", generator=g).bfloat16()
        b = th.randint(-2, 3, (n, k), device="cuda", generator=g).bfloat16()
        bias = th.randint(-2, 3, (n,), device="cuda", generator=g).float()
        product = a.float() @ b.float().t()                 # whole numbers: exact in f32, and rounded once to bf16
        ldc = n + pad
        for epilogue, want in ((0, product), (3, product.relu()), (2, (product + bias).relu())):     # none, ReLU, bias and ReLU
            out = th.full((m * ldc + offset + 40,), 7.0, device="cuda", dtype=dt)
            c = out[offset:offset + m * ldc].view(m, ldc)
            cfg = GemmConfig.preset(preset)
            cfg.split_k = split
            art.gemm(a.data_ptr(), b.data_ptr(), c.data_ptr(), m, n, k, cfg=cfg, ldc=ldc, out_dtype=out_dtype, epilogue=epilogue,
                     bias=bias.data_ptr() if epilogue == 2 else None, async_=True)
            art.synchronize()
            assert th.equal(c[:, :n], want.to(dt)), (m, n, k, pad, offset, split, epilogue)
            c[:, :n] = 7
            assert (out == 7).all()


def test_an_odd_row_length_costs_its_stores_alone(th, art):
    """33 x 1001 beside 33 x 1000, f32: 7.3 and 6.6 us; it was 10.2 and 6.9 with rows shifted together in 16-byte pieces."""
    m, k = 33, 512
    a = th.randn((m, k), device="cuda").bfloat16()
    took = {1000: [], 1001: []}
    bufs = {n: (th.randn((n, k), device="cuda").bfloat16(), th.empty((m, n), device="cuda")) for n in took}
    for _ in range(15):
        for n, (b, c) in bufs.items():
            start, end = th.cuda.Event(enable_timing=True), th.cuda.Event(enable_timing=True)
            start.record()
            for _ in range(100):
                art.gemm(a.data_ptr(), b.data_ptr(), c.data_ptr(), m, n, k, async_=True)
            end.record()
            end.synchronize()
            took[n].append(start.elapsed_time(end))
    assert sorted(took[1001])[7] < 1.3 * sorted(took[1000])[7]
