"""Vocabulary losses on every tile of their products, with several tiles to a CTA: sizes as in use choose the large tiles, which
small sizes never reach.  The gradients' tiles are forced by preset; the head's follow from the sizes on a GPU of 148 SMs."""
import math

import pytest

import t0_gpu_b200 as t
from t0_gpu_b200 import OUT_BF16, OUT_F32, GemmConfig, ops
from test_vocab_losses_gpu import art, check_linear, th  # noqa: F401

pytestmark = pytest.mark.gpu

PRESETS = ["b200_128x64", "b200_128x128", "b200_128x256", "b200_256x128", "b200_256x256", "b200_512x256", "b200_256x512"]


@pytest.fixture(scope="module", params=PRESETS)
def forced(request, th):  # noqa: F811
    """A runtime whose gradient products run on one preset."""
    with pytest.MonkeyPatch.context() as m:
        m.setenv("T0_FORCE_CONFIG", request.param)
        r = t.GpuRuntime()
    s = th.cuda.Stream()
    with th.cuda.stream(s):
        r.set_stream(s.cuda_stream)
        yield r
        r.synchronize()
    r.close()


@pytest.mark.parametrize("gdt", [OUT_F32, OUT_BF16])
@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("vocab", [20000, 20001])
def test_gradient_tiles(th, forced, vocab, trans_w, gdt):  # noqa: F811
    """Rows counted on the device (a third is left out), in one piece and in pieces that add up; stores by TMA and off 16 bytes."""
    check_linear(th, forced, 600, 1100, vocab, trans_w, gdt=gdt)
    check_linear(th, forced, 600, 1100, vocab, trans_w, gdt=gdt, piece_rows=256, topk=5, temperature=2.0)
    check_linear(th, forced, 200, 1100, vocab, trans_w, gdt=gdt)


# Sums of an odd and an even number of 512-product pieces; up to thirteen tiles to a CTA or a pair of them.
@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("rows,dim,vocab", [
    (600, 2100, 16000), (520, 1600, 24000), (300, 4096, 8192), (130, 640, 40000), (900, 640, 5000),     # pairs of CTAs, 256 x 256
    (300, 1100, 20001), (64, 600, 40000), (16, 1024, 50257),                                            # 128 x 256
    (900, 64, 5000), (1000, 200, 30000), (1000, 1100, 4688), (1000, 1600, 4624), (100, 64, 50257),      # 128 x 128
])
def test_head_tiles(th, art, rows, dim, vocab, trans_w):  # noqa: F811
    check_linear(th, art, rows, dim, vocab, trans_w, gdt=OUT_F32)
    check_linear(th, art, rows, dim, vocab, trans_w, grads=False, ignore=rows > 256)


@pytest.mark.parametrize("keep", [list(range(520)), [3, 511, 900], []])
def test_large_tiles_with_few_rows_left(th, art, keep):  # noqa: F811
    """The launches are sized for 1000 rows, the products run over what has a target."""
    for trans_w in (False, True):
        check_linear(th, art, 1000, 1100, 13001, trans_w, keep=keep, ignore=False)
        check_linear(th, art, 1000, 1100, 13001, trans_w, keep=keep, ignore=False, piece_rows=512, gdt=OUT_F32)


@pytest.mark.parametrize("rows,vocab", [(200, 2000), (300, 8192)])
def test_logits_of_a_long_contraction_are_summed_in_pieces(th, art, rows, vocab):  # noqa: F811
    """The tensor core truncates its running sum at every step of 16 products, by a share of the sum so far.  Over 4096 positive
    products the sum grows evenly, and the steps' sums add up to (256 + 1) / 2 of the last; in eight pieces of 512 that start
    anew it is (32 + 1) / 2 of it, 0.128 times as much, and the pieces are added with rounding.  So log-sum-exp has 0.128 times
    the bias that it has from the logits of a plain product; twice that is allowed."""
    dim = 4096
    g = th.Generator(device="cuda")
    g.manual_seed(vocab)
    x = th.randn((rows, dim), device="cuda", generator=g).abs().bfloat16()
    w = (th.randn((vocab, dim), device="cuda", generator=g).abs() / 40).bfloat16()       # logits of about 65
    tgt = th.randint(0, vocab, (rows,), device="cuda", generator=g).to(th.int32)
    z, losses, lse = th.empty((rows, vocab), device="cuda"), th.empty(rows, device="cuda"), th.empty(rows, device="cuda")
    art.gemm(x.data_ptr(), w.data_ptr(), z.data_ptr(), rows, vocab, dim, cfg=GemmConfig.preset("b200_128x128"), async_=True)
    ops.linear_cross_entropy(art, x.data_ptr(), w.data_ptr(), tgt.data_ptr(), rows, dim, vocab, trans_w=True, x_dtype=OUT_BF16, w_dtype=OUT_BF16,
                             grads=False, losses=losses.data_ptr(), lse=lse.data_ptr())
    art.synchronize()
    want = th.logsumexp(x.double() @ w.double().t(), 1)
    plain = (th.logsumexp(z.double(), 1) - want).mean().item()
    pieces = (lse.double() - want).mean().item()
    assert plain < 0 and abs(pieces) <= 2 * 0.128 * abs(plain), (pieces, plain)
    assert math.isfinite(losses.sum().item())
