"""Vocabulary losses where their contract ends: rows that the logits leave without a distribution.  Bounds as in
test_vocab_losses_gpu.py."""
import math

import pytest

from t0_gpu_b200 import OUT_BF16, OUT_F32, T0Error, ops
from test_vocab_losses_gpu import U32, UB, UH, art, check_logits, losses_and_dz, make_teacher, target_rows, th  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("rows,vocab,topk,x_dtype,piece_rows", [
    (40, 300, 0, OUT_BF16, 0),         # x is copied for the head's gradient only, rows joined with their gradient
    (256, 50000, 0, OUT_BF16, 0),      # the same, joined by a kernel of its own
    (40, 300, 0, OUT_F32, 0),          # x is copied first
    (40, 300, 3, OUT_F32, 0),          # ... together with the teacher's words
    (40, 300, 3, OUT_BF16, 0),
    (300, 300, 0, OUT_BF16, 0),        # rows with a target gathered
    (300, 300, 3, OUT_F32, 0),
    (300, 300, 0, OUT_BF16, 128),      # in pieces
    (100, 300, 0, OUT_BF16, 33),
])
def test_a_row_without_finite_logits_reaches_no_gradient(th, art, rows, vocab, topk, x_dtype, piece_rows, trans_w):  # noqa: F811
    """An infinity in the hidden state and a column of the head with one sign: every logit is -inf, and the row is left out of
    the gradients (0 * inf would be NaN in the head's)."""
    dim = 64
    g = th.Generator(device="cuda")
    g.manual_seed(rows + vocab + topk)
    w = (th.randn((vocab, dim), device="cuda", generator=g) / 8).bfloat16()
    w[:, 0] = -0.25 - w[:, 0].abs()
    x = (th.randn((rows, dim), device="cuda", generator=g) * 2).bfloat16()
    dead = th.zeros(rows, device="cuda", dtype=th.bool)
    dead[::5] = True
    dead[-1] = True
    xd = x.double().masked_fill(dead[:, None], 0.0)
    x[dead, 0] = math.inf
    x = x if x_dtype == OUT_BF16 else x.float()
    if topk:
        ids, teacher = make_teacher(th, rows, topk, vocab, 5, False)
        q, ent, live = target_rows(th, ids, teacher, 1.0, vocab)
    else:
        tgt = th.randint(0, vocab, (rows,), device="cuda", generator=g)
        tgt[1::7] = -1
        live = tgt >= 0
        q = th.zeros((rows, vocab), dtype=th.float64, device="cuda")
        q[th.arange(rows, device="cuda"), tgt.clamp_min(0)] = live.double()
        ent = th.zeros(rows, dtype=th.float64, device="cuda")
        tgt = tgt.to(th.int32)
    live = live & ~dead
    wd = w.double()
    z = xd @ wd.t()
    scale = th.full((rows,), 1.0 / rows, device="cuda", dtype=th.float64)
    losses_ref, dz, p, lse_ref = losses_and_dz(th, z, q, ent, live, 1.0, scale)
    head = w if trans_w else w.t().contiguous()
    losses, lse = th.full((rows,), 7.0, device="cuda"), th.full((rows,), 7.0, device="cuda")
    dx, dw = th.full((rows, dim), 7.0, device="cuda"), th.full(head.shape, 7.0, device="cuda")
    kw = dict(trans_w=trans_w, x_dtype=x_dtype, w_dtype=OUT_BF16, losses=losses.data_ptr(), lse=lse.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(),
              piece_rows=piece_rows)
    if topk:
        ops.linear_topk_distill(art, x.data_ptr(), head.data_ptr(), ids.data_ptr(), teacher.data_ptr(), rows, dim, vocab, topk, **kw)
    else:
        ops.linear_cross_entropy(art, x.data_ptr(), head.data_ptr(), tgt.data_ptr(), rows, dim, vocab, **kw)
    art.synchronize()
    xa, wa = xd.abs(), wd.abs()
    ez = dim * U32 * (xa @ wa.t()).amax(1)
    down = z.amax(1, keepdim=True) - z
    tol = 2 * ez + ((down * (q > 0)).amax(1) + 16 + lse_ref.abs()) * 8 * U32
    assert ((losses.double() - losses_ref).abs() <= tol).all()
    assert (losses[~live] == 0).all() and (lse[~live] == 0).all() and (dx[~live] == 0).all()
    a = (live / rows)[:, None]
    edz = UB * dz.abs() + a * (p * (2 * ez[:, None] + down * 4 * U32 + 8 * U32 + UH + UB * UH) + 2.0 ** -24 * p.amax(1, keepdim=True))
    full = dz.abs() + edz
    for got, want, err in ((dx, dz @ wd, edz @ wa + vocab * U32 * (full @ wa)),
                           (dw if trans_w else dw.t(), dz.t() @ xd, edz.t() @ xa + rows * U32 * (full.t() @ xa))):
        assert ((got.double() - want).abs() <= err + U32 * (want.abs() + err) + 1e-30).all()


@pytest.mark.parametrize("trans_w", [False, True])
def test_an_empty_call_checks_the_gradient_it_clears(th, art, trans_w):  # noqa: F811
    """No rows: the head's gradient becomes zeros, in a buffer that holds it or not at all."""
    dim, vocab = 64, 80
    w = th.ones((dim * vocab,), device="cuda").bfloat16()
    small, whole = art.alloc_zero(4096), art.alloc_zero(dim * vocab * 4)
    kw = dict(trans_w=trans_w, x_dtype=OUT_BF16, w_dtype=OUT_BF16, losses=w.data_ptr(), x_needs=False)
    with pytest.raises(T0Error, match="dw needs"):
        ops.linear_cross_entropy(art, w.data_ptr(), w.data_ptr(), w.data_ptr(), 0, dim, vocab, dw=small, **kw)
    for lddw in (None, (dim if trans_w else vocab) + 8):
        rows = (vocab if trans_w else dim)
        out = th.full((rows, lddw or (dim if trans_w else vocab)), 7.0, device="cuda")
        ops.linear_cross_entropy(art, w.data_ptr(), w.data_ptr(), w.data_ptr(), 0, dim, vocab, dw=out.data_ptr(), lddw=lddw, **kw)
        art.synchronize()
        cols = dim if trans_w else vocab
        assert (out[:, :cols] == 0).all() and (out[:, cols:] == 7).all()
    ops.linear_cross_entropy(art, w.data_ptr(), w.data_ptr(), w.data_ptr(), 0, dim, vocab, dw=whole, **kw)
    art.synchronize()
    assert not art.is_poisoned()


def test_an_empty_call_with_rows_two_gib_apart(th, art):  # noqa: F811
    pitch = 2 ** 29 + 8
    out = th.full((2 * pitch,), 7.0, device="cuda")
    w = th.ones((64,), device="cuda").bfloat16()
    ops.linear_cross_entropy(art, w.data_ptr(), w.data_ptr(), w.data_ptr(), 0, 2, 20, x_dtype=OUT_BF16, w_dtype=OUT_BF16, losses=w.data_ptr(),
                             x_needs=False, dw=out.data_ptr(), lddw=pitch)
    art.synchronize()
    rows = out.view(2, pitch)
    assert (rows[:, :20] == 0).all() and (rows[:, 20:] == 7).all()


@pytest.mark.parametrize("pitch", [2 ** 61, 2 ** 62 - 3, 2 ** 63, 2 ** 64 - 8, 2 ** 46])
def test_pitches_that_leave_the_address_space_are_refused(th, art, pitch):  # noqa: F811
    """(rows - 1) * pitch * element size may come out small in 64 bits; no row would be where that says."""
    rows, dim, vocab, topk = 5, 64, 80, 2
    x, w = art.alloc_zero(rows * vocab * 4), art.alloc_zero(dim * vocab * 4)
    z, out = art.alloc_zero(rows * vocab * 4), art.alloc_zero(dim * vocab * 4)
    ids = art.alloc_zero(rows * vocab * 4)

    def refused(f, *a, **kw):
        with pytest.raises(T0Error, match="pitch of"):
            f(art, *a, **kw)
        assert not art.is_poisoned()

    refused(ops.topk_distill, z, ids, z, rows, vocab, topk, ld=pitch, losses=out, dlogits=x)
    refused(ops.topk_distill, z, ids, z, rows, vocab, topk, ldk=pitch, losses=out, dlogits=x)
    kw = dict(x_dtype=OUT_BF16, w_dtype=OUT_BF16, losses=out, dx=x, dw=w)
    for name in ("ldx", "ldw", "lddx", "lddw"):
        refused(ops.linear_cross_entropy, x, w, ids, rows, dim, vocab, **{name: pitch}, **kw)
    refused(ops.linear_topk_distill, x, w, ids, z, rows, dim, vocab, topk, ldk=pitch, **kw)
    refused(ops.linear_cross_entropy, x, w, ids, 0, dim, vocab, lddw=pitch, **kw)
    art.synchronize()


@pytest.mark.parametrize("rows,dim,vocab,piece_rows", [(2 ** 32 - 1, 64, 1000, 0), (2 ** 32 - 1, 64, 1000, 2 ** 31), (2 ** 31, 8, 8, 256), (16, 2 ** 30, 2 ** 30, 0),
                                                       (16, 64, 2 ** 32 - 1, 0)])
def test_no_scratch_for_sizes_that_no_call_takes(th, art, rows, dim, vocab, piece_rows):  # noqa: F811
    assert ops.linear_loss_scratch_bytes(art, rows, dim, vocab, piece_rows=piece_rows) == 0
    assert ops.linear_loss_scratch_bytes(art, 16, 64, 1000, topk=1025) == 0


@pytest.mark.parametrize("rows,cols,topk,stride", [(2000, 16000, 31, 512), (64, 131000, 256, 512), (1000, 16000, 120, 128)])
def test_words_a_power_of_two_apart_cost_what_others_cost(th, art, rows, cols, topk, stride):  # noqa: F811
    """Finding words named twice takes the same time whatever the ids (ids with the same low bits once took 2.6 to 6 times as long)."""
    g = th.Generator(device="cuda")
    g.manual_seed(rows + topk)
    z = th.randn((rows, cols), device="cuda", generator=g)
    dz, losses = th.empty_like(z), th.empty(rows, device="cuda")
    teacher = th.randn((rows, topk), device="cuda", generator=g)
    spread = th.stack([th.randperm(cols, device="cuda", generator=g)[:topk] for _ in range(rows)]).to(th.int32)
    apart = (th.arange(topk, device="cuda") * stride % cols).to(th.int32).repeat(rows, 1)
    assert apart[0].unique().numel() == topk

    def run(ids):
        ops.topk_distill(art, z.data_ptr(), ids.data_ptr(), teacher.data_ptr(), rows, cols, topk, losses=losses.data_ptr(), dlogits=dz.data_ptr())

    took = {}
    for _ in range(21):
        for name, ids in (("spread", spread), ("apart", apart)):
            a, b = th.cuda.Event(enable_timing=True), th.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(4):
                run(ids)
            b.record()
            b.synchronize()
            took.setdefault(name, []).append(a.elapsed_time(b))
    assert sorted(took["apart"])[10] < 1.6 * sorted(took["spread"])[10]


# Rows in one CTA's registers, in those of a cluster, in CTAs of 128 threads, streamed, and off 16-byte boundaries.
FORMS = [(12, 500, 0), (12, 32000, 0), (700, 700, 0), (150, 40000, 0), (12, 500, 1)]


@pytest.mark.parametrize("dtype", [OUT_F32, OUT_BF16])
@pytest.mark.parametrize("temperature", [1.0, 1.5])
@pytest.mark.parametrize("rows,cols,offset", FORMS)
def test_logits_of_any_size(th, art, rows, cols, offset, temperature, dtype):  # noqa: F811
    """Rows masked as a whole with -1e9, -1e30 and the like, whose words are then equally likely; rows whose largest logits are
    large themselves; masks of that size beside ordinary logits."""
    def edit(z):
        for r, v in enumerate((-1e4, -1e9, -1e20, -1e30, -1e37, 1e7, 1e9, 1e30)):
            z[r] = v
        z[8, 1:] = -1e30
        z[9, ::2] = -1e9
        z[10, :cols // 2] = -3e8
        z[10, cols // 2:] = -3e8 - 2 ** 23
        z[11] = 3e6
        z[11, 7] = 3e6 + 2 ** 14

    check_logits(th, art, rows, cols, 5, dtype=dtype, temperature=temperature, ragged=False, edit=edit, offset=offset)


@pytest.mark.parametrize("rows,cols,offset", FORMS)
def test_slices_whose_maxima_differ_little_and_are_large(th, art, rows, cols, offset):  # noqa: F811
    """Maxima of a row's slices around 2^21, 2^22 and 2^23 over log2(e), a few apart."""
    def edit(z):
        for r, v in enumerate((2 ** 21, 2 ** 22, 2 ** 23, -2 ** 21, -2 ** 22, -2 ** 23)):
            z[r] = v * math.log(2) + th.randint(-3, 4, (cols,), device="cuda")
            z[r, ::100] += th.arange(len(z[r, ::100]), device="cuda") % 5

    check_logits(th, art, rows, cols, 5, ragged=False, edit=edit, offset=offset)


@pytest.mark.parametrize("rows,cols,offset", FORMS)
def test_gradients_of_unlikely_words(th, art, rows, cols, offset):  # noqa: F811
    """One word takes almost all of the probability; the others' gradients, 2^-25 to 2^-37 of its, stay.  bf16 in and out: the
    exponentials may have gone through fp16, 2^15 times what they are relative to the largest: 2^-11 of themselves or 2^-40 of the
    largest off, then rounded to bf16."""
    g = th.Generator(device="cuda")
    g.manual_seed(cols)
    buf = th.empty(rows * cols + offset, device="cuda", dtype=th.bfloat16)
    z = buf[offset:].view(rows, cols)
    z.copy_(th.randn((rows, cols), device="cuda", generator=g) - 18)
    z[:, 5] = 4
    ids = th.tensor([[5, 9]], device="cuda", dtype=th.int32).repeat(rows, 1)
    teacher = th.zeros((rows, 2), device="cuda")
    losses, out = th.empty(rows, device="cuda"), th.empty_like(buf)
    dz = out[offset:].view(rows, cols)
    ops.topk_distill(art, z.data_ptr(), ids.data_ptr(), teacher.data_ptr(), rows, cols, 2, logits_dtype=OUT_BF16, grad_dtype=OUT_BF16, scale=1.0,
                     losses=losses.data_ptr(), dlogits=dz.data_ptr())
    art.synchronize()
    zd = z.double()
    p = th.softmax(zd, 1)
    down = zd.amax(1, keepdim=True) - zd
    others = th.ones(cols, device="cuda", dtype=th.bool)
    others[[5, 9]] = False
    bound = UB * p + (1 + UB) * (p * (UH + (down * 4 + 16) * 2 * U32) + 2.0 ** -40 * p.amax(1, keepdim=True))
    assert ((dz.double() - p).abs() <= bound)[:, others].all()
    assert (dz[:, others] > 0).all() and p[:, others].min() < 2.0 ** -34 and p[:, others].max() < 2.0 ** -24


@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("rows,vocab", [(40, 300), (300, 500)])
def test_head_gradients_of_unlikely_words(th, art, rows, vocab, trans_w):  # noqa: F811
    """One word takes almost all of the probability in every row: the head's gradient at the others, p of 2^-26 to 2^-36, is a
    sum of terms with one sign.  Bounds as for the other linear tests, with 2^-40 of the part's largest below fp16's range."""
    dim = 64
    g = th.Generator(device="cuda")
    g.manual_seed(rows)
    x = th.rand((rows, dim), device="cuda", generator=g).bfloat16()
    x[:, 0] = 8
    w = (th.randn((vocab, dim), device="cuda", generator=g) / 8).bfloat16()
    w[:, 0] = 0
    w[5, 0] = 2.75
    tgt = th.full((rows,), 5, device="cuda", dtype=th.int32)
    head = w if trans_w else w.t().contiguous()
    losses, dx, dw = th.empty(rows, device="cuda"), th.empty((rows, dim), device="cuda"), th.empty(head.shape, device="cuda")
    ops.linear_cross_entropy(art, x.data_ptr(), head.data_ptr(), tgt.data_ptr(), rows, dim, vocab, trans_w=trans_w, x_dtype=OUT_BF16, w_dtype=OUT_BF16,
                             scale=1.0, losses=losses.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr())
    art.synchronize()
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    p = th.softmax(z, 1)
    ez = dim * U32 * (xd @ wd.abs().t()).amax(1, keepdim=True)
    down = z.amax(1, keepdim=True) - z
    ep = 2 * ez + down * 4 * U32 + 8 * U32
    edz = UB * p + p * (ep + UH + UB * UH) + 2.0 ** -40 * p.amax(1, keepdim=True)
    others = th.ones(vocab, device="cuda", dtype=th.bool)
    others[5] = False
    got = (dw if trans_w else dw.t()).double()
    want, err = p.t() @ xd, edz.t() @ xd + rows * U32 * ((p + edz).t() @ xd)
    assert ((got - want).abs() <= err + U32 * (want + err))[others].all()
    assert (got[others] > 0).all() and p[:, others].min() < 2.0 ** -33


def test_a_scratch_without_room_for_partial_sums(th, art):  # noqa: F811
    """A scratch sized before a tuning that splits dx's sum: dx is summed in one piece, losses and dw are the same bits; a scratch
    that ends earlier is refused."""
    rows, dim, vocab = 64, 256, 20000
    g = th.Generator(device="cuda")
    g.manual_seed(2)
    x = th.randn((rows, dim), device="cuda", generator=g).bfloat16()
    w = (th.randn((vocab, dim), device="cuda", generator=g) / 16).bfloat16()
    tgt = th.randint(0, vocab, (rows,), device="cuda", generator=g).to(th.int32)
    whole = ops.linear_loss_scratch_bytes(art, rows, dim, vocab, trans_w=True, x_dtype=OUT_BF16)
    got = []
    for size in (whole, whole - 256):
        losses, dx, dw = th.empty(rows, device="cuda"), th.empty((rows, dim), device="cuda"), th.empty((vocab, dim), device="cuda")
        scratch = art.alloc(size)
        ops.linear_cross_entropy(art, x.data_ptr(), w.data_ptr(), tgt.data_ptr(), rows, dim, vocab, trans_w=True, x_dtype=OUT_BF16, w_dtype=OUT_BF16,
                                 losses=losses.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(), scratch=scratch)
        art.synchronize()
        got.append((losses, dx, dw))
    (l0, dx0, dw0), (l1, dx1, dw1) = got
    assert th.equal(l0, l1) and th.equal(dw0, dw1)
    # the same products in another order: each sum is off by at most vocab 2^-23 of the sum of their sizes, |dz| <= p + q
    z = x.double() @ w.double().t()
    size = (th.softmax(z, 1) / rows) @ w.double().abs() + w.double().abs()[tgt.long()] / rows
    assert ((dx0 - dx1).double().abs() <= 2 * vocab * U32 * size).all()
    small = art.alloc(rows * vocab * 2)      # the exponentials alone
    with pytest.raises(T0Error, match="scratch must be"):
        ops.linear_cross_entropy(art, x.data_ptr(), w.data_ptr(), tgt.data_ptr(), rows, dim, vocab, trans_w=True, x_dtype=OUT_BF16, w_dtype=OUT_BF16,
                                 losses=l0.data_ptr(), dx=dx0.data_ptr(), dw=dw0.data_ptr(), scratch=small)


def test_a_gradient_scale_outside_f32_is_refused(th, art):  # noqa: F811
    """scale / temperature multiplies every gradient: infinite, it would leave no finite one."""
    x = th.zeros((4, 64), device="cuda")
    ids = th.zeros((4, 2), device="cuda", dtype=th.int32)
    a = x.data_ptr()
    for scale in (3e38, -3e38):
        with pytest.raises(T0Error, match="scale"):
            ops.topk_distill(art, a, ids.data_ptr(), a, 4, 64, 2, temperature=0.1, scale=scale, losses=a, dlogits=a)
        with pytest.raises(T0Error, match="scale"):
            ops.linear_topk_distill(art, a, a, ids.data_ptr(), a, 4, 8, 8, 2, temperature=0.1, scale=scale, x_dtype=OUT_BF16, w_dtype=OUT_BF16, losses=a, dx=a, dw=a)
    art.synchronize()
