"""Vocabulary losses (cross entropy and distillation from hidden states or logits) against their definitions in 64 bits.

Bounds.  u32 = 2^-23 covers one f32 operation of the tensor cores or of ex2.approx (rounded or truncated), u_b = 2^-8 and
u_h = 2^-11 a rounding to bf16 and fp16.  A logit is a sum of `dim` exact products: |dz| <= dim u32 sum|x w| =: ez.  A
probability is exp of a difference of such logits times 1 / T, divided by a sum of such: relative error
  ep = 2 ez / T + (max z - z) / T * 4 u32 + 8 u32,
and a loss, a sum of differences of logarithms, is off by at most 2 ez / T + (|z - max z| / T + 16) 8 u32.  The gradient of a
logit, a (p - q), is stored in bf16 after exp went through fp16 (absolute 2^-25 of the part's largest below fp16's normal
range); dx and dw are sums of those times bf16 operands, plus their f32 summation and the rounding of the result."""
import math

import numpy as np
import pytest

import t0_gpu_b200 as t
from t0_gpu_b200 import OUT_BF16, OUT_F32, T0Error, ops

pytestmark = pytest.mark.gpu

U32, UB, UH = 2.0 ** -23, 2.0 ** -8, 2.0 ** -11


@pytest.fixture(scope="module")
def th():
    import torch

    return torch


@pytest.fixture(scope="module")
def art(th):
    """A runtime on a torch stream, so that tensors made by torch are ordered with its launches."""
    r = t.GpuRuntime()
    s = th.cuda.Stream()
    with th.cuda.stream(s):
        r.set_stream(s.cuda_stream)
        yield r
        r.synchronize()
    r.close()


def make_teacher(th, rows, topk, vocab, seed, ragged):
    g = np.random.default_rng(seed)
    ids = np.stack([g.choice(vocab, size=min(topk, vocab), replace=False) for _ in range(rows)]).astype(np.int64)
    if topk > vocab:
        ids = np.concatenate([ids, np.full((rows, topk - vocab), -1)], 1)
    logits = g.normal(size=(rows, topk)) * 3
    if ragged:
        for r in range(rows):
            have = r % (topk + 1)
            ids[r, have:] = -1
            logits[r, have:] = [np.nan, np.inf, -np.inf][r % 3]
    return th.tensor(ids.astype(np.int32), device="cuda"), th.tensor(logits.astype(np.float32), device="cuda")


def target_rows(th, ids, teacher, temperature, vocab):
    """q [rows, vocab], sum over words of q log q, live rows -- all in 64 bits."""
    ids = ids.long()
    have = (ids >= 0) & (ids < vocab) & ~(th.isneginf(teacher) & (ids >= 0))
    lq = (teacher.double() / temperature).masked_fill(~have, -math.inf)
    live = have.any(1)
    lq = th.where(live[:, None], lq - th.logsumexp(lq, 1, keepdim=True), lq)
    q = th.zeros((ids.shape[0], vocab), dtype=th.float64, device="cuda")
    pk = lq.exp()
    q.scatter_add_(1, ids.clamp(0, vocab - 1), pk.masked_fill(~have, 0.0))
    ent = (pk * lq.masked_fill(~have, 0.0)).masked_fill(~have, 0.0).sum(1)
    return q, ent, live


def losses_and_dz(th, z, q, ent, live, temperature, row_scale):
    z = z / temperature
    top = z.amax(1, keepdim=True)
    some = live & ~th.isneginf(top[:, 0])
    top = top.masked_fill(~some[:, None], 0.0)
    log_s = (z - top).exp().sum(1, keepdim=True).log()
    lp = (z - top) - log_s                      # not z - logsumexp: beside z = -3e38 that would lose log_s, in 64 bits too
    lse = top + log_s
    losses = ent - (q * lp.masked_fill(q == 0, 0.0)).sum(1)
    p = lp.exp().masked_fill(~some[:, None], 0.0)
    dz = (p * q.sum(1, keepdim=True) - q) * (row_scale / temperature)[:, None]
    losses, dz = losses.masked_fill(~some, 0.0), dz.masked_fill(~some[:, None], 0.0)
    return losses, dz, p, lse[:, 0]


def check_linear(th, art, rows, dim, vocab, trans_w, *, topk=0, temperature=1.0, grads=True, x_dtype=OUT_BF16, gdt=OUT_BF16, weights=True, ignore=True,
                 piece_rows=0, ldx_pad=0, ldw_pad=0, ragged=True, big=1.0, offset=0, keep=None, ldd_pad=0, x_needs=True, w_needs=True):
    g = th.Generator(device="cuda")
    g.manual_seed(rows * 7919 + dim * 31 + vocab)
    w_rows, w_cols = (vocab, dim) if trans_w else (dim, vocab)
    wbuf = (th.randn((w_rows * (w_cols + ldw_pad) + offset,), device="cuda", generator=g) / math.sqrt(dim)).bfloat16()
    w = wbuf[offset:].view(w_rows, w_cols + ldw_pad)[:, :w_cols]
    wd = (w if trans_w else w.t()).double()                                     # [vocab, dim]
    xt = th.bfloat16 if x_dtype == OUT_BF16 else th.float32
    x = (th.randn((rows, dim + ldx_pad), device="cuda", generator=g) * 2 * big).to(xt)[:, :dim]
    ldx, ldw = dim + ldx_pad, w_cols + ldw_pad
    keep = None if keep is None else th.tensor([r in keep for r in range(rows)], device="cuda")
    if topk:
        ids, teacher = make_teacher(th, rows, topk, vocab, rows + topk, ragged)
        if keep is not None:
            ids[~keep] = -1
        q, ent, live = target_rows(th, ids, teacher, temperature, vocab)
    else:
        tgt = th.randint(0, vocab, (rows,), device="cuda", generator=g)
        x = x.clone() if not ldx_pad else x
        if ignore:
            tgt[::3] = -1
        if keep is not None:
            tgt[~keep] = -1
        live = tgt >= 0
        q = th.zeros((rows, vocab), dtype=th.float64, device="cuda")
        q[th.arange(rows, device="cuda"), tgt.clamp_min(0)] = live.double()
        ent = th.zeros(rows, dtype=th.float64, device="cuda")
        tgt = tgt.to(th.int32)
    if (ignore or keep is not None) and (grads or rows > 256):
        x[~live] = math.nan                                                     # a row that is left out may hold anything
    rw = th.rand(rows, device="cuda", generator=g) * 2 if weights else None
    scale = 1.0 / rows
    row_scale = (rw.double() if weights else th.ones(rows, device="cuda", dtype=th.float64)) * scale
    xd = x.bfloat16().double().masked_fill(~live[:, None], 0.0)
    z = xd @ wd.t()
    losses_ref, dz, p, lse_ref = losses_and_dz(th, z, q, ent, live, temperature, row_scale)
    losses, lse = th.full((rows,), 7.0, device="cuda"), th.full((rows,), 7.0, device="cuda")
    odt = th.bfloat16 if gdt == OUT_BF16 else th.float32
    dxb = th.full((rows + 1, dim + ldd_pad), 7.0, device="cuda", dtype=odt)
    dwb = th.full((w_rows + 1, w_cols + ldd_pad), 7.0, device="cuda", dtype=odt)
    dx, dw = dxb[:, :dim], dwb[:, :w_cols]
    kw = dict(grads=grads, trans_w=trans_w, x_dtype=x_dtype, w_dtype=OUT_BF16, dx_dtype=gdt, dw_dtype=gdt, ldx=ldx, ldw=ldw, losses=losses.data_ptr(),
              lse=lse.data_ptr(), dx=dx.data_ptr() if grads else None, dw=dw.data_ptr() if grads else None, piece_rows=piece_rows,
              lddx=dim + ldd_pad, lddw=w_cols + ldd_pad, x_needs=x_needs, w_needs=w_needs, row_weights=rw.data_ptr() if weights else None)
    if topk:
        ops.linear_topk_distill(art, x.data_ptr(), w.data_ptr(), ids.data_ptr(), teacher.data_ptr(), rows, dim, vocab, topk, temperature=temperature, **kw)
    else:
        ops.linear_cross_entropy(art, x.data_ptr(), w.data_ptr(), tgt.data_ptr(), rows, dim, vocab, **kw)
    art.synchronize()
    xa, wa = xd.abs(), wd.abs()
    ez = (dim * U32) * (xa @ wa.t()).amax(1) / temperature                       # per row
    down = (z.amax(1, keepdim=True) - z) / temperature
    reach = (down * (q > 0)).amax(1)
    tol = 2 * ez + (reach + 16 + lse_ref.abs()) * 8 * U32
    assert ((losses.double() - losses_ref).abs() <= tol).all(), ((losses.double() - losses_ref).abs() / tol).max()
    assert (losses[~live] == 0).all()
    assert ((lse.double() - lse_ref)[live].abs() <= tol[live]).all() and (lse[~live] == 0).all()
    if not grads:
        assert (dx == 7).all() and (dw == 7).all()
        return
    a = (row_scale / temperature).abs()[:, None] * live[:, None]
    ep = 2 * ez[:, None] + down * 4 * U32 + 8 * U32
    edz = UB * dz.abs() + a * (p * (ep + UH + UB * UH) + 2.0 ** -24 * p.amax(1, keepdim=True))
    full = dz.abs() + edz
    uo = UB if gdt == OUT_BF16 else U32
    dx_ref, edx = dz @ wd, edz @ wa + vocab * U32 * (full @ wa)
    bound = edx + uo * (dx_ref.abs() + edx) + 1e-30
    err = (dx[:rows].double() - dx_ref).abs()
    assert not x_needs or (err <= bound).all(), (err / bound).max()
    dw_ref, edw = dz.t() @ xd, edz.t() @ xa + rows * U32 * (full.t() @ xa)
    bound = edw + uo * (dw_ref.abs() + edw) + 1e-30
    got = dw[:w_rows].double() if trans_w else dw[:w_rows].double().t()
    err = (got - dw_ref).abs()
    assert not w_needs or (err <= bound).all(), (err / bound).max()
    # nothing behind the last row, behind a row's end, or where no gradient was asked for
    assert (dxb[rows] == 7).all() and (dwb[w_rows] == 7).all() and (dxb[:, dim:] == 7).all() and (dwb[:, w_cols:] == 7).all()
    assert (x_needs or (dxb == 7).all()) and (w_needs or (dwb == 7).all())
    assert not x_needs or (dx[:rows][~live] == 0).all()


LINEAR_SIZES = [(1, 64, 64), (1, 8, 1), (3, 40, 17), (33, 64, 129), (128, 128, 1000), (130, 200, 513), (257, 96, 2048), (300, 1000, 777), (64, 72, 5001)]


@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("rows,dim,vocab", LINEAR_SIZES)
def test_linear_ce(th, art, rows, dim, vocab, trans_w):
    check_linear(th, art, rows, dim, vocab, trans_w)


@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("rows,dim,vocab,topk", [(1, 64, 64, 1), (2, 8, 5, 9), (33, 64, 129, 4), (130, 200, 513, 33), (257, 96, 2048, 100), (40, 64, 3001, 1024)])
def test_linear_topk_distill(th, art, rows, dim, vocab, topk, trans_w):
    check_linear(th, art, rows, dim, vocab, trans_w, topk=topk, temperature=2.0)


@pytest.mark.parametrize("topk", [0, 5])
@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("rows,dim,vocab", [(1, 64, 64), (70, 100, 999), (300, 256, 4000)])
def test_linear_losses_alone(th, art, rows, dim, vocab, trans_w, topk):
    check_linear(th, art, rows, dim, vocab, trans_w, topk=topk, grads=False, ignore=False)


@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("x_dtype,gdt", [(OUT_F32, OUT_F32), (OUT_F32, OUT_BF16), (OUT_BF16, OUT_F32)])
def test_linear_types(th, art, x_dtype, gdt, trans_w):
    check_linear(th, art, 65, 136, 777, trans_w, x_dtype=x_dtype, gdt=gdt)
    check_linear(th, art, 65, 136, 776, trans_w, x_dtype=x_dtype, gdt=gdt, topk=7)


@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("gdt", [OUT_F32, OUT_BF16])
@pytest.mark.parametrize("vocab", [640, 601])
def test_linear_in_pieces_of_rows(th, art, vocab, gdt, trans_w):
    check_linear(th, art, 300, 128, vocab, trans_w, gdt=gdt, piece_rows=128)
    check_linear(th, art, 100, 60, vocab, trans_w, gdt=gdt, piece_rows=33, topk=6)


@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("keep", [[], [699], [5, 64, 300], list(range(64)), list(range(600, 665)), list(range(700))])
def test_linear_rows_left_out(th, art, keep, trans_w):
    """Products run over the rows with a target alone once there is more than a tile of rows: none, one, whole 64-row blocks."""
    for piece_rows in (0, 33, 256):
        check_linear(th, art, 700, 72, 200, trans_w, keep=keep, piece_rows=piece_rows, ignore=len(keep) < 700)
        check_linear(th, art, 700, 64, 136, trans_w, keep=keep, piece_rows=piece_rows, topk=3, gdt=OUT_F32, ragged=False)
    check_linear(th, art, 700, 72, 200, trans_w, keep=keep, grads=False)


@pytest.mark.parametrize("trans_w", [False, True])
def test_linear_pitches_and_offsets(th, art, trans_w):
    check_linear(th, art, 50, 64, 320, trans_w, ldx_pad=8, ldw_pad=16)
    check_linear(th, art, 50, 64, 320, trans_w, ldx_pad=3, ldw_pad=5)
    check_linear(th, art, 50, 64, 320, trans_w, offset=1)
    check_linear(th, art, 50, 64, 320, trans_w, grads=False, ignore=False, ldx_pad=1, offset=3)


@pytest.mark.parametrize("trans_w", [False, True])
@pytest.mark.parametrize("gdt", [OUT_F32, OUT_BF16])
@pytest.mark.parametrize("rows", [50, 300])
def test_linear_gradient_pitches(th, art, rows, gdt, trans_w):
    for pad in (8, 3):
        check_linear(th, art, rows, 72, 321, trans_w, gdt=gdt, ldd_pad=pad, piece_rows=0 if pad == 8 else 128)


@pytest.mark.parametrize("rows", [50, 300])
@pytest.mark.parametrize("x_needs,w_needs", [(True, False), (False, True)])
def test_linear_one_gradient(th, art, rows, x_needs, w_needs):
    check_linear(th, art, rows, 64, 200, True, x_needs=x_needs, w_needs=w_needs)
    check_linear(th, art, rows, 64, 200, False, topk=4, x_needs=x_needs, w_needs=w_needs)


@pytest.mark.parametrize("trans_w,dim,vocab", [(True, 5, 700), (True, 157, 3001), (True, 499, 700), (True, 1030, 333), (False, 64, 157), (False, 99, 2101)])
def test_linear_heads_with_rows_off_16_bytes(th, art, trans_w, dim, vocab):
    """Copies in rows of 32, 64, 128 and 256 threads, the last ones partly idle."""
    check_linear(th, art, 6, dim, vocab, trans_w)
    check_linear(th, art, 182, dim, vocab, trans_w, topk=3)


@pytest.mark.parametrize("trans_w", [False, True])
def test_linear_large_logits(th, art, trans_w):
    check_linear(th, art, 100, 64, 700, trans_w, big=40.0)


# ------------------------------------------------------------------------------------------------ on given logits

def check_logits(th, art, rows, cols, topk, *, dtype=OUT_F32, gdt=None, temperature=1.0, pad=0, offset=0, ragged=True, mask=0, in_place=False, weights=True,
                 grads=True, ids=None, teacher=None, edit=None):
    gdt = dtype if gdt is None else gdt
    dt, odt = (th.bfloat16 if k == OUT_BF16 else th.float32 for k in (dtype, gdt))
    g = th.Generator(device="cuda")
    g.manual_seed(rows * 7919 + cols * 31 + topk)
    ld = cols + pad
    buf = (th.randn((rows * ld + offset + 64,), device="cuda", generator=g) * 4).to(dt)
    view = buf[offset:offset + rows * ld].view(rows, ld)
    if ids is None:
        ids, teacher = make_teacher(th, rows, topk, cols, rows + topk, ragged)
    if mask:
        view[:, cols - mask:cols] = -math.inf
    if edit:
        edit(view)
    q, ent, live = target_rows(th, ids, teacher, temperature, cols)
    view[~live, :cols] = math.nan if rows % 2 else math.inf                      # rows that are left out may hold anything
    z = view[:, :cols].double().masked_fill(~live[:, None], 0.0)
    before = buf.clone()
    rw = th.rand(rows, device="cuda", generator=g) * 2 if weights else None
    row_scale = (rw.double() if weights else th.ones(rows, device="cuda", dtype=th.float64)) / rows
    losses_ref, dz, p, lse = losses_and_dz(th, z, q, ent, live, temperature, row_scale)
    losses = th.full((rows + 1,), 7.0, device="cuda")
    out = buf if in_place else th.full((rows * ld + offset + 64,), 7.0, device="cuda", dtype=odt)
    kept = out.clone()
    dview = out[offset:offset + rows * ld].view(rows, ld)
    ops.topk_distill(art, view.data_ptr(), ids.data_ptr(), teacher.data_ptr(), rows, cols, topk, temperature=temperature, logits_dtype=dtype, grad_dtype=gdt,
                     ld=ld, losses=losses.data_ptr(), dlogits=dview.data_ptr() if grads else None, grads=grads, row_weights=rw.data_ptr() if weights else None)
    art.synchronize()
    zmax = z.amax(1, keepdim=True)
    down = ((zmax - z) / temperature).nan_to_num(0.0, 0.0, 0.0)
    reach = (down * (q > 0)).amax(1)
    tol = (reach + 16 + ent.abs()) * 8 * U32
    got = losses[:rows].double()
    masked = th.isinf(losses_ref)                                                # a target is masked
    assert (got[masked] == losses_ref[masked]).all()
    # A loss within its bound of the largest f32 may round to infinity.
    fin = ~masked & ~((losses_ref + tol > th.finfo(th.float32).max) & th.isposinf(got))
    assert ((got - losses_ref).abs()[fin] <= tol[fin]).all(), ((got - losses_ref).abs() / tol)[fin].max()
    assert losses[rows] == 7
    if not in_place:
        assert th.equal(buf.view(th.int16 if dtype == OUT_BF16 else th.int32), before.view(th.int16 if dtype == OUT_BF16 else th.int32))
    if not grads:
        assert (out == 7).all()
        return
    a = (row_scale / temperature).abs()[:, None] * live[:, None]
    uo = UB if gdt == OUT_BF16 else U32
    bound = uo * dz.abs() + a * (p * (down * 4 + 16) + q * (8 + 4 * ent.abs()[:, None])) * U32 * 2 + 1e-37
    if dtype == gdt == OUT_BF16:      # exponentials kept in fp16 between the passes, relative to the largest of their slice
        bound += a * (1 + uo) * (p * UH + 2.0 ** -24 * p.amax(1, keepdim=True))
    err = (dview[:, :cols].double() - dz).abs()
    assert (err <= bound).all(), (err / bound).max()
    assert (dview[:, :cols][~live] == 0).all()
    if pad:
        assert th.equal(dview[:, cols:].float().nan_to_num(1e9), kept[offset:offset + rows * ld].view(rows, ld)[:, cols:].float().nan_to_num(1e9))
    assert th.equal(out[offset + rows * ld:], kept[offset + rows * ld:]) and th.equal(out[:offset], kept[:offset])


LOGIT_SIZES = [(1, 1, 1), (1, 7, 3), (5, 33, 4), (3, 1000, 20), (40, 4097, 8), (300, 2050, 16), (2, 32000, 64), (5, 50257, 9), (150, 13000, 5), (3, 150001, 1024)]


@pytest.mark.parametrize("dtype", [OUT_F32, OUT_BF16])
@pytest.mark.parametrize("rows,cols,topk", LOGIT_SIZES)
def test_topk_distill(th, art, rows, cols, topk, dtype):
    check_logits(th, art, rows, cols, topk, dtype=dtype)


@pytest.mark.parametrize("dtype,gdt", [(OUT_F32, OUT_BF16), (OUT_BF16, OUT_F32)])
def test_topk_distill_mixed_types(th, art, dtype, gdt):
    check_logits(th, art, 9, 1001, 6, dtype=dtype, gdt=gdt)
    check_logits(th, art, 9, 1024, 6, dtype=dtype, gdt=gdt, temperature=3.0)


@pytest.mark.parametrize("dtype", [OUT_F32, OUT_BF16])
@pytest.mark.parametrize("pad,offset", [(0, 0), (5, 0), (8, 1), (3, 3)])
def test_topk_distill_pitches_offsets_masks_in_place(th, art, dtype, pad, offset):
    for in_place in (False, True):
        check_logits(th, art, 7, 2000, 6, dtype=dtype, pad=pad, offset=offset, in_place=in_place, mask=9 if pad else 0, temperature=1.5)
    check_logits(th, art, 7, 2000, 6, dtype=dtype, pad=pad, offset=offset, grads=False)


@pytest.mark.parametrize("dtype", [OUT_F32, OUT_BF16])
def test_topk_distill_long_rows_are_read_twice(th, art, dtype):
    cols = 450_000 if dtype == OUT_F32 else 900_001
    check_logits(th, art, 3, cols, 5, dtype=dtype)
    check_logits(th, art, 2, cols, 5, dtype=dtype, in_place=True)


def test_topk_distill_offsets_past_32_bits(th, art):
    """4.3e9 logits, in place: all rows but the last two are left out and become zeros."""
    rows, cols = 33100, 130000
    z = th.empty((rows, cols), device="cuda", dtype=th.bfloat16)
    z[-2:] = th.randn((2, cols), device="cuda").bfloat16()
    z[0], z[rows // 2], last = math.nan, math.nan, z[-2:].double()
    ids = th.full((rows, 3), -1, device="cuda", dtype=th.int32)
    ids[-2:] = th.tensor([[5, 77, cols - 1], [0, 1, 2]], device="cuda", dtype=th.int32)
    teacher = th.randn((rows, 3), device="cuda")
    losses = th.empty(rows, device="cuda")
    ops.topk_distill(art, z.data_ptr(), ids.data_ptr(), teacher.data_ptr(), rows, cols, 3, logits_dtype=OUT_BF16, grad_dtype=OUT_BF16,
                     losses=losses.data_ptr(), dlogits=z.data_ptr(), scale=1.0)
    art.synchronize()
    q, ent, live = target_rows(th, ids[-2:], teacher[-2:], 1.0, cols)
    ref, dz, p, _ = losses_and_dz(th, last, q, ent, live, 1.0, th.ones(2, device="cuda", dtype=th.float64))
    assert ((losses[-2:].double() - ref).abs() <= 1e-4).all() and (losses[:-2] == 0).all()
    assert ((z[-2:].double() - dz).abs() <= UB * dz.abs() + (1 + UB) * (p * (UH + 64 * U32) + 2.0 ** -24 * p.amax(1, keepdim=True)) + q * 32 * U32).all()
    assert (z[0] == 0).all() and (z[rows // 2] == 0).all() and (z[-3] == 0).all()


def test_topk_distill_values_at_the_edge(th, art):
    """Logits at the type's lowest value, a row of nothing but it, rows of -inf alone, huge differences."""
    lowest = th.finfo(th.float32).min

    def edit(z):
        z[0] = lowest
        z[1, 1:] = lowest
        z[2] = -math.inf
        z[3, ::2] = -math.inf
        z[4, 5] = 3e38

    check_logits(th, art, 6, 500, 3, ragged=False, edit=edit)


def test_topk_distill_same_word_twice(th, art):
    ids = th.tensor([[3, 3, 9, 3], [0, 0, 0, 0], [5, -1, 5, 6]], device="cuda", dtype=th.int32)
    teacher = th.tensor([[1.0, 0.5, 2.0, -1.0], [1.0, 1.0, 1.0, 1.0], [0.0, math.nan, 2.0, 1.0]], device="cuda")
    check_logits(th, art, 3, 40, 4, ids=ids, teacher=teacher)
    rows, dim, vocab = 3, 16, 40
    x = th.randn((rows, dim), device="cuda").bfloat16()
    w = th.randn((vocab, dim), device="cuda").bfloat16()
    z = (x.double() @ w.double().t())
    q, ent, live = target_rows(th, ids, teacher, 1.0, vocab)
    losses_ref, dz, p, _ = losses_and_dz(th, z, q, ent, live, 1.0, th.full((rows,), 1.0 / rows, device="cuda", dtype=th.float64))
    losses, dx = th.empty(rows, device="cuda"), th.empty((rows, dim), device="cuda")
    ops.linear_topk_distill(art, x.data_ptr(), w.data_ptr(), ids.data_ptr(), teacher.data_ptr(), rows, dim, vocab, 4, trans_w=True, x_dtype=OUT_BF16,
                            w_dtype=OUT_BF16, losses=losses.data_ptr(), dx=dx.data_ptr())
    art.synchronize()
    assert ((losses.double() - losses_ref).abs() <= 1e-4).all()      # |z| < 40: 2 ez = 2 * 16 * 2^-23 * 16 * 16 < 1e-3 / 10
    edz = UB * dz.abs() + p * (UH + 1e-4) / rows + 1e-8
    assert ((dx.double() - dz @ w.double()).abs() <= edz @ w.double().abs() + 1e-5).all()


@pytest.mark.parametrize("rows,cols,topk,offset", [(700, 1000, 20, 0), (3, 32000, 200, 0), (5, 50257, 1024, 0), (150, 40000, 64, 0), (150, 40000, 1000, 0), (4, 3000, 300, 1)])
def test_topk_distill_same_word_twice_in_every_form(th, art, rows, cols, topk, offset):
    """Rows with no word twice, with one pair, with many and with one word alone, next to each other; a stride of 2^k between
    words that differ."""
    g = th.Generator(device="cuda")
    g.manual_seed(rows + cols)
    ids = th.stack([th.randperm(cols, device="cuda", generator=g)[:topk] for _ in range(rows)]).to(th.int32)
    ids[0, -1] = ids[0, 0]
    ids[1] = cols - 1
    ids[2] %= 7
    if rows > 3:
        ids[3] = th.arange(topk, device="cuda", dtype=th.int32) * 512 % cols
    teacher = th.randn((rows, topk), device="cuda", generator=g) * 2
    check_logits(th, art, rows, cols, topk, ids=ids, teacher=teacher, offset=offset)


# ------------------------------------------------------------------------------------------- in a user's program

@pytest.mark.parametrize("rows,d,V", [(64, 256, 1000), (300, 128, 2048)])
def test_mlp_step_without_logits(th, rows, d, V):
    """MlpTrainer(keep_logits=False): the step of the trainer that keeps them, up to the roundings of the logits' gradient."""
    from t0_gpu_b200.mlp import MlpConfig, MlpTrainer

    rt = t.GpuRuntime()
    cfg = MlpConfig(d_in=d, hidden=[d, d], n_classes=V)
    g = th.Generator(device="cuda")
    g.manual_seed(5)
    s = th.cuda.Stream()
    with th.cuda.stream(s):
        x = th.randn((rows, d), device="cuda", generator=g)
        targets = th.randint(0, V, (rows,), device="cuda", generator=g).to(th.int32)
        a = MlpTrainer(rt, cfg, rows, seed=3, autotune=False)
        b = MlpTrainer(rt, cfg, rows, seed=3, autotune=False, keep_logits=False)
        a.forward_backward(x, targets)
        b.forward_backward(x, targets)
        rt.synchronize()
        h, w, dz = a.h16[-1].double(), a.w16[-1].double(), a.dlogits16.double()
        # |z| <= sum |h w|; a loss is a difference of logarithms of sums of exponentials of such (bounds at the top of this file)
        ez = d * U32 * (h.abs() @ w.abs()).amax(1)
        assert ((a.losses - b.losses).abs() <= 4 * ez + 64 * U32 * (1 + a.losses.abs())).all()
        # dz: rounded to bf16 on both sides, and through fp16 on one, of exponentials that differ by the logits' error
        p = th.softmax(a.logits.double(), 1)
        e = 2 * UB * dz.abs() + (p * (UH + 4 * ez[:, None] + 2.0 ** -18) + 2.0 ** -24) / rows
        bound = h.abs().t() @ e + rows * U32 * (h.abs().t() @ dz.abs())
        assert ((a.dw[-1] - b.dw[-1]).double().abs() <= bound).all()
        for _ in range(3):
            b.step(x, targets)
        assert math.isfinite(b.mean_loss()) and not hasattr(b, "logits")
    rt.synchronize()
    rt.close()


def test_ops_run_together_with_f32_buffers(rt):
    """A training step of a student head through ops alone, f32 buffers in and out: cross entropy, distillation from logits
    that `matmul` made, distillation from hidden states, all on the same head, and an optimizer step on their sum."""
    rng = np.random.default_rng(3)
    rows, dim, vocab, topk = 40, 64, 200, 5
    x = rng.standard_normal((rows, dim)).astype(np.float32)
    w = (rng.standard_normal((dim, vocab)) / 8).astype(np.float32)
    tgt = rng.integers(0, vocab, rows).astype(np.uint32)
    tgt[::7] = ops.NO_WORD
    ids = np.stack([rng.choice(vocab, topk, replace=False) for _ in range(rows)]).astype(np.uint32)
    teacher = rng.standard_normal((rows, topk)).astype(np.float32)
    xb, wb, tb, ib, lb = rt.upload_f32(x), rt.upload_f32(w), rt.upload(tgt), rt.upload(ids), rt.upload_f32(teacher)
    ce, dx_ce, dw_ce = ops.linear_cross_entropy(rt, xb, wb, tb, rows, dim, vocab)
    kd, dx_kd, dw_kd = ops.linear_topk_distill(rt, xb, wb, ib, lb, rows, dim, vocab, topk, temperature=2.0, weight_id=77)
    z, backward = ops.matmul(rt, xb, wb, rows, dim, vocab, weight_id=77)
    kd2, dz = ops.topk_distill(rt, z, ib, lb, rows, vocab, topk, temperature=2.0)
    dx2, dw2 = backward(dz)
    get = lambda b, shape: b.read_as(np.float32, int(np.prod(shape))).reshape(shape)   # noqa: E731
    assert np.abs(get(kd, rows) - get(kd2, rows)).max() <= 1e-5          # the same logits: 64 products of |x w| < 2, 2^-23 each
    # both round the same dz to bf16 (and fp16 on one side): 2^-8 + 2^-11 of sum |dz w| each
    dzn, w16 = np.abs(get(dz, (rows, vocab))), np.abs(w)
    assert (np.abs(get(dx_kd, (rows, dim)) - get(dx2, (rows, dim))) <= (2 * UB + 2 * UH) * (dzn @ w16.T) * 1.01 + 1e-6).all()
    assert (np.abs(get(dw_kd, (dim, vocab)) - get(dw2, (dim, vocab))) <= (2 * UB + 2 * UH) * (np.abs(x).T @ dzn) * 1.01 + 1e-6).all()
    losses, grad = ops.cross_entropy(rt, z, tb, rows, vocab)
    got = get(ce, rows)
    assert abs(losses - got.sum() / rows) <= 1e-5 and (got[::7] == 0).all()
    n = dim * vocab
    rt._check(t._lib.lib().t0b_residual_add(rt.handle, dw_ce.gpu_addr(), dw_kd.gpu_addr(), n, 1))
    m, v = rt.alloc_zero(n * 4), rt.alloc_zero(n * 4)
    ops.adamw_step(rt, wb, dw_ce, m, v, n, 1, weight_id=77)
    ce2, none_x, none_w = ops.linear_cross_entropy(rt, xb, wb, tb, rows, dim, vocab, grads=False, weight_id=77)
    assert none_x is None and none_w is None and get(ce2, rows).sum() != got.sum()
    # the f32 head was converted anew: with and without a cached copy the same
    ce3, _, _ = ops.linear_cross_entropy(rt, xb, wb, tb, rows, dim, vocab, grads=False)
    assert np.array_equal(get(ce2, rows), get(ce3, rows))


def _ce(art, th, x, w, tgt, **kw):
    rows, dim = x.shape
    vocab = w.shape[0]
    losses, dx, dw = th.empty(rows, device="cuda"), th.empty((rows, dim), device="cuda"), th.empty((vocab, dim), device="cuda")
    ops.linear_cross_entropy(art, x.data_ptr(), w.data_ptr(), tgt.data_ptr(), rows, dim, vocab, trans_w=True, x_dtype=OUT_BF16, w_dtype=OUT_BF16,
                             losses=losses.data_ptr(), dx=dx.data_ptr(), dw=dw.data_ptr(), **kw)
    return losses, dx, dw


def _ce_data(th, rows, dim, vocab, seed):
    g = th.Generator(device="cuda")
    g.manual_seed(seed)
    x = th.randn((rows, dim), device="cuda", generator=g).bfloat16()
    w = (th.randn((vocab, dim), device="cuda", generator=g) / math.sqrt(dim)).bfloat16()
    return x, w, th.randint(0, vocab, (rows,), device="cuda", generator=g).to(th.int32)


def test_same_bits_every_time_and_on_another_stream(th, art):
    x, w, tgt = _ce_data(th, 500, 128, 3000, 1)
    first = _ce(art, th, x, w, tgt)
    art.synchronize()
    first = [v.clone() for v in first]
    other = th.cuda.Stream()
    other.wait_stream(th.cuda.current_stream())
    for k in range(4):
        if k == 2:
            art.set_stream(other.cuda_stream)
        got = _ce(art, th, x, w, tgt)
        art.synchronize()
        assert all(th.equal(a, b) for a, b in zip(first, got))
    art.set_stream(th.cuda.current_stream().cuda_stream)


def test_two_runtimes_at_once(th):
    import threading

    x, w, tgt = _ce_data(th, 300, 128, 2000, 2)
    th.cuda.synchronize()
    rts = [t.GpuRuntime() for _ in range(2)]
    outs = [[None] * 6 for _ in rts]

    def work(k):
        for j in range(6):
            outs[k][j] = _ce(rts[k], th, x, w, tgt)
        rts[k].synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(2)]
    [q.start() for q in threads]
    [q.join() for q in threads]
    assert all(th.equal(a, b) for o in outs for got in o for a, b in zip(outs[0][0], got))
    [r.close() for r in rts]


def test_captured_and_replayed(th, art):
    """Two graphs with a scratch each, replayed on new inputs between eager calls; without a scratch a captured call is refused."""
    rows, dim, vocab = 400, 64, 1500
    x, w, tgt = _ce_data(th, rows, dim, vocab, 3)
    z = th.randn((rows, 700), device="cuda")
    ids, teacher = make_teacher(th, rows, 6, 700, 4, True)
    eager = [v.clone() for v in _ce(art, th, x, w, tgt)]
    art.synchronize()
    L = t._lib.lib()
    nbytes = ops.linear_loss_scratch_bytes(art, rows, dim, vocab, trans_w=True, x_dtype=OUT_BF16)
    graphs, outs = [], []
    for k in range(2):
        scratch = art.alloc(nbytes)
        losses, dz = th.empty(rows, device="cuda"), th.empty_like(z)
        import ctypes as C

        art.synchronize()
        art._check(L.t0b_graph_begin(art.handle))
        out = _ce(art, th, x, w, tgt, scratch=scratch)
        ops.topk_distill(art, z.data_ptr(), ids.data_ptr(), teacher.data_ptr(), rows, 700, 6, losses=losses.data_ptr(), dlogits=dz.data_ptr())
        handle = C.c_uint64()
        art._check(L.t0b_graph_end(art.handle, C.byref(handle)))
        graphs.append((handle.value, scratch))
        outs.append((out, losses, dz))
    art._check(L.t0b_graph_begin(art.handle))
    with pytest.raises(T0Error, match="scratch"):
        _ce(art, th, x, w, tgt)
    handle = C.c_uint64()
    art._check(L.t0b_graph_end(art.handle, C.byref(handle)))
    art._check(L.t0b_graph_destroy(art.handle, handle))
    x2, _, _ = _ce_data(th, rows, dim, vocab, 9)
    for step in range(2):
        for handle, _ in graphs:
            art._check(L.t0b_graph_launch(art.handle, handle, 1))
        big = _ce(art, th, *_ce_data(th, 900, dim, 5000, 8))          # a larger eager call: the context's workspace grows
        art.synchronize()
        want = eager if step == 0 else [v.clone() for v in _ce(art, th, x, w, tgt)]
        art.synchronize()
        for out, losses, dz in outs:
            assert all(th.equal(a, b) for a, b in zip(want, out))
        x.copy_(x2)
        del big
    want_l, want_dz = th.empty(rows, device="cuda"), th.empty_like(z)
    ops.topk_distill(art, z.data_ptr(), ids.data_ptr(), teacher.data_ptr(), rows, 700, 6, losses=want_l.data_ptr(), dlogits=want_dz.data_ptr())
    art.synchronize()
    assert all(th.equal(want_l, o[1]) and th.equal(want_dz, o[2]) for o in outs)
    for handle, _ in graphs:
        art._check(L.t0b_graph_destroy(art.handle, handle))


def test_an_index_outside_the_vocabulary_is_reported_and_left_out(th, art):
    x, w, tgt = _ce_data(th, 300, 64, 100, 4)
    bad = tgt.clone()
    bad[7] = 100
    good = tgt.clone()
    good[7] = -1
    want = [v.clone() for v in _ce(art, th, x, w, good)]
    art.synchronize()
    for sl in (slice(0, 300), slice(0, 40)):
        got = _ce(art, th, x[sl].contiguous(), w, bad[sl].contiguous())
        with pytest.raises(T0Error, match="110"):
            art.synchronize()
        if sl.stop == 300:
            assert all(th.equal(a, b) for a, b in zip(want, got))
    z = th.randn((3, 50), device="cuda")
    ids = th.tensor([[1, 50], [60, 70], [3, 4]], device="cuda", dtype=th.int32)
    teacher = th.zeros((3, 2), device="cuda")
    losses, dz = th.empty(3, device="cuda"), th.empty_like(z)
    ops.topk_distill(art, z.data_ptr(), ids.data_ptr(), teacher.data_ptr(), 3, 50, 2, losses=losses.data_ptr(), dlogits=dz.data_ptr())
    with pytest.raises(T0Error, match="110"):
        art.synchronize()
    ce = -th.log_softmax(z.double(), 1)
    assert abs(losses[0].item() - ce[0, 1].item()) < 1e-5 and losses[1] == 0 and (dz[1] == 0).all() and losses[2] > 0
    assert art.device_status(True) in (0, 110)


def test_gradients_against_differences(th, art):
    """Central differences of the losses' sum: the formulas' gradients are those of the losses the library reports."""
    rows, cols, topk = 4, 37, 5
    g = th.Generator(device="cuda")
    g.manual_seed(11)
    z = th.randn((rows, cols), device="cuda", generator=g)
    ids, teacher = make_teacher(th, rows, topk, cols, 2, False)
    losses, dz = th.empty(rows, device="cuda"), th.empty_like(z)
    run = lambda zz, out: ops.topk_distill(art, zz.data_ptr(), ids.data_ptr(), teacher.data_ptr(), rows, cols, topk, temperature=1.5, scale=1.0,   # noqa: E731
                                           losses=losses.data_ptr(), dlogits=out, grads=out is not None)
    run(z, dz.data_ptr())
    h = 2.0 ** -6
    for col in (0, 5, int(ids[0, 0]), cols - 1):
        diff = th.zeros(rows, device="cuda", dtype=th.float64)
        for sign in (1, -1):
            zz = z.clone()
            zz[:, col] += sign * h
            run(zz, None)
            art.synchronize()
            diff += sign * losses.double()
        # third derivative of the loss <= 1 / T^3: h^2 / 6; f32 losses of size < 8: 2 * 8 * 8 * 2^-23 / (2 h)
        assert ((diff / (2 * h) - dz[:, col].double()).abs() <= h * h / 6 + 64 * U32 / h).all()


def test_empty_calls(th, art):
    w = th.ones((30, 16), device="cuda").bfloat16()
    x = th.ones((1, 16), device="cuda").bfloat16()
    dw = th.full((30, 16), 7.0, device="cuda")
    ops.linear_cross_entropy(art, x.data_ptr(), w.data_ptr(), x.data_ptr(), 0, 16, 30, trans_w=True, x_dtype=OUT_BF16, w_dtype=OUT_BF16, losses=x.data_ptr(),
                             dx=x.data_ptr(), dw=dw.data_ptr())
    art.synchronize()
    assert (dw == 0).all() and (x == 1).all()
    ops.topk_distill(art, x.data_ptr(), x.data_ptr(), x.data_ptr(), 0, 16, 4, losses=x.data_ptr(), grads=False)
    art.synchronize()
    assert (x == 1).all()


def test_refusals(th, art):
    x, w, tgt = _ce_data(th, 8, 32, 64, 5)
    ids, teacher = make_teacher(th, 8, 3, 64, 1, False)
    out = th.empty((64, 64), device="cuda")
    p, o = x.data_ptr(), out.data_ptr()

    def linear(match, targets=tgt.data_ptr(), xp=p, wp=w.data_ptr(), rows=8, dim=32, vocab=64, **kw):
        kw = {**dict(trans_w=True, x_dtype=OUT_BF16, w_dtype=OUT_BF16, losses=o, dx=o, dw=o), **kw}
        with pytest.raises(T0Error, match=match) as e:
            ops.linear_cross_entropy(art, xp, wp, targets, rows, dim, vocab, **kw)
        assert e.value.code in (-1, -5) and not art.is_poisoned()

    linear("null", targets=0)
    linear("null", xp=0)
    linear("null", wp=0)
    linear("empty head", vocab=0)
    linear("empty head", dim=0)
    linear("pitch", ldx=31)
    linear("pitch", ldw=16)
    linear("x_dtype", x_dtype=5)
    linear("gradient type", dx_dtype=9)
    linear("aligned", xp=p + 1)
    linear("aligned", targets=tgt.data_ptr() + 2)
    linear("finite", scale=math.nan)
    linear("scratch", scratch=art.alloc(1024))          # U alone takes 8 * 64 * 2 bytes
    small = art.alloc(16)
    linear("does not|needs", xp=small, rows=4096)

    def distill(match, zp=o, topk=3, cols=64, **kw):
        with pytest.raises(T0Error, match=match):
            ops.topk_distill(art, zp, kw.pop("ids", ids.data_ptr()), kw.pop("teacher", teacher.data_ptr()), 8, cols, topk, losses=o, grads=False, **kw)
        with pytest.raises(T0Error, match=match if "logits" not in match and "columns" not in match else None):
            ops.linear_topk_distill(art, p if zp else 0, w.data_ptr(), kw.pop("ids", ids.data_ptr()) if match != "null" else 0, teacher.data_ptr(), 8, 32,
                                    64 if cols else 0, topk, trans_w=True, x_dtype=OUT_BF16 if "logits_dtype" not in kw else 7, w_dtype=OUT_BF16, losses=o,
                                    grads=False, **{k: v for k, v in kw.items() if k in ("temperature", "ldk", "scale")})

    distill("null", zp=0)
    distill("topk", topk=0)
    distill("topk", topk=1025)
    distill("topk", ldk=2)
    distill("temperature", temperature=0.0)
    distill("temperature", temperature=-1.0)
    distill("temperature", temperature=math.inf)
    distill("temperature", temperature=1e-39)
    distill("logits_dtype", logits_dtype=7)
    distill("columns", cols=0)
    with pytest.raises(T0Error, match="their type"):
        ops.topk_distill(art, o, ids.data_ptr(), teacher.data_ptr(), 8, 64, 3, grad_dtype=OUT_BF16, losses=o, dlogits=o)
    with pytest.raises(ValueError):
        ops.linear_cross_entropy(art, p, w.data_ptr(), tgt.data_ptr(), 8, 32, 64, x_dtype=OUT_BF16, w_dtype=3)
    with pytest.raises(ValueError, match="captured"):
        ops.linear_cross_entropy(art, p, w.data_ptr(), tgt.data_ptr(), 8, 32, 64, x_dtype=OUT_BF16, scratch=art.alloc(1 << 20))
    art.synchronize()
