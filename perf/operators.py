"""Vocabulary losses of a language model, measured: what is called, on what data, and the same in elementary torch operations.

Three operators, all at the end of a network whose last layer is a head with one column for each word of a vocabulary:

  linear_ce       softmax cross entropy of `x @ head` against target words, with the gradients of x and of the head
                  (training) or the losses alone (evaluation); the logits are never handed out
  topk_distill    Kullback-Leibler divergence from a teacher's distribution over its `topk` best words to the student's
                  softmax, from the student's logits; with the logits' gradient, or the losses alone
  linear_distill  the same from x and the head, with their gradients, or the losses alone

A case is a dict of plain values; `listed` names the measured ones, `draw` makes more of the same ranges.  `run` computes
in plain torch (float32, rounded once) or, with `own`, makes the framework's calls.  `exact` is the definition in 64 bits.
"""
import math

import torch

own = False

_BF16, _F32 = torch.bfloat16, torch.float32
_DTYPES = {"bf16": _BF16, "f32": _F32}


# ---------------------------------------------------------------------------------------------------------------- cases

def listed():
    def linear_ce(name, rows, dim, vocab, grads, head, ignored, weights):
        return dict(name=name, op="linear_ce", rows=rows, dim=dim, vocab=vocab, grads=grads, head=head, ignored=ignored, weights=weights)

    def topk_distill(name, rows, vocab, topk, grads, dtype, temperature, ragged, masked):
        return dict(name=name, op="topk_distill", rows=rows, vocab=vocab, topk=topk, grads=grads, dtype=dtype, temperature=temperature,
                    ragged=ragged, masked=masked)

    def linear_distill(name, rows, dim, vocab, topk, grads, head, temperature, ragged):
        return dict(name=name, op="linear_distill", rows=rows, dim=dim, vocab=vocab, topk=topk, grads=grads, head=head,
                    temperature=temperature, ragged=ragged)

    return [
        # scoring a handful of tokens: launches and the one pass over the head are what is paid for
        linear_ce("ce_score_16", 16, 1024, 32000, False, "vocab_dim", 0.0, False),
        # one device's rows of the MLP training configuration (1024 x 4096 -> 32000), head stored as Linear stores it
        linear_ce("ce_train_mlp_1024", 1024, 4096, 32000, True, "dim_vocab", 0.0, False),
        # a padded batch: rows without a target, weighted tokens, odd counts and an odd vocabulary
        linear_ce("ce_train_ragged_777", 777, 1000, 50257, True, "vocab_dim", 0.1, True),
        # a long batch at a large vocabulary: the largest training step
        linear_ce("ce_train_4096", 4096, 4096, 128000, True, "vocab_dim", 0.02, False),
        # perplexity of a long text: losses alone
        linear_ce("ce_eval_8191", 8191, 2048, 50257, False, "vocab_dim", 0.0, False),
        # a small student's step on a short batch
        topk_distill("distill_train_24", 24, 32000, 8, True, "f32", 1.0, False, False),
        # the losses of a validation batch, odd vocabulary, rows with fewer teacher words than the others
        topk_distill("distill_eval_2048", 2048, 50257, 20, False, "f32", 2.0, True, False),
        # a training batch with bf16 logits; the vocabulary's padded tail is masked
        topk_distill("distill_train_4096", 4096, 128000, 64, True, "bf16", 2.0, True, True),
        # float32 logits and gradient, odd sizes
        topk_distill("distill_train_1001", 1001, 32003, 32, True, "f32", 1.0, True, True),
        # a short batch straight from the hidden states
        linear_distill("lin_distill_train_128", 128, 1024, 32000, 16, True, "vocab_dim", 1.0, False),
        # losses alone
        linear_distill("lin_distill_eval_1500", 1500, 2048, 50257, 50, False, "dim_vocab", 2.0, True),
        # the large training batch, head stored as Linear stores it
        linear_distill("lin_distill_train_4096", 4096, 2048, 128000, 64, True, "dim_vocab", 2.0, True),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear_ce", "topk_distill", "linear_distill"])
    grads = rng.random() < 0.7
    vocab = _spread(rng, 500, 130000)
    if rng.random() < 0.5:
        vocab = max(512, vocab // 128 * 128)
    if op == "topk_distill":
        rows = _spread(rng, 1, max(1, min(8192, 4096 * 128000 // vocab)))
        return dict(op=op, rows=rows, vocab=vocab, topk=_spread(rng, 1, 128), grads=grads, dtype=rng.choice(["f32", "bf16"]) if rows * vocab <= 1 << 28 else "bf16",
                    temperature=rng.choice([1.0, 1.5, 2.0, 4.0]), ragged=rng.random() < 0.5, masked=rng.random() < 0.5)
    dim = _spread(rng, 64, 5120)
    dim = dim if rng.random() < 0.2 else max(64, dim // 64 * 64)
    rows = _spread(rng, 1, max(1, min(8192, 4096 * 4096 * 128000 // 2 // (vocab * dim))))
    case = dict(op=op, rows=rows, dim=dim, vocab=vocab, grads=grads, head=rng.choice(["vocab_dim", "dim_vocab"]))
    if op == "linear_ce":
        return dict(case, ignored=rng.choice([0.0, 0.02, 0.1, 0.5]), weights=rng.random() < 0.5)
    return dict(case, topk=_spread(rng, 1, 128), temperature=rng.choice([1.0, 1.5, 2.0, 4.0]), ragged=rng.random() < 0.5)


def work(case):
    """Every product once, every input read once, every output written once; rows that a mask leaves out need no product."""
    rows, vocab, grads = case["rows"], case["vocab"], case["grads"]
    k = case.get("topk", 0)
    side = rows * (8 * k + 4 + 4 if k else 4 + 4)       # ids and teacher logits or targets, and the losses
    if case["op"] == "topk_distill":
        elem = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": float(rows * vocab * elem * (2 if grads else 1) + side), "flops": float(rows * vocab * (8 if grads else 4))}
    dim = case["dim"]
    live = rows * (1.0 - case.get("ignored", 0.0))
    moved = 2 * (rows * dim + vocab * dim) * (2 if grads else 1)
    return {"bytes": float(moved + side), "flops": live * dim * vocab * (6.0 if grads else 2.0)}


# ----------------------------------------------------------------------------------------------------------------- data

def _teacher(case, gen, device):
    """ids int32 [rows, topk], distinct within a row, -1 where the teacher gave fewer words; its logits float32, best first."""
    rows, k = case["rows"], min(case["topk"], case["vocab"] - _masked_tail(case))
    span = (case["vocab"] - _masked_tail(case)) // k
    ids = torch.arange(k, device=device) * span + torch.randint(0, span, (rows, k), device=device, generator=gen)
    ids = ids.gather(1, torch.rand((rows, k), device=device, generator=gen).argsort(1))
    gaps = -torch.log(torch.rand((rows, k), device=device, generator=gen).clamp_min(1e-6))
    logits = 20.0 - gaps.cumsum(1) * (8.0 / k + 0.25)
    if case["ragged"]:
        have = torch.randint(0, k + 1, (rows, 1), device=device, generator=gen)
        ids = torch.where(torch.arange(k, device=device) < have, ids, torch.full_like(ids, -1))
    return ids.to(torch.int32), logits.to(_F32)


def _masked_tail(case):
    return 60 if case.get("masked") else 0


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    state = {"case": case}
    if case["op"] != "linear_ce":
        state["ids"], state["teacher"] = _teacher(case, gen, device)
    if case["op"] == "topk_distill":
        # a student that agrees in part: its logits at the teacher's words are raised towards the teacher's
        dtype = _DTYPES[case["dtype"]]
        z = torch.empty((rows, vocab), device=device, dtype=dtype)
        for r in range(0, rows, 512):
            part = torch.randn((min(512, rows - r), vocab), device=device, generator=gen) * 2.0
            ids = state["ids"][r:r + 512].long()
            lift = (state["teacher"][r:r + 512] * 0.6 + torch.randn(ids.shape, device=device, generator=gen)) * (ids >= 0)
            part.scatter_add_(1, ids.clamp_min(0), lift)
            if case["masked"]:
                part[:, vocab - _masked_tail(case):] = -math.inf
            z[r:r + 512] = part.to(dtype)
        state["logits"] = z
        return state
    dim = case["dim"]
    w = (torch.randn((vocab, dim), device=device, generator=gen) / math.sqrt(dim)).to(_BF16)
    x = torch.randn((rows, dim), device=device, generator=gen) * 2.0
    if case["op"] == "linear_ce":
        targets = torch.randint(0, vocab, (rows,), device=device, generator=gen)
        x += w[targets].float() * (torch.rand((rows, 1), device=device, generator=gen) * 20.0)    # from unsure to sure
        if case["ignored"]:
            targets = torch.where(torch.rand(rows, device=device, generator=gen) < case["ignored"], torch.full_like(targets, -1), targets)
        state["targets"] = targets.to(torch.int32)
        state["weights"] = torch.rand(rows, device=device, generator=gen) * 2.0 if case["weights"] else None
    else:
        for k in range(min(4, state["ids"].shape[1])):
            ids = state["ids"][:, k].long()
            x += w[ids.clamp_min(0)].float() * ((ids >= 0) * (12.0 - 2.0 * k))[:, None]
    state["x"] = x.to(_BF16)
    state["w"] = w if case["head"] == "vocab_dim" else w.t().contiguous()
    return state


# ----------------------------------------------------------------------------------------------------------- plain form

def _softmax_parts(z):
    """z - max, exp of it, its sum: float32 [rows, vocab]."""
    z = z - z.amax(1, keepdim=True)
    e = z.exp()
    return z, e, e.sum(1, keepdim=True)


def _teacher_probs(ids, teacher, temperature):
    """The teacher's probabilities over the words it gave, and their logarithms; 0 and 0 at the empty places."""
    have = ids >= 0
    t = teacher.float() / temperature
    t = t - torch.where(have, t, torch.full_like(t, -math.inf)).amax(1, keepdim=True).clamp_min(-3e38)
    e = t.exp() * have
    s = e.sum(1, keepdim=True)
    some = s > 0
    s = torch.where(some, s, torch.ones_like(s))
    return torch.where(have, e / s, torch.zeros_like(e)), torch.where(have, t - s.log(), torch.zeros_like(t)), some


def _distill_plain(z, ids, teacher, temperature, scale, grads):
    at = ids.long().clamp_min(0)
    q, log_q, some = _teacher_probs(ids, teacher, temperature)
    z, e, s = _softmax_parts(z.float() / temperature)
    losses = (q * (log_q - (z.gather(1, at) - s.log()))).sum(1)
    if not grads:
        return losses, None
    g = e / s * some
    g.scatter_add_(1, at, -q)
    return losses, g * (scale / temperature)


def _head_plain(x, w, head):
    return x.float() @ (w.float().t() if head == "vocab_dim" else w.float())


def _head_grads_plain(x, w, g, head):
    if head == "vocab_dim":
        return (g @ w.float()).to(_BF16), (g.t() @ x.float()).to(_BF16)
    return (g @ w.float().t()).to(_BF16), (x.float().t() @ g).to(_BF16)


def _run_plain(state):
    case = state["case"]
    scale = 1.0 / case["rows"]
    if case["op"] == "topk_distill":
        losses, g = _distill_plain(state["logits"], state["ids"], state["teacher"], case["temperature"], scale, case["grads"])
        return {"losses": losses} if g is None else {"losses": losses, "dlogits": g.to(state["logits"].dtype)}
    z = _head_plain(state["x"], state["w"], case["head"])
    if case["op"] == "linear_ce":
        targets = state["targets"].long()
        live = targets >= 0
        at = targets.clamp_min(0)[:, None]
        z, e, s = _softmax_parts(z)
        losses = torch.where(live, (s.log() - z.gather(1, at))[:, 0], torch.zeros_like(s[:, 0]))
        if not case["grads"]:
            return {"losses": losses}
        g = e / s
        g.scatter_add_(1, at, torch.full_like(s, -1.0))
        g = g * ((live if state["weights"] is None else live * state["weights"]) * scale)[:, None]
    else:
        losses, g = _distill_plain(z, state["ids"], state["teacher"], case["temperature"], scale, case["grads"])
        if g is None:
            return {"losses": losses}
    dx, dw = _head_grads_plain(state["x"], state["w"], g, case["head"])
    return {"losses": losses, "dx": dx, "dw": dw}


# ------------------------------------------------------------------------------------------------- the framework's calls

_RT = None


def _runtime():
    """The runtime that a program keeps; its launches and torch's own work share one stream."""
    global _RT
    if _RT is None:
        from t0_gpu_b200 import GpuRuntime

        _RT = GpuRuntime(torch.cuda.current_device())
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(stream)
        _RT.set_stream(stream.cuda_stream)
    return _RT


def _run_own(state):
    from t0_gpu_b200 import OUT_BF16, OUT_F32, ops

    rt, case = _runtime(), state["case"]
    rows, vocab, grads = case["rows"], case["vocab"], case["grads"]
    losses = torch.empty(rows, device="cuda", dtype=_F32)
    if case["op"] == "topk_distill":
        z = state["logits"]
        kind = OUT_BF16 if z.dtype == _BF16 else OUT_F32
        dz = torch.empty_like(z) if grads else None
        ops.topk_distill(rt, z.data_ptr(), state["ids"].data_ptr(), state["teacher"].data_ptr(), rows, vocab, state["ids"].shape[1],
                         temperature=case["temperature"], logits_dtype=kind, grad_dtype=kind, losses=losses.data_ptr(), grads=grads,
                         dlogits=dz.data_ptr() if grads else None)
        return {"losses": losses, "dlogits": dz} if grads else {"losses": losses}
    x, w = state["x"], state["w"]
    dx, dw = (torch.empty_like(x), torch.empty_like(w)) if grads else (None, None)
    common = dict(trans_w=case["head"] == "vocab_dim", x_dtype=OUT_BF16, w_dtype=OUT_BF16, dx_dtype=OUT_BF16, dw_dtype=OUT_BF16, grads=grads,
                  losses=losses.data_ptr(), dx=dx.data_ptr() if grads else None, dw=dw.data_ptr() if grads else None)
    if case["op"] == "linear_ce":
        weights = state["weights"]
        ops.linear_cross_entropy(rt, x.data_ptr(), w.data_ptr(), state["targets"].data_ptr(), rows, case["dim"], vocab,
                                 row_weights=None if weights is None else weights.data_ptr(), **common)
    else:
        ops.linear_topk_distill(rt, x.data_ptr(), w.data_ptr(), state["ids"].data_ptr(), state["teacher"].data_ptr(), rows, case["dim"], vocab,
                                state["ids"].shape[1], temperature=case["temperature"], **common)
    return {"losses": losses, "dx": dx, "dw": dw} if grads else {"losses": losses}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------------------- exact

def exact(case, seed):
    """The definitions in 64 bits: p = softmax(z / T); loss = -sum q log p + sum q log q; dz = (p sum(q) - q) scale / T."""
    state = prepare(case, seed)
    rows, vocab = case["rows"], case["vocab"]
    t = float(case.get("temperature", 1.0))
    linear = case["op"] != "topk_distill"
    if linear:
        wt = state["w"].double() if case["head"] == "vocab_dim" else state["w"].double().t()      # [vocab, dim]
        x = state["x"].double()
    losses, dx, dz = [], [], []
    dw = torch.zeros_like(wt) if linear and case["grads"] else None
    for r in range(0, rows, 1024):
        z = (x[r:r + 1024] @ wt.t() if linear else state["logits"][r:r + 1024].double()) / t
        n = z.shape[0]
        log_p = z - torch.logsumexp(z, 1, keepdim=True)
        q = torch.zeros_like(z)
        if case["op"] == "linear_ce":
            target = state["targets"][r:r + 1024].long()
            q[torch.arange(n, device=z.device), target.clamp_min(0)] = (target >= 0).double()
            spread = torch.zeros(n, device=z.device, dtype=torch.float64)
        else:
            ids = state["ids"][r:r + 1024].long()
            log_q = (state["teacher"][r:r + 1024].double() / t).masked_fill(ids < 0, -math.inf)
            log_q = log_q - torch.logsumexp(log_q, 1, keepdim=True)
            log_q = log_q.masked_fill(ids < 0, -math.inf)        # a row without words: minus infinity everywhere
            q.scatter_add_(1, ids.clamp_min(0), log_q.exp())
            spread = (log_q.exp() * log_q.masked_fill(ids < 0, 0.0)).sum(1)
        losses.append(spread - (q * log_p.masked_fill(q == 0, 0.0)).sum(1))
        if case["grads"]:
            weight = torch.full((n, 1), 1.0 / rows / t, device=z.device, dtype=torch.float64)
            if state.get("weights") is not None:
                weight = weight * state["weights"][r:r + 1024].double()[:, None]
            g = log_p.exp() * q.sum(1, keepdim=True).gt(0)
            g.sub_(q).mul_(weight)
            if linear:
                dx.append(g @ wt)
                dw += g.t() @ x[r:r + 1024]
            else:
                dz.append(g)
        del z, log_p, q
    out = {"losses": torch.cat(losses)}
    if case["grads"] and linear:
        out["dx"], out["dw"] = torch.cat(dx), dw if case["head"] == "vocab_dim" else dw.t()
    elif case["grads"]:
        out["dlogits"] = torch.cat(dz)
    return out
