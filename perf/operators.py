"""The losses between a model's answers and what it learns from them, as cases that can be timed and checked.

A case is a dict of plain values; `op` names the operator and the rest are its sizes:

  logprobs  log probabilities of given tokens from logits, with the distributions' entropies and top
            alternatives (`token_logprobs`); `grad` adds the backward of the first two
  head      the same (no alternatives) from hidden states and the vocabulary matrix, without stored
            logits (`lm_head_logprobs`); `grad` adds the backward
  distill   Kullback-Leibler divergence from a teacher's top logits, forward and backward (`topk_distill`)
  balance   load-balance and router-z loss of routed pools with per-pool counts, forward and backward
            (`pool_balance`)

`run` computes an operator in elementary torch operations in 32 bits, or, where `own` is set, through
the framework.  `exact` restates the definitions in 64 bits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
F64 = torch.float64

MAX_LOGITS = 4096 * 131072       # logits of the largest listed case of logprobs
MAX_HEAD = 8192 * 32768 * 1024   # products of the largest listed head
BAN_STEP, BAN_AT = 97, 13        # columns a program never samples (their logits are -inf)


# ----------------------------------------------------------------------------- the cases

def listed():
    return [
        # four sequences' next tokens with a handful of alternatives: one answer of a server, all latency
        dict(name="logprobs_4x8192", op="logprobs", T=4, V=8192, dtype="fp32", top=8, tau=1.0, banned=True, grad=False),
        # the teacher's targets of one training batch (128 x 64 tokens, vocabulary 2048), softened
        dict(name="logprobs_teacher", op="logprobs", T=8192, V=2048, dtype="fp32", top=64, tau=2.0, banned=False,
             grad=False),
        # policy training on sampled tokens with an entropy bonus, odd sizes, rows off any alignment
        dict(name="logprobs_policy", op="logprobs", T=4099, V=32771, dtype="bf16", top=0, tau=0.7, banned=True,
             grad=True),
        # scoring a corpus with a large vocabulary and a few alternatives
        dict(name="logprobs_corpus", op="logprobs", T=4096, V=131072, dtype="bf16", top=20, tau=1.0, banned=False,
             grad=False),
        # the head of one short batch of the small model
        dict(name="head_200", op="head", T=200, d=512, V=2048, tau=1.0, grad=True),
        # scoring a ragged batch at the scaled step's width and vocabulary
        dict(name="head_score_1000", op="head", T=1000, d=1024, V=8200, tau=1.0, grad=False),
        # policy training from hidden states with a large vocabulary
        dict(name="head_8192", op="head", T=8192, d=1024, V=32768, tau=1.0, grad=True),
        # one short batch distilled from sixteen kept alternatives
        dict(name="distill_64", op="distill", T=64, V=2048, K=16, dtype="fp32", tau=2.0, tail=False),
        # the training batch (128 x 64 tokens) distilled from 64 kept alternatives
        dict(name="distill_8192", op="distill", T=8192, V=2048, K=64, dtype="fp32", tau=2.0, tail=False),
        # a large odd vocabulary, the teacher's remaining mass as one more alternative
        dict(name="distill_tail", op="distill", T=4099, V=32771, K=32, dtype="bf16", tau=1.0, tail=True),
        # the routed layer of the training step: 8192 tokens, top-8 of 64 pools
        dict(name="balance_8192", op="balance", T=8192, C=64, k=8, dtype="fp32", masked=False),
        # a long accumulated batch, top-16 of 256 pools, padding left out
        dict(name="balance_131071", op="balance", T=131071, C=256, k=16, dtype="fp32", masked=True),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(lo * (hi / lo) ** rng.random() + 0.5)))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "head", "distill", "distill", "balance"])
    if op == "logprobs":
        V = _spread(rng, 1000, 131072)
        T = _spread(rng, 1, max(1, min(16384, MAX_LOGITS // V // 4)))
        grad = rng.random() < 0.5
        return dict(op=op, T=T, V=V, dtype=rng.choice(["bf16", "fp32"]), top=0 if grad else rng.choice([0, 1, 5, 20, 64, 128]),
                    tau=rng.choice([0.7, 1.0, 2.0]), banned=rng.random() < 0.5, grad=grad)
    if op == "head":
        d = rng.choice([256, 512, 1024])
        V = 8 * _spread(rng, 125, 4096)
        T = _spread(rng, 16, min(8192, MAX_HEAD // (d * V)))
        return dict(op=op, T=T, d=d, V=V, tau=rng.choice([0.7, 1.0]), grad=rng.random() < 0.7)
    if op == "distill":
        V = _spread(rng, 1000, 65536)
        T = _spread(rng, 1, max(1, min(16384, MAX_LOGITS // V // 8)))
        return dict(op=op, T=T, V=V, K=rng.choice([1, 8, 16, 50, 64, 128]), dtype=rng.choice(["bf16", "fp32"]),
                    tau=rng.choice([1.0, 2.0]), tail=rng.random() < 0.5)
    C = rng.choice([16, 32, 48, 64, 100, 128, 256])
    return dict(op=op, T=_spread(rng, 1, 131072), C=C, k=rng.choice([1, 2, 4, 8, 16]),
                dtype=rng.choice(["bf16", "fp32"]), masked=rng.random() < 0.5)


def work(case):
    """The bytes every input and output holds once, and the operations of the formulas."""
    op, T = case["op"], case["T"]
    if op == "balance":
        es, C, k = (4 if case["dtype"] == "fp32" else 2), case["C"], case["k"]
        return {"bytes": 2 * T * C * es + T * k * 4 + (T if case["masked"] else 0) + 4 * C, "flops": 14 * T * C}
    V = case["V"]
    if op == "head":
        d, g = case["d"], case["grad"]
        moved = (T + V) * d * 2 * (2 if g else 1) + T * (8 + 4 + 4 + (8 if g else 0))
        return {"bytes": moved, "flops": 2 * T * d * V * (3 if g else 1)}
    es = 4 if case["dtype"] == "fp32" else 2
    if op == "logprobs":
        g = case["grad"]
        return {"bytes": T * V * es * (2 if g else 1) + T * (8 + 4 + 4 + 8 * case["top"] + (8 if g else 0)),
                "flops": T * V * (12 if g else 6)}
    return {"bytes": T * V * es * 2 + T * (8 * case["K"] + 8), "flops": T * V * 10}


# ----------------------------------------------------------------------------- inputs

def _tokens(T, V, banned, g):
    """Sampled tokens (never a banned one), with a sixteenth of the positions padded (-1)."""
    tok = torch.randint(0, V, (T,), device=DEV, generator=g)
    if banned:
        tok = torch.where(tok % BAN_STEP == BAN_AT, (tok - 1).clamp_min(0), tok)
    pad = torch.rand(T, device=DEV, generator=g) < 1 / 16
    return torch.where(pad, -1, tok)


def _logits(T, V, g):
    """Logits with popular and rare columns."""
    x = torch.randn(T, V, device=DEV, generator=g).mul_(2.0)
    return x.add_(torch.randn(V, device=DEV, generator=g).mul_(1.5))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, T = case["op"], case["T"]
    st = dict(case=case)
    if op == "balance":
        C, k = case["C"], case["k"]
        x = torch.randn(T, C, device=DEV, generator=g) + 0.7 * torch.randn(C, device=DEV, generator=g)
        x = x.to(DTYPES[case["dtype"]])
        st["ids"] = torch.topk(x.float(), k, dim=1).indices.to(torch.int32).contiguous()
        st["mask"] = (torch.rand(T, device=DEV, generator=g) < 7 / 8) if case["masked"] else None
        st["x"] = x.requires_grad_()
        st["g"] = (torch.rand((), device=DEV, generator=g) + 0.5, torch.rand((), device=DEV, generator=g) + 0.5)
        return st
    V = case["V"]
    if op == "head":
        d = case["d"]
        st["tok"] = _tokens(T, V, False, g)
        w = torch.randn(V, d, device=DEV, generator=g).mul_(2.0 / math.sqrt(d))
        h = torch.randn(T, d, device=DEV, generator=g)
        h += 1.5 * w[st["tok"].clamp_min(0)]  # the model leans towards the token that came
        st["h"] = h.to(torch.bfloat16).requires_grad_(case["grad"])
        st["w"] = w.to(torch.bfloat16).requires_grad_(case["grad"])
        st["g"] = (torch.randn(T, device=DEV, generator=g), 0.1 * torch.rand(T, device=DEV, generator=g))
        return st
    dt = DTYPES[case["dtype"]]
    x = _logits(T, V, g)
    if op == "logprobs":
        st["tok"] = _tokens(T, V, case["banned"], g)
        x[torch.arange(T, device=DEV), st["tok"].clamp_min(0)] += 5.0
        if case["banned"]:
            x[:, BAN_AT::BAN_STEP] = -math.inf
        st["x"] = x.to(dt).requires_grad_(case["grad"])
        st["g"] = (torch.randn(T, device=DEV, generator=g), 0.1 * torch.rand(T, device=DEV, generator=g))
        return st
    # the teacher agrees with the student up to noise; some rows keep fewer alternatives, some none
    K, tau = case["K"], case["tau"]
    teacher = x + torch.randn(T, V, device=DEV, generator=g)
    st["x"] = x.to(dt).requires_grad_()
    top, ids = torch.topk(teacher, K, dim=1)
    if case["tail"]:
        top = (top - torch.logsumexp(teacher / tau, 1, keepdim=True) * tau) / tau
    keep = torch.where(torch.rand(T, device=DEV, generator=g) < 1 / 8,
                       (torch.rand(T, device=DEV, generator=g) * (K + 1)).long(), K)
    gone = torch.arange(K, device=DEV)[None, :] >= keep[:, None]
    st["ids"] = torch.where(gone, -1, ids).to(torch.int32)
    st["t"] = top.float().contiguous()
    st["g"] = torch.rand(T, device=DEV, generator=g) + 0.5
    return st


# ----------------------------------------------------------------------------- one pass

def _ops():
    pkg = str(Path(__file__).resolve().parent.parent / "speedup-thingy_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from rte_amd.kernels import hip_ops

    return hip_ops


def run(state):
    case = state["case"]
    return (_run_own if own else _PLAIN[case["op"]])(state, case)


def _run_own(st, case):
    ops, op = _ops(), case["op"]
    if op == "logprobs":
        if not case["grad"]:
            out = ops.token_logprobs(st["x"], st["tok"], n_top=case["top"], temperature=case["tau"])
            return tuple(out[:4 if case["top"] else 2])
        lp, ent, _, _ = ops.token_logprobs(st["x"], st["tok"], temperature=case["tau"])
        (dx,) = torch.autograd.grad((lp, ent), (st["x"],), st["g"])
        return lp.detach(), ent.detach(), dx
    if op == "head":
        lp, ent = ops.lm_head_logprobs(st["h"], st["w"], st["tok"], temperature=case["tau"])
        if not case["grad"]:
            return lp, ent
        dh, dw = torch.autograd.grad((lp, ent), (st["h"], st["w"]), st["g"])
        return lp.detach(), ent.detach(), dh, dw
    if op == "distill":
        loss = ops.topk_distill(st["x"], st["ids"], st["t"], temperature=case["tau"], tail=case["tail"])
        (dx,) = torch.autograd.grad(loss, st["x"], st["g"])
        return loss.detach(), dx
    bal, z, counts = ops.pool_balance(st["x"], st["ids"], mask=st["mask"])
    (dx,) = torch.autograd.grad((bal, z), st["x"], st["g"])
    return bal.detach(), z.detach(), counts, dx


def _top_of(x, k):
    """The k largest of each row and their columns: value descending, ties to the lower column."""
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long() << 32
    key += (x.shape[1] - 1) - torch.arange(x.shape[1], device=x.device)
    cols = torch.topk(key, k, dim=1).indices
    return x.gather(1, cols), cols.to(torch.int32)


def _plain_rows(x, tok, tau):
    """(log probabilities [T, V], of the tokens [T], entropies [T], max) of softmax(x / tau)."""
    z = x.float() / tau
    z = z - z.amax(1, keepdim=True)
    lse = z.exp().sum(1, keepdim=True).log()
    lp = z - lse
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, 0.0).sum(1)
    valid = tok >= 0
    picked = torch.where(valid, lp.gather(1, tok.clamp_min(0)[:, None])[:, 0], 0.0)
    return lp, p, picked, ent, valid


def _plain_rows_grad(lp, p, ent, tok, valid, g, tau):
    """d(sum g_0 picked + g_1 entropy) / dx."""
    ga = torch.where(valid, g[0], 0.0)
    d = torch.where(p > 0, -p * (ga[:, None] + g[1][:, None] * (lp + ent[:, None])), 0.0)
    d.scatter_add_(1, tok.clamp_min(0)[:, None], ga[:, None])
    return d / tau


def _plain_logprobs(st, case):
    x, tok, tau = st["x"].detach(), st["tok"], case["tau"]
    lp, p, picked, ent, valid = _plain_rows(x, tok, tau)
    if case["grad"]:
        return picked, ent, _plain_rows_grad(lp, p, ent, tok, valid, st["g"], tau).to(x.dtype)
    if case["top"]:
        _, cols = _top_of(x.float(), case["top"])
        return picked, ent, lp.gather(1, cols.long()), cols
    return picked, ent


def _plain_head(st, case):
    h, w, tok, tau = st["h"].detach().float(), st["w"].detach().float(), st["tok"], case["tau"]
    lp, p, picked, ent, valid = _plain_rows(h @ w.t(), tok, tau)
    if not case["grad"]:
        return picked, ent
    d = _plain_rows_grad(lp, p, ent, tok, valid, st["g"], tau)
    return picked, ent, (d @ w).to(st["h"].dtype), (d.t() @ h).to(st["w"].dtype)


def _plain_distill(st, case):
    """Sums over the vocabulary in 32 bits; what belongs to the list in 64, with the student's total put
    together from the list and the rest: the terms of a student near its teacher cancel to the square of
    their difference."""
    x, ids, t, tau = st["x"].detach(), st["ids"].long(), st["t"].double(), case["tau"]
    here = ids >= 0
    at = ids.clamp_min(0)
    some = here.any(1)
    z = x.float() / tau
    z = z - z.amax(1, keepdim=True)
    zl = torch.where(here, z.gather(1, at).double(), -math.inf)
    e = z.exp()
    on = torch.zeros_like(e).scatter_add_(1, at, here.float()) > 0
    rest_e = torch.where(on, 0.0, e)
    so = rest_e.sum(1).double()
    s = so + zl.exp().sum(1)
    q = e / s.float()[:, None]
    if case["tail"]:
        lt = torch.where(here, t, -math.inf)
    else:
        tt = torch.where(here, t / tau, -math.inf)
        tt = tt - torch.where(some, tt.amax(1), 0.0)[:, None]
        lt = tt - tt.exp().sum(1, keepdim=True).clamp_min(1e-300).log()
    p = lt.exp()
    loss = torch.where(p > 0, p * (lt - (zl - s.log()[:, None])), 0.0).sum(1)
    onto = torch.zeros_like(q).scatter_add_(1, at, p.float())
    if case["tail"]:
        rest = (1.0 - p.sum(1)).clamp_min(0.0)
        loss = loss + torch.where((rest > 0) & some, rest * (rest.log() - (so.log() - s.log())), 0.0)
        onto = onto + rest_e * (rest / so).float()[:, None]
    d = (q - onto) * (st["g"] * tau)[:, None]
    return torch.where(some, loss * (tau * tau), 0.0).float(), torch.where(some[:, None], d, 0.0).to(x.dtype)


def _plain_balance(st, case):
    x, ids, mask = st["x"].detach(), st["ids"].long(), st["mask"]
    T, C = x.shape
    z = x.float()
    m = z.amax(1, keepdim=True)
    e = (z - m).exp()
    s = e.sum(1, keepdim=True)
    p = e / s
    lse = (m + s.log())[:, 0]
    ok = torch.ones(T, device=x.device) if mask is None else mask.float()
    n = ok.sum().clamp_min(1.0)
    hits = torch.zeros(T, C, device=x.device).scatter_add_(1, ids, torch.ones_like(ids, dtype=torch.float32))
    counts = (hits * ok[:, None]).sum(0)
    f = counts / counts.sum().clamp_min(1.0)
    bal = C * (f * ((p * ok[:, None]).sum(0) / n)).sum()
    zl = (lse.square() * ok).sum() / n
    gb, gz = st["g"]
    d = p * (gb * C * (f - (p * f).sum(1, keepdim=True)) + (gz * 2.0 * lse)[:, None]) * (ok / n)[:, None]
    return bal, zl, counts.to(torch.int32), d.to(x.dtype)


_PLAIN = {"logprobs": _plain_logprobs, "head": _plain_head, "distill": _plain_distill, "balance": _plain_balance}


# ----------------------------------------------------------------------------- 64-bit results

def _by_rows(fn, T, V):
    """fn(lo, hi) over ranges of rows of at most 2^27 values, the tuples joined."""
    step = max(1, (1 << 27) // max(V, 1))
    parts = [fn(lo, min(T, lo + step)) for lo in range(0, T, step)]
    return tuple(torch.cat(c) for c in zip(*parts))


def _exact_softmax_rows(z, tok, g, tau):
    """Of the 64-bit scores z = x / tau: (log p of the tokens, entropies, gradient in x or None, log p)."""
    lp = torch.log_softmax(z, 1)
    p = torch.softmax(z, 1)
    ent = torch.special.entr(p).sum(1)
    own_row = torch.arange(len(tok), device=tok.device)
    at = tok.clamp_min(0)
    valid = (tok >= 0).to(F64)
    picked = torch.where(tok >= 0, lp[own_row, at], torch.zeros((), dtype=F64, device=tok.device))
    if g is None:
        return picked, ent, None, lp
    a, b = g[0].to(F64) * valid, g[1].to(F64)
    d = -a[:, None] * p + b[:, None] * (torch.special.entr(p) - p * ent[:, None])
    d[own_row, at] += a
    return picked, ent, d / tau, lp


def exact(case, seed):
    st = prepare(case, seed)
    return {"logprobs": _exact_logprobs, "head": _exact_head, "distill": _exact_distill,
            "balance": _exact_balance}[case["op"]](st, case)


def _exact_logprobs(st, case):
    x, tok, k = st["x"].detach(), st["tok"], case["top"]

    def rows(lo, hi):
        g = [v[lo:hi] for v in st["g"]] if case["grad"] else None
        picked, ent, d, lp = _exact_softmax_rows(x[lo:hi].to(F64) / case["tau"], tok[lo:hi], g, case["tau"])
        if case["grad"]:
            return picked, ent, d
        # a stable descending sort of the few candidates at least as large as the k-th value
        vals = x[lo:hi].to(F64)
        if k == 0:
            return picked, ent
        kth = torch.topk(vals, k, dim=1).values[:, -1:]
        n = int((vals >= kth).sum(1).max())
        cand = torch.topk((vals >= kth).to(torch.int8).float(), n, dim=1).indices.sort(1).values
        cv = vals.gather(1, cand)
        order = torch.sort(cv, dim=1, descending=True, stable=True).indices[:, :k]
        cols = cand.gather(1, order)
        return picked, ent, lp.gather(1, cols), cols.to(torch.int32)

    return _by_rows(rows, *x.shape)


def _exact_head(st, case):
    h, w, tok = st["h"].detach().to(F64), st["w"].detach().to(F64), st["tok"]
    dw = torch.zeros_like(w)

    def rows(lo, hi):
        g = [v[lo:hi] for v in st["g"]] if case["grad"] else None
        z = h[lo:hi] @ w.t() / case["tau"]
        picked, ent, d, _ = _exact_softmax_rows(z, tok[lo:hi], g, case["tau"])
        if d is None:
            return picked, ent
        dw.addmm_(d.t(), h[lo:hi])
        return picked, ent, d @ w

    out = _by_rows(rows, len(tok), case["V"])
    return out if not case["grad"] else (*out, dw)


def _exact_distill(st, case):
    x, tau = st["x"].detach(), case["tau"]

    def rows(lo, hi):
        z = x[lo:hi].to(F64) / tau
        ids, t, g = st["ids"][lo:hi].long(), st["t"][lo:hi].to(F64), st["g"][lo:hi].to(F64)
        zero = torch.zeros((), dtype=F64, device=z.device)
        target = torch.zeros(z.shape[0], z.shape[1] + 1, dtype=F64, device=z.device)
        here = ids >= 0
        col = torch.where(here, ids, z.shape[1])  # missing entries fall into a spare column
        if case["tail"]:
            pj = torch.where(here, t.exp(), zero)
        else:
            pj = torch.softmax(torch.where(here, t / tau, torch.full_like(t, -math.inf)), 1)
            pj = torch.where(here, pj, zero)
        target.scatter_(1, col, pj)
        target = target[:, :-1].contiguous()
        lq = torch.log_softmax(z, 1)
        q = lq.exp()
        loss = torch.special.xlogy(target, target).sum(1) - (target * lq).sum(1)
        d = q - target
        if case["tail"]:
            on = torch.zeros(z.shape[0], z.shape[1] + 1, dtype=torch.bool, device=z.device)
            on.scatter_(1, col, here)
            zr = z.masked_fill(on[:, :-1], -math.inf)
            rest = (1.0 - pj.sum(1)).clamp_min(0.0)
            lqr = torch.logsumexp(zr, 1) - torch.logsumexp(z, 1)
            loss = loss + torch.special.xlogy(rest, rest) - rest * lqr
            d = d - rest[:, None] * torch.softmax(zr, 1)
        some = here.any(1)
        return (torch.where(some, loss * tau * tau, zero), torch.where(some[:, None], d * (g * tau)[:, None], zero))

    return _by_rows(rows, *x.shape)


def _exact_balance(st, case):
    x, ids, mask = st["x"].detach().to(F64), st["ids"].long(), st["mask"]
    T, C = x.shape
    rows = torch.arange(T, device=x.device) if mask is None else mask.nonzero()[:, 0]
    n = max(1, rows.numel())
    counts = torch.bincount(ids[rows].reshape(-1), minlength=C)
    f = counts.to(F64) / max(1, int(counts.sum()))
    p = torch.softmax(x[rows], 1)
    lse = torch.logsumexp(x[rows], 1)
    bal = C * (p.sum(0) / n) @ f
    z = (lse ** 2).sum() / n
    gb, gz = (v.to(F64) for v in st["g"])
    u = gb * C / n * f[None, :] + (gz * 2.0 / n) * lse[:, None]
    # the softmax's gradient for the pool term, the log-sum-exp's for the other
    dp = gb * C / n * f[None, :]
    d = p * (u - (p * dp).sum(1, keepdim=True))
    dx = torch.zeros_like(x)
    dx[rows] = d
    return bal, z, counts.to(torch.int32), dx
