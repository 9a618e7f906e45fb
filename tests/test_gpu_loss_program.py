"""The token losses and the pool balance in one training program: a teacher's answers scored and their top alternatives
kept, a routed student that learns from them with its pools kept balanced, and a policy's log probabilities taken from
its hidden states.  Gradients against the same program with the losses written out in torch."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
V, B, S, K, TAU = 640, 4, 24, 16, 2.0


@pytest.fixture(scope="module")
def H():
    from rte_amd.kernels import hip_ops

    return hip_ops


def model(seed, clusters=8):
    from rte_amd.config import ModelConfig
    from rte_amd.layers import ClusterPoolSwiGLU
    from rte_amd.models import DenseModel

    torch.manual_seed(seed)
    cfg = ModelConfig(topology="dense", vocab_size=V, d_model=128, n_heads=2, d_ff=32 * clusters, n_dense_layers=2,
                      n_prelude=1, n_coda=1, t_max=1, depth_choices=[1], attn_banks=1, ffn_banks=1, head_groups=1,
                      ffn_groups=1, active_head_groups=1, active_ffn_groups=1, recipe_count=2, ffn_kind="cluster_pool",
                      ffn_clusters=clusters, ffn_top_k=2)
    m = DenseModel(cfg).to(DEV)
    with torch.no_grad():
        for p in m.parameters():
            if p.ndim == 2:
                p.normal_(0.0, p.shape[1] ** -0.5)
    pools = [x for x in m.modules() if isinstance(x, ClusterPoolSwiGLU)]
    assert len(pools) == 2
    return m, pools


def data(seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    tokens = torch.randint(0, V, (B, S), device=DEV, generator=g)
    return tokens, torch.randint(0, V, (B, S), device=DEV, generator=g)


def plain_distill(logits, ids, tl):
    """tail True in torch: the list's terms and one for the rest."""
    lq = torch.log_softmax(logits.double() / TAU, -1)
    p = tl.double().exp()
    q = lq.gather(-1, ids.long())
    on = torch.zeros_like(lq, dtype=torch.bool).scatter_(-1, ids.long(), True)
    rest = 1 - p.sum(-1)
    lr = torch.logsumexp(lq.masked_fill(on, float("-inf")), -1)
    return ((p * (tl.double() - q)).sum(-1) + rest * (rest.log() - lr)) * TAU * TAU


def plain_balance(logits, ids):
    C = logits.shape[-1]
    z = logits.double().reshape(-1, C)
    counts = torch.bincount(ids.reshape(-1).long(), minlength=C).double()
    return (C * (torch.softmax(z, -1).mean(0) * counts / counts.sum()).sum(), torch.logsumexp(z, -1).square().mean())


def grads(loss, m):
    ps = [p for p in m.parameters() if p.requires_grad]
    return torch.autograd.grad(loss, ps, allow_unused=True)


@pytest.mark.parametrize("clusters", [8, 12])
def test_distilled_routed_student(H, clusters):
    teacher, _ = model(1, clusters)
    student, pools = model(2, clusters)
    tokens, targets = data(3)
    with torch.no_grad():
        t_logits = teacher(tokens, targets).logits
        _, _, tl, ids = H.token_logprobs(t_logits, targets, n_top=K, temperature=TAU)
    balances = []
    for pool in pools:
        pool.balance_into = balances

    def program(distill, balance):
        balances.clear()
        out = student(tokens, targets)
        loss = out.loss / S + distill(out.logits, ids, tl).mean()
        for i in range(len(pools)):
            bal, z = balance(i)
            loss = loss + 0.5 * bal + 0.01 * z
        return loss

    def framework(i):
        bal, z, counts = balances[i]
        assert len(balances) == 2 and int(counts.sum()) == B * S * 2
        return bal, z

    real = H.pool_balance
    loss = program(lambda x, i, t: H.topk_distill(x, i, t, temperature=TAU, tail=True), framework)
    got = grads(loss, student)
    rows = []
    H.pool_balance = lambda logits, i, **k: rows.append((logits, i)) or real(logits, i, **k)
    try:
        want_loss = program(plain_distill, lambda i: plain_balance(*rows[i]))
    finally:
        H.pool_balance = real
    want = grads(want_loss.float(), student)
    assert abs(float(loss.detach() - want_loss.detach())) < 1e-5 * abs(float(want_loss.detach()))
    # the models' own products round their gradients to bf16; equal logit gradients go through the same kernels, and
    # those here differ by 2^-20 of themselves, which moves a rounding now and then
    for a, b in zip(got, want):
        assert (a is None) == (b is None)
        if a is not None:
            assert float((a - b).norm()) <= 2.0 ** -8 * float(b.norm()) + 1e-9
    routers = [float(g.norm()) for g, (n, _) in zip(got, student.named_parameters()) if "router" in n]
    assert len(routers) == 2 and all(r > 0 for r in routers)


def test_policy_from_hidden_states(H):
    """Advantage-weighted log probabilities with an entropy bonus: from the stored logits and from hidden states."""
    m, _ = model(4)
    tokens, targets = data(5)
    targets[:, ::7] = -100
    adv = torch.randn(B, S, device=DEV, generator=torch.Generator(device=DEV).manual_seed(6))
    out = m(tokens)
    lp, ent, _, _ = H.token_logprobs(out.logits, targets)
    by_logits = grads(-(adv * lp).mean() - 0.01 * ent.mean(), m)
    out = m(tokens)
    lp2, ent2 = H.lm_head_logprobs(out.meta.hidden, m.vocab_weight, targets)
    by_hidden = grads(-(adv * lp2).mean() - 0.01 * ent2.mean(), m)
    assert float((lp - lp2).detach().abs().max()) < 1e-4 and float((ent - ent2).detach().abs().max()) < 1e-4
    # both round the logits' gradient to bf16 once, the head's products at other places
    for a, b in zip(by_logits, by_hidden):
        assert (a is None) == (b is None)
        if a is not None:
            assert float((a - b).norm()) <= 2.0 ** -6 * float(b.norm()) + 1e-9


def test_training_step_captured(H):
    """Teacher scoring, distillation, balance and their backward in one graph, replayed with new tokens."""
    teacher, _ = model(7)
    student, pools = model(8)
    tokens, targets = data(9)
    balances = []
    for pool in pools:
        pool.balance_into = balances

    def step(accumulate=False):
        with torch.no_grad():
            _, _, tl, ids = H.token_logprobs(teacher(tokens, targets).logits, targets, n_top=K)
        out = student(tokens, targets)
        loss = out.loss / S + H.topk_distill(out.logits, ids, tl).mean()
        for bal, z, _ in balances:
            loss = loss + 0.1 * bal + 0.01 * z
        balances.clear()
        ps = [p for p in student.parameters()]
        if not accumulate:
            return loss.detach(), [g for g in grads(loss, student) if g is not None]
        for p in ps:
            p.grad = None
        loss.backward()
        return loss.detach(), [p.grad for p in ps if p.grad is not None]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss, gs = step(accumulate=True)
    for i in range(4):
        a, b = data(10 + i)
        tokens.copy_(a)
        targets.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        have, hg = loss.clone(), [g.clone() for g in gs]
        want, wg = step()
        torch.cuda.synchronize()
        assert torch.equal(have, want), i
        for x, y in zip(hg, wg):
            assert torch.equal(x, y), i
