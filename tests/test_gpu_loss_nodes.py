"""The token losses and the pool balance as nodes of autograd graphs: results changed in place, gradients of
gradients, graphs used twice, inputs changed under a graph, modes without gradients, other streams, checkpoints."""

from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu

T, V, K, D = 37, 515, 5, 128


@pytest.fixture(scope="module")
def H():
    from rte_amd.kernels import hip_ops

    return hip_ops


def operands():
    g = torch.Generator().manual_seed(11)
    x = torch.randn((T, V), generator=g).cuda()
    tok = torch.randint(0, V, (T,), generator=g).cuda()
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(T)]).cuda()
    tl = torch.randn((T, K), generator=g).cuda()
    h = torch.randn((T, D), generator=g).bfloat16().cuda()
    w = (torch.randn((V, D), generator=g) * 0.1).bfloat16().cuda()
    return x, tok, ids, tl, h, w


def programs(H):
    """name -> (a leaf, the function of it whose results carry gradients)"""
    x, tok, ids, tl, h, w = operands()
    return {
        "token": (x, lambda a: H.token_logprobs(a, tok)[:2]),
        "distill": (x, lambda a: (H.topk_distill(a, ids, tl),)),
        "balance": (x, lambda a: H.pool_balance(a, ids)[:2]),
        "head": (h, lambda a: H.lm_head_logprobs(a, w, tok)),
        "head weights": (w, lambda a: H.lm_head_logprobs(h, a, tok)),
    }


NAMES = ["token", "distill", "balance", "head", "head weights"]


def grad(f, a, scale=1.0, **kw):
    a = a.detach().clone().requires_grad_()
    loss = sum(scale * r.sum() for r in f(a))
    return torch.autograd.grad(loss, a, **kw)[0]


@pytest.mark.parametrize("name", NAMES)
def test_results_changed_in_place(H, name):
    """A loss may be scaled in place: the gradient is the scaled one (by 2, exactly).  token_logprobs' and
    lm_head_logprobs' entropy is kept for their backward, so only the first result is changed."""
    a, f = programs(H)[name]
    leaf = a.clone().requires_grad_()
    r = f(leaf)
    first = r[0].mul_(2.0)
    got = torch.autograd.grad(first.sum(), leaf)[0]
    leaf2 = a.clone().requires_grad_()
    want = torch.autograd.grad(2.0 * f(leaf2)[0].sum(), leaf2)[0]
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", NAMES)
def test_gradient_of_gradient_refused(H, name):
    """create_graph gives the gradient, and an error where that gradient is differentiated."""
    a, f = programs(H)[name]
    want = grad(f, a)
    leaf = a.clone().requires_grad_()
    got = torch.autograd.grad(sum(r.sum() for r in f(leaf)), leaf, create_graph=True)[0]
    assert torch.equal(got, want)
    with pytest.raises(RuntimeError, match="cannot be differentiated|once_differentiable"):
        got.float().square().sum().backward()


@pytest.mark.parametrize("name", NAMES)
def test_graph_used_twice_and_released(H, name):
    a, f = programs(H)[name]
    leaf = a.clone().requires_grad_()
    loss = sum(r.sum() for r in f(leaf))
    one = torch.autograd.grad(loss, leaf, retain_graph=True)[0]
    two = torch.autograd.grad(loss, leaf)[0]
    assert torch.equal(one, two)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, leaf)


@pytest.mark.parametrize("name", NAMES)
def test_operand_changed_under_a_graph(H, name):
    a, f = programs(H)[name]
    leaf = a.clone().requires_grad_()
    mid = leaf * 1.0
    loss = sum(r.sum() for r in f(mid))
    with torch.no_grad():
        mid.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("name", NAMES)
def test_without_gradients(H, name):
    a, f = programs(H)[name]
    want = [r.detach() for r in f(a.clone().requires_grad_())]
    with torch.no_grad():
        off = f(a.clone().requires_grad_())
    with torch.inference_mode():
        inf = [r.clone() for r in f(a)]
    plain = f(a)
    for r in (off, inf, plain):
        assert all(torch.equal(p, q) and not p.requires_grad for p, q in zip(r, want))


@pytest.mark.parametrize("name", NAMES)
def test_backward_called_from_another_stream(H, name):
    a, f = programs(H)[name]
    want = grad(f, a)
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaf = a.detach().clone().requires_grad_()
        loss = sum(r.sum() for r in f(leaf))
    other.wait_stream(side)
    with torch.cuda.stream(other):
        got = torch.autograd.grad(loss, leaf)[0]
    torch.cuda.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("name", NAMES)
def test_checkpointed(H, name):
    a, f = programs(H)[name]
    want = grad(f, a)
    got = grad(lambda x: checkpoint(f, x, use_reentrant=False), a)
    assert torch.equal(got, want)


def test_errors_of_the_entry_points_reach_the_caller(H):
    """A refusal of the C entry is an ordinary error: a list of 129 entries, handed past the wrapper's check."""
    from rte_amd import _lib

    x, _, _, _, _, _ = operands()
    ids = torch.zeros((T, 129), dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="rte_topk_distill_fwd failed"):
        _lib.ops().topk_distill(x, ids, ids.float(), 1.0, False, _lib.stream_ptr(x.device))


def test_more_pools_per_row_than_there_can_be_are_refused(H):
    x = torch.randn(3, 8, device="cuda")
    with pytest.raises(ValueError, match="pool_balance"):
        H.pool_balance(x, torch.zeros((3, 1025), dtype=torch.int32, device="cuda"))
    _, _, counts = H.pool_balance(x, torch.zeros((3, 1024), dtype=torch.int32, device="cuda"))
    assert counts.tolist() == [3 * 1024] + [0] * 7


def test_operands_that_do_not_match_are_refused_by_the_nodes(H):
    from rte_amd import _lib

    ops = _lib.ops()
    x, tok, ids, tl, h, w = operands()
    s = _lib.stream_ptr(x.device)
    bad = [lambda: ops.token_logprobs(x, tok[1:], 0, 1.0, s), lambda: ops.token_logprobs(x, tok.cpu(), 0, 1.0, s),
           lambda: ops.token_logprobs(x.half(), tok, 0, 1.0, s), lambda: ops.token_logprobs(x, tok, -1, 1.0, s),
           lambda: ops.topk_distill(x, ids[1:], tl, 1.0, False, s), lambda: ops.topk_distill(x, ids, tl[:, 1:], 1.0, False, s),
           lambda: ops.pool_balance(x, ids[1:], None, s), lambda: ops.pool_balance(x, ids, tok, s),
           lambda: ops.lm_head_logprobs(h, w, h, w[:, :64], tok, 1.0, 1 << 20, s),
           lambda: ops.lm_head_logprobs(h, w, h.float(), w, tok, 1.0, 1 << 20, s),
           lambda: ops.lm_head_logprobs(h, w, h, w, tok[1:], 1.0, 1 << 20, s)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
