"""The C entries of the token losses and the pool balance refuse what they cannot compute, without a device: sizes,
limits, missing pointers and short workspaces are looked at before anything is launched."""

from __future__ import annotations

import pytest

BUF = 1 << 20  # stands for a device pointer: a refused call never reads it


@pytest.fixture(scope="module")
def lib():
    from rte_amd import _lib

    return _lib.load()


def refused(lib, name, *args):
    assert getattr(lib, name)(*args) != 0, args
    assert lib.rte_last_error()


def test_token_logprobs(lib):
    def fwd(x=BUF, ld=64, T=4, V=64, tok=BUF, t=1.0, n=8, lp=BUF, ent=BUF, tl=BUF, ti=BUF, ws=BUF, wsn=1 << 40):
        refused(lib, "rte_token_logprobs_fwd", x, ld, 1, T, V, tok, t, n, lp, ent, tl, ti, BUF, ws, wsn, None)

    fwd(T=-1), fwd(V=0), fwd(ld=-1), fwd(n=-1), fwd(n=129, V=1000), fwd(n=65), fwd(t=0.0), fwd(t=float("nan"))
    fwd(t=float("inf")), fwd(x=None), fwd(tok=None), fwd(lp=None), fwd(ent=None), fwd(tl=None), fwd(ti=None)
    fwd(V=100000, wsn=lib.rte_token_logprobs_workspace_bytes(4, 100000, 8) - 1), fwd(V=100000, ws=None)
    fwd(T=(1 << 31) - 1, V=1 << 20)
    for a in ((None, 64, 1, 4, 64, BUF, 1.0, BUF, BUF, BUF, BUF, BUF), (BUF, 64, 1, 4, 64, BUF, 1.0, None, BUF, BUF, BUF, BUF),
              (BUF, 64, 1, 4, 64, BUF, -1.0, BUF, BUF, BUF, BUF, BUF), (BUF, 64, 1, 4, 0, BUF, 1.0, BUF, BUF, BUF, BUF, BUF),
              (BUF, 64, 1, 4, 64, BUF, 1.0, BUF, BUF, BUF, BUF, None)):
        refused(lib, "rte_token_logprobs_bwd", *a, None)
    assert lib.rte_token_logprobs_fwd(None, 64, 1, 0, 64, None, 1.0, 0, None, None, None, None, None, None, 0, None) == 0
    assert lib.rte_token_logprobs_bwd(None, 64, 1, 0, 64, None, 1.0, None, None, None, None, None, None) == 0


def test_lm_head_logprobs(lib):
    ok = lib.rte_lm_head_logprobs_ok
    assert ok(1, 128, 1) and ok(8192, 1024, 32768)
    assert not any(ok(*a) for a in ((0, 128, 10), (10, 128, 0), (10, 64, 10), (10, 160, 10), (1 << 23, 128, 10), (10, 128, 1 << 23)))
    need = lib.rte_lm_head_logprobs_workspace_bytes(100, 1000)

    def fwd(h=BUF, w=BUF, T=100, d=128, V=1000, tok=BUF, t=1.0, lp=BUF, ent=BUF, st=BUF, ws=BUF, wsn=need):
        refused(lib, "rte_lm_head_logprobs_fwd", h, w, T, d, V, tok, t, lp, ent, st, ws, wsn, None)

    fwd(d=100), fwd(T=0), fwd(V=0), fwd(t=0.0), fwd(t=float("nan")), fwd(h=None), fwd(w=None), fwd(tok=None), fwd(lp=None)
    fwd(ent=None), fwd(st=None), fwd(ws=None), fwd(wsn=need - 1), fwd(h=BUF + 2), fwd(w=BUF + 8)
    size = lib.rte_lm_head_logprobs_bwd_workspace_bytes
    room = size(100, 128, 1000, 256, 1, 1)
    assert room > 2 * 100 * 256 and size(100, 128, 1000, 100, 1, 1) == 0 and size(100, 100, 1000, 256, 1, 1) == 0

    def bwd(h=BUF, w=BUF, T=100, d=128, V=1000, tok=BUF, t=1.0, st=BUF, ent=BUF, width=256, dh=BUF, dw=BUF, ws=BUF, wsn=room):
        refused(lib, "rte_lm_head_logprobs_bwd", h, w, T, d, V, tok, t, st, ent, BUF, BUF, width, dh, dw, 0, ws, wsn, None)

    bwd(width=0), bwd(width=100), bwd(d=100), bwd(t=-1.0), bwd(st=None), bwd(ent=None), bwd(dh=BUF + 2), bwd(dw=BUF + 4)
    bwd(ws=None), bwd(wsn=room - 1), bwd(tok=None), bwd(h=None), bwd(w=None), bwd(T=0)
    bwd(T=1 << 22, V=1 << 20, width=1 << 20, wsn=1 << 50)
    assert lib.rte_lm_head_logprobs_bwd(BUF, BUF, 100, 128, 1000, BUF, 1.0, BUF, BUF, None, None, 64, None, None, 0, None, 0,
                                        None) == 0  # nothing wanted


def test_topk_distill(lib):
    def fwd(x=BUF, ld=64, T=4, V=64, ids=BUF, tl=BUF, K=8, t=1.0, loss=BUF, cols=BUF, coef=BUF, ws=BUF,
            wsn=1 << 40):
        refused(lib, "rte_topk_distill_fwd", x, ld, 1, T, V, ids, tl, K, t, 0, loss, BUF, cols, coef, ws, wsn, None)

    fwd(T=-1), fwd(V=0), fwd(ld=-1), fwd(K=0), fwd(K=129), fwd(t=0.0), fwd(t=float("nan")), fwd(t=float("inf"))
    fwd(x=None), fwd(ids=None), fwd(tl=None), fwd(loss=None), fwd(cols=None), fwd(coef=None)
    fwd(V=100000, wsn=lib.rte_topk_distill_workspace_bytes(4, 100000, 8) - 1), fwd(V=100000, ws=None)
    fwd(T=(1 << 31) - 1, V=1 << 20)
    for a in ((BUF, 64, 1, 4, 64, 0, 1.0, BUF, BUF, BUF, BUF, BUF), (BUF, 64, 1, 4, 64, 8, 0.0, BUF, BUF, BUF, BUF, BUF),
              (BUF, 64, 1, 4, 64, 8, 1.0, None, BUF, BUF, BUF, BUF), (BUF, 64, 1, 4, 64, 8, 1.0, BUF, BUF, BUF, None, BUF)):
        refused(lib, "rte_topk_distill_bwd", *a, None)
    assert lib.rte_topk_distill_fwd(None, 64, 1, 0, 64, None, None, 8, 1.0, 0, None, None, None, None, None, 0, None) == 0


def test_pool_balance(lib):
    need = lib.rte_pool_balance_workspace_bytes(1000, 64)
    assert need > 0 and lib.rte_pool_balance_workspace_bytes(0, 64) == 0

    def fwd(x=BUF, ld=64, T=1000, C=64, ids=BUF, k=8, out=BUF, cnt=BUF, frac=BUF, ws=BUF, wsn=need):
        refused(lib, "rte_pool_balance_fwd", x, ld, 1, T, C, ids, k, None, out, cnt, frac, ws, wsn, None)

    fwd(T=1 << 28, k=8, wsn=1 << 40)
    fwd(T=-1), fwd(C=0), fwd(C=1025), fwd(k=0), fwd(ld=-1), fwd(x=None), fwd(ids=None), fwd(out=None), fwd(cnt=None)
    fwd(frac=None), fwd(ws=None), fwd(wsn=need - 1)
    refused(lib, "rte_pool_balance_bwd", BUF, 64, 1, 4, 1025, None, BUF, None, None, BUF, None)
    refused(lib, "rte_pool_balance_bwd", BUF, 64, 1, 4, 64, None, None, None, None, BUF, None)
    assert lib.rte_pool_balance_bwd(None, 64, 1, 0, 64, None, None, None, None, None, None) == 0


def test_pool_balance_lists_of_at_most_the_largest_pool_count(lib):
    need = lib.rte_pool_balance_workspace_bytes(16, 64)
    refused(lib, "rte_pool_balance_fwd", BUF, 64, 1, 16, 64, BUF, 1025, None, BUF, BUF, BUF, BUF, need, None)
    refused(lib, "rte_pool_balance_fwd", BUF, 64, 1, 16, 64, BUF, (1 << 27) - 1, None, BUF, BUF, BUF, BUF, need, None)


def test_the_nodes_refuse_what_a_kernel_could_not_survive():
    """The registered operators, called past their Python wrappers: operands off the device, for one."""
    import torch

    from rte_amd import _lib

    ops = _lib.ops()
    x, tok, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.long), torch.zeros(4, 2, dtype=torch.int32)
    for needs in (False, True):
        leaf = x.clone().requires_grad_(needs)
        for call in (lambda: ops.token_logprobs(leaf, tok, 0, 1.0, 0), lambda: ops.topk_distill(leaf, ids, ids.float(), 1.0, False, 0),
                     lambda: ops.pool_balance(leaf, ids, None, 0),
                     lambda: ops.lm_head_logprobs(leaf, leaf, leaf.detach().bfloat16(), leaf.detach().bfloat16(), tok, 1.0, 1 << 20, 0)):
            with pytest.raises(RuntimeError, match="device tensors"):
                call()
