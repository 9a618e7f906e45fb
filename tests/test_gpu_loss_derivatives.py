"""The token losses and the pool balance under forward-mode differentiation: refused by each, with and without a graph."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("name", ["token", "distill", "distill teacher", "balance", "head", "head weights"])
def test_forward_mode_is_refused(name, graph):
    from rte_amd.kernels import hip_ops as H

    x, tok = torch.randn(6, 40, device="cuda"), torch.zeros(6, dtype=torch.long, device="cuda")
    ids, tl = torch.zeros(6, 2, dtype=torch.long, device="cuda"), torch.randn(6, 2, device="cuda")
    h, w = torch.randn(6, 128, device="cuda"), torch.randn(40, 128, device="cuda")
    f, a = {"token": (lambda v: H.token_logprobs(v, tok, n_top=3), x),
            "distill": (lambda v: H.topk_distill(v, ids, tl), x),
            "distill teacher": (lambda v: H.topk_distill(x, ids, v), tl),
            "balance": (lambda v: H.pool_balance(v, ids), x),
            "head": (lambda v: H.lm_head_logprobs(v, w, tok), h),
            "head weights": (lambda v: H.lm_head_logprobs(h, v, tok), w)}[name]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(a.clone().requires_grad_(graph), torch.ones_like(a))
        with pytest.raises((RuntimeError, NotImplementedError)):
            f(dual)
    f(a)  # and nothing of it stays
