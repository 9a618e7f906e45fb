"""The token losses and the pool balance in a compiled program: results and gradients as without."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["token", "distill", "balance", "head", "head of a narrow width"])
def test_compiled_program(name):
    from rte_amd.kernels import hip_ops as H

    torch._dynamo.reset()
    g = torch.Generator().manual_seed(3)
    x, tok = torch.randn((64, 512), generator=g).cuda(), torch.randint(0, 512, (64,), generator=g).cuda()
    ids, tl = torch.randint(0, 512, (64, 8), generator=g).cuda(), torch.randn((64, 8), generator=g).cuda()
    h, w = torch.randn((64, 128), generator=g).cuda(), torch.randn((512, 128), generator=g).cuda()
    f, a = {"token": (lambda v: 2 * sum(H.token_logprobs(v * 2, tok, n_top=3)[:2]), x),
            "distill": (lambda v: 2 * H.topk_distill(v * 2, ids, tl), x),
            "balance": (lambda v: 2 * sum(H.pool_balance(v * 2, ids)[:2]), x),
            "head": (lambda v: 2 * sum(H.lm_head_logprobs(v * 2, w, tok)), h),
            "head of a narrow width": (lambda v: 2 * sum(H.lm_head_logprobs(v * 2, w[:, :64], tok)), h[:, :64])}[name]

    def both(fn):
        leaf = a.clone().requires_grad_()
        r = fn(leaf)
        return r.detach(), torch.autograd.grad(r.sum(), leaf)[0]

    want, got = both(f), both(torch.compile(f, backend="eager"))
    assert all(torch.equal(p, q) for p, q in zip(got, want))
