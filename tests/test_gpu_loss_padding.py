"""Padding whose logits hold NaN or infinities: a negative token gives log probability 0 and no gradient, whatever its row
holds, and other rows are as without it."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 700, 2049, 9001, 140001])
@pytest.mark.parametrize("entropy", [False, True])
def test_padded_rows_of_anything(V, dtype, entropy):
    from rte_amd.kernels import hip_ops as H

    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(9, V, device="cuda", generator=g).to(dtype)
    tok = torch.randint(0, V, (9,), device="cuda", generator=g)
    pad = torch.tensor([1, 4, 5, 6], device="cuda")
    tok[pad] = torch.tensor([-1, -100, -1, -1], device="cuda")

    def program(rows):
        leaf = rows.clone().requires_grad_()
        lp, ent, _, _ = H.token_logprobs(leaf, tok)
        loss = lp.sum()
        if entropy:  # padding left out, by values and not by a product with 0
            loss = loss + torch.where(tok >= 0, ent, 0.0).sum()
        return lp.detach(), torch.autograd.grad(loss, leaf)[0]

    want_lp, want = program(x)
    bad = x.clone()
    bad[1] = math.nan
    bad[4, V // 2] = math.nan
    bad[5, 0] = math.inf
    bad[6] = math.inf
    lp, dx = program(bad)
    assert torch.equal(lp, want_lp) and torch.equal(dx, want)
    assert not lp[pad].any() and not dx[pad].any()
