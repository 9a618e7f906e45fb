"""Forward-mode derivatives of the token losses are refused, not left out: the registered operators say so before they
look at anything else, so this runs without a device."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from rte_amd import _lib


@pytest.mark.parametrize("mode", ["plain", "no_grad"])
def test_dual_tensors_are_refused(mode):
    ops = _lib.ops()
    x, tok, ids = torch.randn(4, 8), torch.zeros(4, dtype=torch.long), torch.zeros(4, 2, dtype=torch.int32)
    tl = torch.zeros(4, 2)
    with forward_ad.dual_level(), torch.no_grad() if mode == "no_grad" else torch.enable_grad():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        teacher = forward_ad.make_dual(tl, torch.ones_like(tl))
        for call in (lambda: ops.token_logprobs(dual, tok, 0, 1.0, 0), lambda: ops.topk_distill(dual, ids, tl, 1.0, False, 0),
                     lambda: ops.topk_distill(x, ids, teacher, 1.0, False, 0)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
