"""A program under torch.compile runs the losses' nodes as they are, between its graphs: without a device, the node's own
refusal arrives, not one of a tracer."""

from __future__ import annotations

import pytest
import torch

from rte_amd import _lib


def test_nodes_are_not_traced():
    tok, ids = torch.zeros(4, dtype=torch.long), torch.zeros(4, 2, dtype=torch.int32)
    x = torch.randn(4, 8, requires_grad=True)
    for f in (lambda v: _lib.ops().token_logprobs(v * 2, tok, 0, 1.0, 0)[0] + 1,
              lambda v: _lib.ops().topk_distill(v * 2, ids, torch.zeros(4, 2), 1.0, False, 0) + 1,
              lambda v: _lib.ops().pool_balance(v * 2, ids, None, 0)[0] + 1,
              lambda v: _lib.ops().lm_head_logprobs(v * 2, v, v.bfloat16(), v.bfloat16(), tok, 1.0, 1 << 20, 0)[0] + 1):
        with pytest.raises(RuntimeError, match="expects ROCm device tensors") as refusal:
            torch.compile(f, backend="eager")(x)
        assert type(refusal.value) is RuntimeError, "a tracer's"
