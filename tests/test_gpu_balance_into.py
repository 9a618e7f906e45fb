"""A routed layer that leaves its balance losses while it is checkpointed: one entry, and the gradients of a program without."""

from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu


def test_checkpointed_layer():
    from rte_amd.config import ModelConfig
    from rte_amd.layers import ClusterPoolSwiGLU

    cfg = ModelConfig(topology="dense", vocab_size=32, d_model=128, n_heads=2, d_ff=256, n_dense_layers=2, n_prelude=1,
                      n_coda=1, t_max=1, depth_choices=[1], attn_banks=1, ffn_banks=1, head_groups=1, ffn_groups=1,
                      active_head_groups=1, active_ffn_groups=1, recipe_count=2, ffn_kind="cluster_pool", ffn_clusters=8,
                      ffn_top_k=2)
    torch.manual_seed(0)
    pool = ClusterPoolSwiGLU(cfg).cuda()
    with torch.no_grad():
        for p in pool.parameters():
            p.normal_(0.0, p.shape[1] ** -0.5)
    x = torch.randn(2, 40, 128, device="cuda", requires_grad=True)
    pool.balance_into = []

    def program(call):
        pool.balance_into.clear()
        y = call(x)
        (bal, z, counts), = pool.balance_into
        loss = y.float().square().mean() + 0.5 * bal + 0.1 * z
        got = torch.autograd.grad(loss, (x, *pool.parameters()))
        assert len(pool.balance_into) == 1 and int(counts.sum()) == 160
        return got

    want = program(pool)
    got = program(lambda v: checkpoint(pool, v, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
