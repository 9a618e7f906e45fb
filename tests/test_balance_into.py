"""ClusterPoolSwiGLU.balance_into: which forward passes leave an entry.  The kernels are replaced by torch, so this runs
without a device."""

from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

from rte_amd import layers
from rte_amd.config import ModelConfig


@pytest.fixture
def layer(monkeypatch):
    def routed(x, wr, wug, wd, k, resid=None):
        w, ids = torch.topk(x @ wr.t(), k, dim=-1)
        return x * torch.sigmoid(w.sum(-1, keepdim=True)), ids.reshape(-1, k), w

    def balance(self, x, ids, mask=None):
        p = torch.softmax(x @ self.router.weight.t(), -1)
        return p.square().mean(), p.mean(), torch.bincount(ids.reshape(-1), minlength=self.n_clusters)

    monkeypatch.setattr(layers.hip_ops, "routed_cluster_pool_swiglu", routed)
    monkeypatch.setattr(layers.ClusterPoolSwiGLU, "balance", balance)
    torch.manual_seed(0)
    cfg = ModelConfig(topology="dense", vocab_size=32, d_model=16, n_heads=2, d_ff=128, n_dense_layers=2, n_prelude=1,
                      n_coda=1, t_max=1, depth_choices=[1], attn_banks=1, ffn_banks=1, head_groups=1, ffn_groups=1,
                      active_head_groups=1, active_ffn_groups=1, recipe_count=2, ffn_kind="cluster_pool", ffn_clusters=4,
                      ffn_top_k=2)
    pool = layers.ClusterPoolSwiGLU(cfg)
    with torch.no_grad():
        pool.router.weight.normal_()
    pool.balance_into = []
    return pool


def run(pool, x, call):
    """Gradients of a program that weighs the entries into its loss."""
    pool.balance_into.clear()
    y = call(x)
    loss = y.sum() + sum(b + 0.1 * z for b, z, _ in pool.balance_into)
    n = len(pool.balance_into)
    got = torch.autograd.grad(loss, (x, pool.router.weight))
    assert len(pool.balance_into) == n == 1
    return got


def test_one_entry_per_recorded_pass(layer):
    x = torch.randn(5, 16, requires_grad=True)
    layer(x)
    layer(x)
    assert len(layer.balance_into) == 2 and all(b.requires_grad for b, _, _ in layer.balance_into)


def test_a_checkpoint_s_recomputation_leaves_none(layer):
    x = torch.randn(5, 16, requires_grad=True)
    want = run(layer, x, layer)
    got = run(layer, x, lambda v: checkpoint(layer, v, use_reentrant=False))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    both = torch.nn.Sequential(layer, torch.nn.Linear(16, 16))
    run(layer, x, lambda v: checkpoint(both, v, use_reentrant=False))


def test_passes_without_gradients_leave_none(layer):
    x = torch.randn(5, 16)
    with torch.no_grad():
        layer(x)
    with torch.inference_mode():
        layer(x)
    assert layer.balance_into == []
    assert layer.last_ids is not None
