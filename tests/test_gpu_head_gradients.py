"""lm_head_logprobs: the types of its gradients, and what its backward allocates."""

from __future__ import annotations

import math
import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
F64 = torch.float64


@pytest.fixture(scope="module")
def H():
    from rte_amd.kernels import hip_ops

    return hip_ops


def gen(*seed):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(seed).encode()))


def dlogits64(hb, wb, tok, g):
    """The logits' gradient of sum g log p in 64 bits, [T, V]."""
    p = torch.softmax(hb.to(F64) @ wb.to(F64).t(), 1)
    return (torch.zeros_like(p).scatter_(1, tok[:, None], 1.0) - p) * g.to(F64)[:, None]


@pytest.mark.parametrize("T,d,V,grad", [(96, 128, 1024, None), (300, 256, 1000, None), (100, 192, 1096, 2 * 100 * 300),
                                        (70, 64, 515, None), (2100, 64, 129, None)])
def test_gradient_of_fp32_hidden_states_is_not_rounded(H, T, d, V, grad, monkeypatch):
    """The logits' gradient is rounded to bf16 for the two products; what they sum to in fp32 is the gradient of fp32
    operands.  A rounded result is told by its bits: one fp32 sum in 2^16 is a bf16 number by chance."""
    g = gen(T, d, V)
    if grad is not None:
        monkeypatch.setattr(H.LMHeadLogprobsFn, "GRAD", grad)
    h = torch.randn(T, d, device=DEV, generator=g)
    w = torch.randn(V, d, device=DEV, generator=g) * (2 / math.sqrt(d))
    tok = torch.randint(0, V, (T,), device=DEV, generator=g)
    up = torch.randn(T, device=DEV, generator=g)
    h.requires_grad_(), w.requires_grad_()
    dh, dw = torch.autograd.grad(H.lm_head_logprobs(h, w, tok)[0], (h, w), up)
    assert dh.dtype == dw.dtype == torch.float32
    for got in (dh, dw):
        assert float((got.bfloat16().float() == got).float().mean()) < 0.01
    hb, wb = h.detach().bfloat16(), w.detach().bfloat16()
    d64 = dlogits64(hb, wb, tok, up)
    # each logit's gradient: half a step of bf16, and the logits' own fp32 sums (d 2^-24 of the absolute products)
    za = float((hb.to(F64).abs() @ wb.to(F64).abs().t()).max())
    c = 2.0 ** -24 * (V / 256 + 16 + 8 * za + 2 * d * za)
    size = torch.softmax(hb.to(F64) @ wb.to(F64).t(), 1) * up.to(F64).abs()[:, None]
    size.scatter_add_(1, tok[:, None], up.to(F64).abs()[:, None])
    dl = 1.01 * 2.0 ** -8 * d64.abs() + 4.1 * c * size
    # and the products' own sums in fp32
    sums = 2.0 ** -24 * V * (d64.abs() @ wb.to(F64).abs())
    assert bool(((dh.to(F64) - d64 @ wb.to(F64)).abs() <= dl @ wb.to(F64).abs() + sums + 1e-35).all())


def test_gradients_keep_their_operands_types(H):
    g = gen(2)
    T, d, V = 40, 128, 200
    tok = torch.randint(0, V, (T,), device=DEV, generator=g)
    for dd in (d, 64):
        for th in (torch.float32, torch.bfloat16):
            for tw in (torch.float32, torch.bfloat16):
                h = torch.randn(T, dd, device=DEV, generator=g).to(th).requires_grad_()
                w = (torch.randn(V, dd, device=DEV, generator=g) * 0.2).to(tw).requires_grad_()
                dh, dw = torch.autograd.grad(H.lm_head_logprobs(h, w, tok)[0].sum(), (h, w))
                assert dh.dtype == th and dw.dtype == tw
                # bf16 gradients are the fp32 ones rounded once
                h32, w32 = h.detach().float().requires_grad_(), w.detach().float().requires_grad_()
                dh32, dw32 = torch.autograd.grad(H.lm_head_logprobs(h32, w32, tok)[0].sum(), (h32, w32))
                assert torch.equal(dh, dh32.to(th)) and torch.equal(dw, dw32.to(tw))


@pytest.mark.parametrize("want", ["hidden", "weights"])
def test_nothing_is_allocated_for_a_gradient_that_is_not_wanted(H, want):
    """Widths that the tile product does not take: a frozen head of 300000 x 64 has no fp32 gradient of 77 MB, and frozen
    hidden states of 150000 x 64 none of 19 MB in bf16."""
    g = gen(want, 3)
    T, d, V = (8, 64, 300000) if want == "hidden" else (150000, 64, 8)
    h = torch.randn(T, d, device=DEV, generator=g).bfloat16().requires_grad_(want == "hidden")
    w = (torch.randn(V, d, device=DEV, generator=g) * 0.2).bfloat16().requires_grad_(want == "weights")
    tok = torch.randint(0, V, (T,), device=DEV, generator=g)
    lp, _ = H.lm_head_logprobs(h, w, tok)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    lp.sum().backward()
    torch.cuda.synchronize()
    peak = torch.cuda.max_memory_allocated() - before
    # three of the logits' size (8 x 300000 or 2048 x 8 in fp32, twice, and bf16) beside products' workspaces
    logits = min(T, 2048) * V * 4
    assert (h if want == "hidden" else w).grad is not None
    assert peak < 3 * logits + (1 << 23 if want == "weights" else 1 << 24), peak


def test_backward_of_narrow_widths_runs_on_the_framework_s_kernels(H):
    """Sums over blocks of rows and roundings to bf16 are the products' and the cast's own; torch converts and adds
    nothing."""
    from torch.profiler import ProfilerActivity, profile

    g = gen(4)
    T, d, V = 4500, 64, 136
    h = torch.randn(T, d, device=DEV, generator=g).bfloat16().requires_grad_()
    w = (torch.randn(V, d, device=DEV, generator=g) * 0.2).bfloat16().requires_grad_()
    tok = torch.randint(0, V, (T,), device=DEV, generator=g)
    up = torch.randn(T, device=DEV, generator=g)
    lp, _ = H.lm_head_logprobs(h, w, tok)
    with profile(activities=[ProfilerActivity.CPU]) as prof:
        torch.autograd.grad(lp, (h, w), up)
    torch.cuda.synchronize()
    names = {e.key for e in prof.key_averages()}
    assert "aten::empty" in names  # the backward's thread is seen
    assert not names & {"aten::_to_copy", "aten::copy_", "aten::add_", "aten::add"}, names
