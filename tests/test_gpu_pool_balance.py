"""Load balance of routed pools against its definition in 64 bits.  A softmax in fp32 is right to
2^-24 (C / 16 + 16 + 4 max |u|) of each value (at least sixteen partial sums per row), sums over rows are made of
partials of at most 256 rows and a 64-bit sum of those: 2^-24 times 256 more."""

from __future__ import annotations

import math
import zlib

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
F64 = torch.float64
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def H():
    from rte_amd.kernels import hip_ops

    return hip_ops


def gen(*seed):
    return torch.Generator(device=DEV).manual_seed(zlib.crc32(repr(seed).encode()))


def want64(x, ids, mask, gb, gz):
    T, C = x.shape
    keep = (x > -math.inf).any(1) | torch.isnan(x).any(1)
    if mask is not None:
        keep &= mask
    rows = keep.nonzero()[:, 0]
    n = max(1, rows.numel())
    sel = ids[rows].reshape(-1)
    counts = torch.bincount(sel[(sel >= 0) & (sel < C)].long(), minlength=C)
    f = counts.to(F64) / max(1, int(counts.sum()))
    z = x[rows].to(F64)
    p = torch.softmax(z, 1)
    lse = torch.logsumexp(z, 1)
    bal, zl = C * (p.sum(0) @ f) / n, (lse ** 2).sum() / n
    dot = (p * f).sum(1, keepdim=True)
    dx = torch.zeros(T, C, dtype=F64, device=x.device)
    dx[rows] = p * (gb * C * (f - dot) + 2 * gz * lse[:, None]) / n
    scale = torch.zeros_like(dx)
    scale[rows] = p * (abs(gb) * C * (f + dot) + 2 * abs(gz) * lse.abs()[:, None]) / n
    return bal, zl, counts, dx, scale, lse


def check(H, x, ids, mask=None, gb=0.7, gz=0.3):
    C = x.shape[1]
    leaf = x.detach().requires_grad_()
    bal, z, counts = H.pool_balance(leaf, ids, mask=mask)
    (dx,) = torch.autograd.grad((bal, z), leaf, (torch.tensor(gb, device=DEV), torch.tensor(gz, device=DEV)))
    torch.cuda.synchronize()
    bal, z = bal.detach(), z.detach()
    wb, wz, wc, wd, scale, lse = want64(x.detach(), ids.long(), mask, gb, gz)
    assert counts.dtype == torch.int32 and torch.equal(counts.long(), wc)
    fin = torch.isfinite(x.detach())
    u = float(x.detach()[fin].double().max() - x.detach()[fin].double().min()) if bool(fin.any()) else 0.0
    c = 2.0 ** -24 * (C / 16 + 16 + 4 * min(u, 100.0))
    t = c + 2.0 ** -24 * 256
    lmax = float(lse.abs().max()) if lse.numel() else 0.0
    assert abs(float(bal) - float(wb)) <= t * float(wb) + 1e-30
    # a row at fp32's lowest value has lse^2 = 1.2e77: z, a number of 32 bits, is then infinite
    assert float(z) == math.inf if float(wz) > 3.5e38 else abs(float(z) - float(wz)) <= 2 * t * (float(wz) + lmax + 1e-30)
    err = (dx.to(F64) - wd).abs() - ((4 * c + HALF[x.dtype]) * scale + 2 * c * lmax / max(1, x.shape[0]) * gz + 1e-37)
    assert dx.dtype == x.dtype and bool(torch.isfinite(dx).all()) and (err.numel() == 0 or float(err.max()) <= 0), float(err.max())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("T,C,k", [(1, 1, 1), (1, 16, 4), (3, 7, 2), (127, 64, 8), (128, 64, 8), (129, 32, 4), (1000, 48, 3),
                                   (257, 65, 1), (300, 100, 16), (513, 128, 2), (4097, 256, 16), (77, 257, 5),
                                   (200, 512, 8), (65, 1000, 10), (130, 1024, 16), (20001, 64, 8)])
def test_sizes(H, T, C, k, masked, dtype):
    g = gen(T, C, k, masked, dtype, 1)
    x = (torch.randn(T, C, device=DEV, generator=g) * 2 + torch.randn(C, device=DEV, generator=g)).to(DT[dtype])
    ids, _ = H.route_topk(x.float(), min(k, C))
    mask = torch.rand(T, device=DEV, generator=g) < 0.7 if masked else None
    check(H, x, ids, mask)


def test_awkward_rows(H):
    """Masked rows of NaN and infinities, rows without a possible pool, disabled pools, the lowest value as a mask,
    missing and foreign ids, a pool named twice, ids of 64 bits that do not fit."""
    g = gen(2)
    T, C, k = 300, 40, 4
    x = torch.randn(T, C, device=DEV, generator=g)
    x[:, 5] = -math.inf
    x[:, 6] = torch.finfo(torch.float32).min
    x[10] = -math.inf
    x[11] = torch.finfo(torch.float32).min
    ids = torch.topk(x, k, dim=1).indices
    ids[20, 1:] = -1
    ids[21] = C
    ids[22] = 3
    ids[23, 0] = (1 << 33) + 2
    mask = torch.ones(T, dtype=torch.bool, device=DEV)
    mask[100:140] = False
    x[100] = math.nan
    x[101] = math.inf
    x[102, 3] = math.nan
    check(H, x, ids, mask)
    check(H, x[103:], ids[103:].int())


def test_nothing_left(H):
    """No rows, every row masked, no row with a possible pool: losses 0, counts 0, gradient 0."""
    for x, mask in ((torch.zeros(0, 8, device=DEV), None), (torch.ones(5, 8, device=DEV), torch.zeros(5, dtype=torch.bool, device=DEV)),
                    (torch.full((5, 8), -math.inf, device=DEV), None)):
        leaf = x.requires_grad_()
        ids = torch.zeros(x.shape[0], 2, dtype=torch.int32, device=DEV)
        bal, z, counts = H.pool_balance(leaf, ids, mask=mask)
        (dx,) = torch.autograd.grad(bal + z, leaf)
        assert float(bal.detach()) == 0 and float(z.detach()) == 0 and not counts.any() and not dx.any() and dx.shape == x.shape


def test_nan_is_seen(H):
    x = torch.randn(64, 32, device=DEV)
    x[7, 3] = math.nan
    bal, z, _ = H.pool_balance(x, torch.zeros(64, 1, dtype=torch.int32, device=DEV))
    assert math.isnan(float(bal)) and math.isnan(float(z))


def test_strides_and_forms(H):
    g = gen(3)
    wide = torch.randn(2, 50, 70, device=DEV, generator=g)
    x = wide[..., 3:67]
    ids = torch.randint(0, 64, (2, 50, 3), device=DEV, generator=g)
    mask = torch.rand(2, 50, device=DEV, generator=g) < 0.5
    leaf = x.detach().requires_grad_()
    bal, z, counts = H.pool_balance(leaf, ids, mask=mask)
    (dx,) = torch.autograd.grad(bal, leaf)
    wb, wz, wc, wd, _, _ = want64(x.reshape(100, 64), ids.reshape(100, 3), mask.reshape(100), 1.0, 0.0)
    assert torch.equal(counts.long(), wc) and abs(float(bal - wb)) < 1e-5 and abs(float(z - wz)) < 1e-4
    assert float((dx.reshape(100, 64).double() - wd).abs().max()) < 1e-6
    (dz,) = torch.autograd.grad(H.pool_balance(leaf, ids, mask=mask)[1], leaf)
    _, _, _, wd, _, _ = want64(x.reshape(100, 64), ids.reshape(100, 3), mask.reshape(100), 0.0, 1.0)
    assert float((dz.reshape(100, 64).double() - wd).abs().max()) < 1e-6
    even = H.pool_balance(torch.zeros(64, 64, device=DEV), torch.arange(64, device=DEV)[:, None])
    assert abs(float(even[0]) - 1.0) < 1e-5 and bool((even[2] == 1).all())


def test_by_differences(H):
    """Central differences along a random direction: e^2 / 6 of a third derivative below 50 and rounding over e."""
    g = gen(4)
    x = torch.randn(90, 24, device=DEV, generator=g)
    u = torch.randn(90, 24, device=DEV, generator=g)
    ids, _ = H.route_topk(x, 3)
    e = 2.0 ** -6
    for i in (0, 1):
        leaf = x.clone().requires_grad_()
        (dx,) = torch.autograd.grad(H.pool_balance(leaf, ids)[i], leaf)
        diff = (H.pool_balance(x + e * u, ids)[i].double() - H.pool_balance(x - e * u, ids)[i].double()) / (2 * e)
        assert abs(float(diff - (dx.double() * u.double()).sum())) < 50 * e * e / 6 + 40 * 2.0 ** -22 / e


def test_captured_and_repeated(H):
    g = gen(5)
    x = torch.randn(5000, 64, device=DEV, generator=g, requires_grad=True)
    ids, _ = H.route_topk(x.detach(), 8)

    def both():
        bal, z, counts = H.pool_balance(x, ids)
        return (bal.detach(), z.detach(), counts, *torch.autograd.grad(bal + z, x))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(5000, 64, device=DEV, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        have = [t.clone() for t in out]
        for a, b in zip(have, both()):
            assert torch.equal(a, b), i


def test_refused(H):
    x = torch.randn(6, 8, device=DEV)
    ids = torch.zeros(6, 2, dtype=torch.int32, device=DEV)
    mask = torch.ones(6, dtype=torch.bool, device=DEV)
    for a, m in (((x, ids[:5]), None), ((x, ids[:, :0]), None), ((x, ids), mask[:5]), ((x, ids), mask.float()),
                 ((x[:, :0], ids), None), ((torch.zeros(6, 1025, device=DEV), ids), None)):
        with pytest.raises(ValueError):
            H.pool_balance(*a, mask=m)
    with pytest.raises(TypeError):
        H.pool_balance(x, ids.float())
    with pytest.raises(TypeError):
        H.pool_balance(x.half(), ids)
    with pytest.raises(RuntimeError):
        H.pool_balance(x, ids.cpu())
