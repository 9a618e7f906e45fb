"""Log probabilities of tokens (from logits and from hidden states) and the divergence from a teacher's top
logits, against the definitions in 64 bits.

Tolerances, fixed from the arithmetic: with u = (x - max) / t, a row's exponentials carry the rounding of u
(|u| 2^-24 each, twice with the division) and of exp itself, and their sum at most V / 256 + 16 additions in
sequence, so every sum is right to C = 2^-24 (V / 256 + 16 + 4 max |u|) of its size (`ulps`).  Outputs of 16
bits add half a step, 2^-8 of the value."""

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


def ulps(V, umax):
    return 2.0 ** -24 * (V / 256 + 16 + 4 * umax)


def near(got, want, tol, what):
    """Equal where want is not finite, within tol elsewhere."""
    got, want = got.detach().to(F64), want.detach().to(F64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN at other places"
    odd = ~fin & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd]), f"{what}: infinities differ"
    err = ((got - want).abs() - torch.as_tensor(tol, dtype=F64, device=got.device).expand(want.shape))[fin]
    assert err.numel() == 0 or float(err.max()) <= 0, f"{what}: off by {float(err.max()):.3g} over the tolerance"


def rows64(x, t):
    """log p, p and entropy of softmax(x / t) in 64 bits; a row with no possible column has log p -inf, p 0."""
    z = x.detach().to(F64) / t
    m = z.amax(-1, keepdim=True)
    u = z - torch.where(m == -math.inf, 0.0, m)
    s = u.exp().sum(-1, keepdim=True)
    lp = u - torch.where(s == 0, 0.0, s.log())
    p = lp.exp()
    return lp, p, -torch.where(p == 0, 0.0, p * lp).sum(-1)


def logprobs64(x, tok, t, g_lp, g_h):
    V = x.shape[-1]
    lp, p, h = rows64(x, t)
    at = tok.clamp(0, V - 1)[:, None]
    picked = lp.gather(1, at)[:, 0]
    out = torch.where(tok < 0, 0.0, torch.where(tok >= V, math.nan, picked))
    g = torch.where((tok >= 0) & (tok < V), g_lp, 0.0).to(F64)
    some = (x.detach() > -math.inf).any(1) | torch.isnan(x.detach()).any(1)
    lpc = lp.clamp_min(-1e4)
    one = torch.zeros_like(lp).scatter_(1, at, 1.0)
    d = (one * g[:, None] - p * (g[:, None] + g_h.to(F64)[:, None] * (lpc + h[:, None]))) / t
    # sum of the terms' sizes; log p and the entropy are each off by C itself, however small they are
    scale = (one * g.abs()[:, None] + p * (g.abs()[:, None] + g_h.abs().to(F64)[:, None] * (lpc.abs() + h[:, None] + 1))) / t
    return out, h, torch.where(some[:, None], d, 0.0), scale, lp


def top64(x, k):
    """Columns by value descending (NaN first), ties to the lower column."""
    key = torch.where(torch.isnan(x), math.inf, x.to(F64))
    key = torch.where(torch.isnan(x), torch.finfo(F64).max, torch.where(key == math.inf, 1e300, key))
    return torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]


def check_logprobs(H, x, tok, n_top, t, g):
    V = x.shape[-1]
    leaf = x.detach().requires_grad_()
    g_lp, g_h = torch.randn(x.shape[0], device=DEV, generator=g), torch.rand(x.shape[0], device=DEV, generator=g)
    lp, ent, top_lp, top_ids = H.token_logprobs(leaf, tok, n_top=n_top, temperature=t)
    (dx,) = torch.autograd.grad((lp, ent), (leaf,), (g_lp, g_h))
    torch.cuda.synchronize()
    want, h, d, scale, all_lp = logprobs64(x, tok, t, g_lp, g_h)
    fin = torch.isfinite(x)
    z = torch.where(fin, x.to(F64) / t, 0.0)
    m = torch.where(fin, z, -math.inf).amax(1, keepdim=True)
    near_m = (m - z)[fin & (z > m - 200)]
    c = ulps(V, float(near_m.max()) if near_m.numel() else 0.0)
    # the exponent's own rounding, 2^-24 of every log probability
    near(lp.detach(), want, c + 2.0 ** -22 * want.abs().nan_to_num(0.0, 0.0, 0.0), "logprob")
    near(ent, h, c * (4 + 2 * h.abs().nan_to_num(0.0) + math.log(V + 1)), "entropy")
    near(dx, d, 4.1 * c * scale.nan_to_num(0.0) + HALF[x.dtype] * d.abs().nan_to_num(0.0) + 1e-37, "gradient")
    if n_top:
        ids = top64(x, n_top)
        assert torch.equal(top_ids.long(), ids), "alternatives"
        w = all_lp.gather(1, ids)
        near(top_lp, w, c + 2.0 ** -22 * w.abs().nan_to_num(0.0, 0.0, 0.0), "top log probabilities")


SIZES = [(1, 1), (3, 2), (1, 7), (5, 63), (4, 64), (3, 65), (2, 511), (7, 512), (5, 513), (3, 1000), (9, 2047),
         (6, 2048), (5, 2049), (2, 4099), (3, 8191), (2, 16384), (3, 16385), (1, 32771), (2, 50001), (2, 65537), (1, 200003),
         # one wave per row
         (1024, 1), (1025, 7), (1026, 255), (1030, 300), (1027, 513), (1100, 770), (1024, 1025), (1029, 2047), (1024, 2048),
         (1031, 2049), (1024, 3500), (1026, 4095), (1024, 4096), (1025, 4097)]


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,V", SIZES)
def test_logprobs_sizes(H, T, V, dtype):
    g = gen(T, V, dtype, 1)
    x = (torch.randn(T, V, device=DEV, generator=g) * 3).to(DT[dtype])
    tok = torch.randint(0, V, (T,), device=DEV, generator=g)
    check_logprobs(H, x, tok, min(V, (5, 64, 1, 128)[(T + V) % 4]), (1.0, 0.7, 2.5)[V % 3], g)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n_top", [1, 2, 31, 63, 64, 65, 100, 127, 128])
@pytest.mark.parametrize("T,V", [(6, 128), (6, 700), (6, 2048), (6, 9000), (6, 40000), (1024, 128), (1026, 700), (1025, 1000),
                                 (1024, 2048), (1024, 3001)])
def test_alternatives(H, T, V, n_top, dtype):
    """Every list length; the values of half the rows sit in a narrow range, with many ties in bf16."""
    g = gen(T, V, n_top, dtype, 2)
    x = torch.randn(T, V, device=DEV, generator=g) * 2
    x[T // 2:] = 1.0 + x[T // 2:] * 0.01
    tok = torch.randint(0, V, (T,), device=DEV, generator=g)
    check_logprobs(H, x.to(DT[dtype]), tok, n_top, 1.0, g)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("V,repeat", [(9, 1), (640, 1), (2048, 1), (5000, 1), (20000, 1), (70001, 1), (9, 64), (300, 64), (640, 64),
                                      (2048, 64), (4000, 64)])
def test_awkward_rows(H, V, repeat, dtype):
    """Ties everywhere, rising and falling rows, rows with few or no possible columns, the type's lowest value as a
    mask, signed zeros, large values in one thread's columns, infinities and NaN."""
    g = gen(V, repeat, dtype, 3)
    low = torch.finfo(DT[dtype]).min
    base = torch.randn(V, device=DEV, generator=g)
    few = torch.randperm(V, device=DEV, generator=g)[:3]
    rows = [torch.zeros(V, device=DEV), torch.full((V,), low, device=DEV), torch.full((V,), -math.inf, device=DEV),
            torch.arange(V, device=DEV) / V * 4, -torch.arange(V, device=DEV) / V * 4]
    for fill in (low, -math.inf):
        r = torch.full((V,), fill, device=DEV)
        r[few] = base[few]
        rows.append(r)
    r = torch.zeros(V, device=DEV)
    r[::2] = -0.0
    rows.append(r)
    r = base.clone()
    r[(torch.arange(V, device=DEV) // 8) % 256 == 3] += 30.0
    rows.append(r)
    r = base.clone()
    r[V // 2:] += 40.0
    rows.append(r)
    for bad in ([math.inf], [math.nan], [math.nan, math.inf, -math.nan], [-math.inf]):
        r = base.clone()
        for i, b in enumerate(bad):
            r[(V // 3 + 2 * i) % V] = b
        rows.append(r)
    rows.append(torch.full((V,), math.nan, device=DEV))
    rows.append(base * 1e4)
    x = torch.stack(rows).to(DT[dtype]).repeat(repeat, 1)  # 16 rows; 1024 of them go by wave
    tok = torch.randint(0, V, (x.shape[0],), device=DEV, generator=g)
    tok[6] = few[0]
    for n_top in (1, 6, min(V, 70)):
        check_logprobs(H, x, tok, n_top, 1.0, g)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,V,n_top", [(1, 200003, 128), (3, 300000, 100), (600, 131073, 17)])
def test_many_ranges(H, T, V, n_top, dtype):
    """Rows cut into more ranges than the join's shared memory holds lists of, one with a single column left."""
    g = gen(T, V, n_top, dtype, 20)
    x = torch.randn(T, V, device=DEV, generator=g).to(DT[dtype])
    x[0, ::3] = 1.5
    check_logprobs(H, x, torch.randint(0, V, (T,), device=DEV, generator=g), n_top, 1.0, g)


def test_padded_and_foreign_tokens(H):
    g = gen(4)
    x = torch.randn(8, 300, device=DEV, generator=g)
    x[5] = -math.inf
    tok = torch.tensor([-1, -100, 299, 300, 0, -1, 7, 1 << 40], device=DEV)
    check_logprobs(H, x, tok, 4, 1.0, g)


@pytest.mark.parametrize("grads", ["lp", "ent"])
@pytest.mark.parametrize("V", [100, 3001, 20001])
def test_one_gradient_alone(H, V, grads):
    g = gen(V, grads, 5)
    x = torch.randn(5, V, device=DEV, generator=g, requires_grad=True)
    tok = torch.randint(0, V, (5,), device=DEV, generator=g)
    up = torch.randn(5, device=DEV, generator=g)
    lp, ent, _, _ = H.token_logprobs(x, tok)
    (dx,) = torch.autograd.grad(lp if grads == "lp" else ent, x, up)
    zero = torch.zeros_like(up)
    _, _, d, scale, _ = logprobs64(x, tok, 1.0, *((up, zero) if grads == "lp" else (zero, up)))
    near(dx, d, 4 * ulps(V, 10.0) * scale + 1e-37, "gradient")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("how", ["slice", "offset", "transposed", "expanded", "3d", "1d", "odd"])
def test_strides(H, how, dtype):
    """Rows cut from wider ones, storage that starts off any alignment, columns that are not contiguous, one row
    given to several tokens, further dimensions."""
    g = gen(how, dtype, 6)
    dt = DT[dtype]
    T, V = 6, 5003
    if how == "slice":
        x = torch.randn(T, V + 9, device=DEV, generator=g).to(dt)[:, 3:3 + V]
    elif how == "offset":
        x = torch.randn(T * V + 1, device=DEV, generator=g).to(dt)[1:].view(T, V)
    elif how == "transposed":
        x = torch.randn(V, T, device=DEV, generator=g).to(dt).t()
    elif how == "expanded":
        x = torch.randn(1, V, device=DEV, generator=g).to(dt).expand(T, V)
    elif how == "3d":
        x = torch.randn(2, 3, V, device=DEV, generator=g).to(dt)
    elif how == "1d":
        x = torch.randn(V, device=DEV, generator=g).to(dt)
    else:
        x = torch.randn(2, 5, V, device=DEV, generator=g).to(dt)[:, 1:4]
    lead = x.shape[:-1]
    tok = torch.randint(0, V, tuple(lead), device=DEV, generator=g, dtype=torch.int32)
    leaf = x.detach().requires_grad_()
    lp, ent, top_lp, top_ids = H.token_logprobs(leaf, tok, n_top=9)
    assert lp.shape == ent.shape == lead and top_ids.shape == top_lp.shape == (*lead, 9)
    (dx,) = torch.autograd.grad((lp.sum() + ent.sum(),), (leaf,))
    flat, ft = x.reshape(-1, V), tok.reshape(-1).long()
    one = torch.ones(flat.shape[0], device=DEV)
    want, h, d, scale, all_lp = logprobs64(flat, ft, 1.0, one, one)
    c = ulps(V, 12.0)
    near(lp.reshape(-1), want, c * 20, "logprob")
    near(ent.reshape(-1), h, c * 30, "entropy")
    near(dx.reshape(-1, V), d, 4.1 * c * scale + HALF[dt] * d.abs() + 1e-37, "gradient")
    assert torch.equal(top_ids.reshape(-1, 9).long(), top64(flat, 9))


def test_rows_past_32_bits(H):
    """2.2e9 logits: the last rows' offsets pass 31 and 32 bits of elements and bytes."""
    V, T = 65537, 33000
    x = torch.zeros(T, V, device=DEV, dtype=torch.bfloat16)
    g = gen(7)
    x[-3:] = torch.randn(3, V, device=DEV, generator=g).bfloat16()
    tok = torch.arange(T, device=DEV) % V
    lp, ent, _, ids = H.token_logprobs(x, tok, n_top=3)
    want, h, _, _, _ = logprobs64(x[-3:], tok[-3:], 1.0, torch.ones(3, device=DEV), torch.ones(3, device=DEV))
    c = ulps(V, 10.0)
    near(lp[-3:], want, c * 20, "logprob")
    near(ent[-3:], h, c * 30, "entropy")
    assert torch.equal(ids[-3:].long(), top64(x[-3:], 3)) and bool((ids[:-3] == torch.arange(3, device=DEV)).all())
    near(lp[:-3], torch.full((T - 3,), -math.log(V), dtype=F64, device=DEV), c * 20, "uniform rows")
    leaf = x.requires_grad_()
    lp, _, _, _ = H.token_logprobs(leaf, tok)
    (dx,) = torch.autograd.grad(lp[-3:].sum(), leaf)
    _, _, d, scale, _ = logprobs64(x[-3:], tok[-3:], 1.0, torch.ones(3, device=DEV), torch.zeros(3, device=DEV))
    near(dx[-3:], d, 4.1 * c * scale + 2.0 ** -8 * d.abs() + 1e-37, "gradient")
    assert int(torch.count_nonzero(dx[:-3])) == 0


def test_empty_and_refused(H):
    x = torch.randn(4, 50, device=DEV)
    tok = torch.zeros(4, dtype=torch.long, device=DEV)
    out = H.token_logprobs(x[:0], tok[:0], n_top=3)
    assert [tuple(o.shape) for o in out] == [(0,), (0,), (0, 3), (0, 3)]
    leaf = x[:0].detach().requires_grad_()
    assert torch.autograd.grad(H.token_logprobs(leaf, tok[:0])[0].sum(), leaf)[0].shape == (0, 50)
    for bad in (dict(n_top=51), dict(n_top=-1), dict(temperature=0.0), dict(temperature=math.nan),
                dict(temperature=math.inf), dict(temperature=-1.0)):
        with pytest.raises(ValueError):
            H.token_logprobs(x, tok, **bad)
    with pytest.raises(ValueError):
        H.token_logprobs(torch.randn(2, 400, device=DEV), tok[:2], n_top=129)
    with pytest.raises(ValueError):
        H.token_logprobs(x, tok[:3])
    with pytest.raises(ValueError):
        H.token_logprobs(x[:, :0], tok)
    with pytest.raises(TypeError):
        H.token_logprobs(x, tok.float())
    with pytest.raises(TypeError):
        H.token_logprobs(x.half(), tok)
    with pytest.raises(RuntimeError):
        H.token_logprobs(x, tok.cpu())
    with pytest.raises(RuntimeError):
        H.token_logprobs(x.cpu(), tok)


# ----------------------------------------------------------------------------- from hidden states

def head64(h, w, tok, t, g_lp, g_h):
    """Results and gradients in 64 bits, with the sums of absolute terms that bound their errors."""
    z = h.detach().to(F64) @ w.detach().to(F64).t()
    out, ent, d, scale, _ = logprobs64(z, tok, t, g_lp, g_h)
    hd, wd = h.detach().to(F64), w.detach().to(F64)
    za = (hd.abs() @ wd.abs().t()).max() / t
    za, zmax = float(za), float(z.abs().max()) / t
    # a logit is off by zerr, a log probability by c; the gradient of a logit is rounded to bf16, and so are the results
    zerr = h.shape[1] * 2.0 ** -24 * za
    c = ulps(w.shape[0], 2 * zmax) + 2 * zerr
    dl = 1.01 * 2.0 ** -8 * d.abs() + (4.1 * c + 2.0 ** -20) * scale
    xh, xw = d @ wd, d.t() @ hd
    return out, ent, xh, xw, dl @ wd.abs() + 2.0 ** -8 * xh.abs(), dl.t() @ hd.abs() + 2.0 ** -8 * xw.abs(), c, zmax


@pytest.mark.parametrize("T,d,V", [(1, 8, 1), (1, 64, 300), (3, 64, 17), (65, 72, 129), (64, 128, 256), (200, 512, 2048),
                                   (129, 256, 1000), (300, 128, 8200), (257, 64, 515), (33, 1024, 4099), (2100, 64, 640), (1, 128, 1), (2, 128, 8), (255, 192, 24), (257, 128, 72), (600, 256, 3000),
                                   (512, 512, 512)])
@pytest.mark.parametrize("t", [1.0, 0.7, 0.01])
def test_head_sizes(H, T, d, V, t):
    """Logits in fp32 from bf16 operands: each off by at most d 2^-24 of the sum of absolute products.  The backward
    rounds a logit's gradient to bf16 (2^-8 of it) before the two products with h and w, and the results again."""
    g = gen(T, d, V, 8)
    h = torch.randn(T, d, device=DEV, generator=g).bfloat16().requires_grad_()
    w = (torch.randn(V, d, device=DEV, generator=g) * (2 / math.sqrt(d))).bfloat16().requires_grad_()
    tok = torch.randint(0, V, (T,), device=DEV, generator=g)
    if T > 2:
        tok[1] = -100
    g_lp, g_h = torch.randn(T, device=DEV, generator=g), torch.rand(T, device=DEV, generator=g)
    lp, ent = H.lm_head_logprobs(h, w, tok, temperature=t)
    dh, dw = torch.autograd.grad((lp, ent), (h, w), (g_lp, g_h))
    out, e, xh, xw, th, tw, c, zmax = head64(h, w, tok, t, g_lp, g_h)
    assert dh.dtype == dw.dtype == torch.bfloat16
    near(lp, out, c + 2.0 ** -22 * out.abs(), "logprob")
    near(ent, e, c * (4 + 2 * zmax + math.log(V + 1)), "entropy")
    # a probability below 2^-126, fp32's least normal number, is 0: times at most (|g| + g_H (|log p| + H)) / t, log p
    # above -88 there, H below 10, |g| below 5, g_H below 1, and |h|, |w| below 8
    least = 2.0 ** -126 * 103 / t * 8
    near(dh, xh, th + V * least, "hidden gradient")
    near(dw, xw, tw + T * least, "weight gradient")


def test_head_forms(H):
    """fp32 master weights and hidden states, further dimensions, one wanted gradient, no tokens, padding alone."""
    g = gen(9)
    T, d, V = 96, 128, 1100
    h = torch.randn(2, 48, d, device=DEV, generator=g).requires_grad_()
    w = (torch.randn(V, d, device=DEV, generator=g) * 0.2).requires_grad_()
    tok = torch.randint(0, V, (2, 48), device=DEV, generator=g, dtype=torch.int32)
    lp, ent = H.lm_head_logprobs(h, w, tok)
    assert lp.shape == ent.shape == (2, 48)
    up = torch.randn(2, 48, device=DEV, generator=g)
    dh, dw = torch.autograd.grad(lp, (h, w), up)
    assert dh.dtype == dw.dtype == torch.float32 and dh.shape == h.shape
    hb, wb = h.detach().bfloat16().reshape(T, d), w.detach().bfloat16()
    z = torch.zeros(T, device=DEV)
    out, _, xh, xw, th, tw, c, zmax = head64(hb, wb, tok.reshape(-1).long(), 1.0, up.reshape(-1), z)
    near(lp.reshape(-1), out, c + 2.0 ** -22 * out.abs(), "logprob")
    near(dh.reshape(T, d), xh, th + 1e-35, "hidden gradient")
    near(dw, xw, tw + 1e-35, "weight gradient")
    only_h = torch.autograd.grad(H.lm_head_logprobs(h, w.detach(), tok)[0], h, up)[0]
    only_w = torch.autograd.grad(H.lm_head_logprobs(h.detach(), w, tok)[0], w, up)[0]
    assert torch.equal(only_h, dh) and torch.equal(only_w, dw)
    lp, ent = H.lm_head_logprobs(h[:0], w, tok[:0])
    assert lp.shape == (0, 48)
    dh, dw = torch.autograd.grad(lp.sum() + ent.sum(), (h, w))
    assert not dh.any() and not dw.any()
    lp, _ = H.lm_head_logprobs(h, w, torch.full_like(tok, -1))
    dh, dw = torch.autograd.grad(lp, (h, w), up)
    assert not lp.any() and not dh.any() and not dw.any()


@pytest.mark.parametrize("V", [640, 1096, 2056])
def test_head_by_vocabulary_ranges(H, V, monkeypatch):
    """A small budget of logit gradients: several ranges, the last of them less than 64 columns."""
    g = gen(V, 18)
    T, d = 100, 192
    h = torch.randn(T, d, device=DEV, generator=g).bfloat16().requires_grad_()
    w = (torch.randn(V, d, device=DEV, generator=g) * 0.2).bfloat16().requires_grad_()
    tok = torch.randint(0, V, (T,), device=DEV, generator=g)
    up = torch.randn(T, device=DEV, generator=g)
    monkeypatch.setattr(H.LMHeadLogprobsFn, "GRAD", 2 * T * 300)
    lp, ent = H.lm_head_logprobs(h, w, tok)
    dh, dw = torch.autograd.grad((lp, ent), (h, w), (up, up))
    out, e, xh, xw, th, tw, c, zmax = head64(h, w, tok, 1.0, up, up)
    near(lp, out, c + 2.0 ** -22 * out.abs(), "logprob")
    near(dh, xh, th + 1e-35, "hidden gradient")
    near(dw, xw, tw + 1e-35, "weight gradient")


def test_head_off_alignment(H):
    """Hidden states and a matrix that start two bytes into a word."""
    g = gen(19)
    T, d, V = 70, 128, 320
    h = torch.randn(T * d + 1, device=DEV, generator=g).bfloat16()[1:].view(T, d)
    w = (torch.randn(V * d + 1, device=DEV, generator=g) * 0.2).bfloat16()[1:].view(V, d)
    tok = torch.randint(0, V, (T,), device=DEV, generator=g)
    a, b = H.lm_head_logprobs(h, w, tok), H.lm_head_logprobs(h.clone(), w.clone(), tok)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_head_agrees_with_the_stored_logits(H):
    """The same logits through lm_head_ce and token_logprobs; in the fp32 precision too."""
    g = gen(10)
    T, d, V = 130, 256, 2048
    h = torch.randn(T, d, device=DEV, generator=g)
    w = torch.randn(V, d, device=DEV, generator=g) * 0.1
    tok = torch.randint(0, V, (T,), device=DEV, generator=g)
    logits, loss = H.lm_head_ce(h, w, tok)
    lp, ent = H.lm_head_logprobs(h, w, tok)
    lp2, ent2, _, _ = H.token_logprobs(logits, tok)
    c = ulps(V, 2 * float(logits.abs().max())) * 8
    near(lp, lp2, c + 1e-6 * lp2.abs(), "logprob")
    near(ent, ent2, 20 * c, "entropy")
    near(-loss, lp2, c + 1e-6 * lp2.abs(), "cross-entropy")
    with H.fp32_precision():
        h32 = h.clone().requires_grad_()
        lp, ent = H.lm_head_logprobs(h32, w, tok)
        (dh,) = torch.autograd.grad(lp.sum(), h32)
    out, e, xh, _, th, _, c, zmax = head64(h, w, tok, 1.0, torch.ones(T, device=DEV), torch.zeros(T, device=DEV))
    near(lp, out, c + 2.0 ** -22 * out.abs(), "fp32 logprob")
    near(dh, xh, 2.0 ** -6 * th, "fp32 gradient")  # a 64th of what bf16 operands may be off


def test_head_refused(H):
    h, w = torch.randn(4, 64, device=DEV), torch.randn(50, 64, device=DEV)
    tok = torch.zeros(4, dtype=torch.long, device=DEV)
    for a in ((h[:, :60], w, tok), (h, w, tok[:3]), (h[:, :60], w[:, :60], tok), (h, w[0], tok)):
        with pytest.raises(ValueError):
            H.lm_head_logprobs(*a)
    with pytest.raises(ValueError):
        H.lm_head_logprobs(h, w, tok, temperature=0)
    with pytest.raises(TypeError):
        H.lm_head_logprobs(h, w, tok.float())
    with pytest.raises(RuntimeError):
        H.lm_head_logprobs(h, w.cpu(), tok)


# ----------------------------------------------------------------------------- distillation from top logits

def distill64(x, ids, tl, t, tail, g):
    T, V = x.shape
    z = x.detach().to(F64) / t
    lq, q, _ = rows64(x, t)
    loss = torch.zeros(T, dtype=F64, device=x.device)
    d = torch.zeros(T, V, dtype=F64, device=x.device)
    scale = q.clone()
    for r in range(T):
        cols, vals, bad = [], [], False
        for c, v in zip(ids[r].tolist(), tl[r].tolist()):
            bad |= c >= V
            if 0 <= c < V and c not in cols:
                cols.append(c)
                vals.append(v)
        if bad:
            loss[r] = math.nan
            continue
        vals = torch.tensor(vals, dtype=F64, device=x.device)
        if not cols or (not tail and bool((vals == -math.inf).all())):
            continue
        at = torch.tensor(cols, device=x.device)
        lp = vals if tail else torch.log_softmax(vals / t, 0)
        p = lp.exp()
        terms = torch.where(p == 0, 0.0, p * (lp - lq[r, at]))
        on = torch.zeros(V, dtype=torch.bool, device=x.device)
        on[at] = True
        grad = q[r].clone()
        grad[at] -= p
        scale[r, at] += p
        total = terms.sum()
        rest = float(max(0.0, 1.0 - float(p.sum()))) if tail else 0.0
        if rest > 0:
            zr = z[r].masked_fill(on, -math.inf)
            lqr = torch.logsumexp(lq[r].masked_fill(on, -math.inf), 0)
            total = total + rest * (math.log(rest) - lqr)
            if bool((zr > -math.inf).any()):
                soft = torch.softmax(zr, 0)
                grad = grad - rest * soft
                scale[r] += rest * soft
        loss[r] = total * t * t
        if bool((x[r] > -math.inf).any()):
            d[r] = grad * float(g[r]) * t
    return loss, d, scale * g.to(F64).abs()[:, None] * t


def check_distill(H, x, ids, tl, t, tail, g):
    T, V = x.shape
    leaf = x.detach().requires_grad_()
    up = torch.rand(T, device=DEV, generator=g) + 0.5
    loss = H.topk_distill(leaf, ids, tl, temperature=t, tail=tail)
    (dx,) = torch.autograd.grad(loss, leaf, up)
    torch.cuda.synchronize()
    want, d, scale = distill64(x.cpu(), ids.cpu(), tl.float().cpu(), t, tail, up.cpu())
    lq, q, _ = rows64(x.cpu(), t)
    umax = float((lq.amax(1, keepdim=True) - lq)[lq > lq.amax(1, keepdim=True) - 200].max()) if V > 1 else 0.0
    c = ulps(V, umax)
    # near agreement the terms cancel to second order; the sums' errors enter each term once
    near(loss.cpu(), want, (2 * c + 2.0 ** -22 * want.abs().nan_to_num(0.0, 0.0, 0.0)) * t * t, "loss")
    near(dx.cpu(), d, (8 * c + HALF[x.dtype]) * scale.nan_to_num(0.0) + 2.0 ** -21 * float(up.max()) * t * q.nan_to_num(0.0)
         + 1e-37, "gradient")


def teacher(x, K, t, tail, g, noise=1.0):
    y = x.float().masked_fill(x == -math.inf, -30.0) + noise * torch.randn(x.shape, device=DEV, generator=g)
    v, ids = torch.topk(y, K, dim=1)
    return ids, (v - torch.logsumexp(y / t, 1, keepdim=True) * t) / t if tail else v


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,V,K", [(1, 1, 1), (3, 2, 1), (3, 5, 5), (4, 64, 64), (3, 65, 7), (5, 513, 128), (3, 2047, 16),
                                   (6, 2048, 64), (4, 2049, 65), (3, 5001, 1), (2, 16384, 127), (3, 16385, 32),
                                   (2, 40001, 100), (2, 70001, 64), (1024, 1, 1), (1025, 64, 64), (1026, 500, 100), (1024, 1001, 16),
                                   (1027, 2048, 64), (1024, 4001, 33)])
def test_distill_sizes(H, T, V, K, dtype, tail):
    g = gen(T, V, K, dtype, tail, 11)
    x = (torch.randn(T, V, device=DEV, generator=g) * 2).to(DT[dtype])
    t = (1.0, 2.0, 0.7)[(V + K) % 3]
    ids, tl = teacher(x, K, t, tail, g)
    check_distill(H, x, ids.int() if K % 2 else ids, tl, t, tail, g)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("V,repeat", [(40, 1), (1500, 1), (2048, 1), (9001, 1), (33001, 1), (40, 74), (1500, 74), (4000, 74)])
def test_distill_awkward_lists(H, V, repeat, tail):
    """Missing entries, none at all, repeated ids, ids past the vocabulary, listed values of -inf, equal ones, a
    student that cannot reach a listed column or any column, mass outside the list that all but vanishes."""
    g = gen(V, repeat, tail, 12)
    K = 9
    x = torch.randn(14, V, device=DEV, generator=g) * 2
    ids, tl = teacher(x, K, 1.0, tail, g)
    ids[0, 3:] = -1
    ids[1] = -1
    ids[2] = ids[2, :1]
    ids[3, 5] = ids[3, 1]
    ids[4, 8] = V
    ids[5, 0] = (1 << 32) + 1
    tl[6, 2:] = -math.inf
    tl[7] = -math.inf
    tl[8] = -math.log(2 * K) if tail else 3.0
    x[9, ids[9, 0]] = -math.inf
    x[10] = -math.inf
    x[11] = -60.0
    x[11, ids[11]] = 10.0                        # the student's rest is e^-70 of its list
    x[12, :] = torch.finfo(torch.float32).min    # a row at the type's lowest value is even
    x[13, : V // 2] = -math.inf
    keep = torch.tensor([i for i in range(14) if i not in (9, 10, 11, 12)], device=DEV)
    many = lambda v, n=1: v.repeat(repeat * n, 1)  # 1024 rows and more go by wave
    check_distill(H, many(x), many(ids), many(tl), 1.0, tail, g)
    check_distill(H, many(x[keep], 2).bfloat16(), many(ids[keep], 2), many(tl[keep], 2), 2.0, tail, g)


def test_distill_agreement_is_zero(H):
    """A student that is its own teacher: loss 0 and no gradient, with the rest as one more alternative; the loss of
    a near one is the square of the difference, not the rounding of its terms."""
    g = gen(13)
    x = torch.randn(50, 3000, device=DEV, generator=g) * 2
    _, _, tl, ids = H.token_logprobs(x, torch.zeros(50, dtype=torch.long, device=DEV), n_top=20, temperature=2.0)
    leaf = x.clone().requires_grad_()
    loss = H.topk_distill(leaf, ids, tl, temperature=2.0, tail=True)
    (dx,) = torch.autograd.grad(loss.sum(), leaf)
    # log probabilities of 2^-22 make a difference of at most that square times K, and 1 - sum p of 2^-22
    assert float(loss.detach().abs().max()) < 1e-9 and float(dx.abs().max()) < 4e-6
    full = H.topk_distill(x[:, :100].contiguous(), torch.arange(100, device=DEV).expand(50, 100), x[:, :100])
    assert float(full.abs().max()) < 1e-6


def test_distill_strides(H):
    g = gen(14)
    V, K = 3001, 12
    wide = torch.randn(2, 4, V + 5, device=DEV, generator=g).bfloat16()
    x = wide[..., 2:2 + V]
    ids, tl = teacher(x.reshape(8, V), K, 1.0, False, g)
    leaf = x.detach().requires_grad_()
    loss = H.topk_distill(leaf, ids.view(2, 4, K), tl.view(2, 4, K).double())
    assert loss.shape == (2, 4)
    (dx,) = torch.autograd.grad(loss.sum(), leaf)
    want, d, scale = distill64(x.reshape(8, V).cpu(), ids.cpu(), tl.cpu(), 1.0, False, torch.ones(8))
    c = ulps(V, 12.0)
    near(loss.reshape(8).cpu(), want, 2 * c + 1e-6, "loss")
    near(dx.reshape(8, V).cpu(), d, (8 * c + 2.0 ** -8) * scale + 1e-6 * scale, "gradient")


def test_distill_refused(H):
    x = torch.randn(4, 50, device=DEV)
    ids, tl = torch.zeros(4, 3, dtype=torch.long, device=DEV), torch.zeros(4, 3, device=DEV)
    assert H.topk_distill(x[:0], ids[:0], tl[:0]).shape == (0,)
    for a in ((x, ids, tl[:, :2]), (x, ids[:3], tl[:3]), (x, ids[:, :0], tl[:, :0]),
              (x, ids.repeat(1, 43), tl.repeat(1, 43)), (x[:, :0], ids, tl)):
        with pytest.raises(ValueError):
            H.topk_distill(*a)
    with pytest.raises(ValueError):
        H.topk_distill(x, ids, tl, temperature=-1.0)
    for a in ((x, ids.float(), tl), (x, ids, tl.long()), (x.half(), ids, tl)):
        with pytest.raises(TypeError):
            H.topk_distill(*a)
    with pytest.raises(RuntimeError):
        H.topk_distill(x, ids.cpu(), tl)


# ----------------------------------------------------------------------------- derivatives by differences

def test_gradients_by_differences(H):
    """Central differences of the fp32 results along a random direction: step e = 2^-6 leaves e^2 / 6 times the
    third derivative (below 1 for these sums) and 2^-22 / e of rounding in each of the T terms."""
    g = gen(15)
    T, V, K = 6, 400, 8
    x = torch.randn(T, V, device=DEV, generator=g)
    u = torch.randn(T, V, device=DEV, generator=g)
    tok = torch.randint(0, V, (T,), device=DEV, generator=g)
    ids, tl = teacher(x, K, 1.0, True, g)
    fns = (lambda y: H.token_logprobs(y, tok)[0], lambda y: H.token_logprobs(y, tok)[1],
           lambda y: H.topk_distill(y, ids, tl, tail=True), lambda y: H.topk_distill(y, ids, tl * 2))
    e = 2.0 ** -6
    for f in fns:
        leaf = x.clone().requires_grad_()
        (dx,) = torch.autograd.grad(f(leaf).sum(), leaf)
        diff = (f(x + e * u).double().sum() - f(x - e * u).double().sum()) / (2 * e)
        have = (dx.double() * u.double()).sum()
        assert abs(float(diff - have)) < T * (e * e * 4 + 16 * 2.0 ** -22 / e), (float(diff), float(have))


# ----------------------------------------------------------------------------- how programs use them

def test_streams_and_repeats(H):
    """Calls on a stream of their own, two streams at once, and the same bits every time."""
    g = gen(16)
    x = torch.randn(40, 30011, device=DEV, generator=g).bfloat16().requires_grad_()
    tok = torch.randint(0, 30011, (40,), device=DEV, generator=g)
    ids, tl = teacher(x.detach(), 24, 1.0, True, g)

    def both():
        lp, ent, tv, ti = H.token_logprobs(x, tok, n_top=50)
        loss = H.topk_distill(x, ids, tl, tail=True)
        return (lp, ent, tv, ti, loss, *torch.autograd.grad((lp.sum() + ent.sum() + loss.sum(),), (x,)))

    first = both()
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for s in sides:
            with torch.cuda.stream(s):
                outs.append(both())
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, first))


@pytest.mark.parametrize("V", [900, 30011])
def test_captured(H, V):
    """Forward and backward captured and replayed several times with new inputs and eager work in between; two graphs
    replayed in turn keep their own workspaces."""
    g = gen(V, 17)
    T, K, d = (1040 if V == 900 else 24), 16, 64
    x = torch.randn(T, V, device=DEV, generator=g, requires_grad=True)
    h = torch.randn(T, d, device=DEV, generator=g).bfloat16().requires_grad_()
    w = (torch.randn(1024, d, device=DEV, generator=g) * 0.2).bfloat16().requires_grad_()
    tok = torch.randint(0, 900, (T,), device=DEV, generator=g)
    ids, tl = teacher(x.detach(), K, 1.0, True, g)

    def logits_side():
        lp, ent, tv, ti = H.token_logprobs(x, tok, n_top=20)
        loss = H.topk_distill(x, ids, tl, tail=True)
        return (lp.detach(), ent.detach(), tv, ti, loss.detach(),
                *torch.autograd.grad((lp.sum() - ent.sum() + loss.sum(),), (x,)))

    def head_side():
        lp, ent = H.lm_head_logprobs(h, w, tok)
        return (lp.detach(), ent.detach(), *torch.autograd.grad((lp.sum() + ent.sum(),), (h, w)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        logits_side(), head_side()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for fn in (logits_side, head_side):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = fn()
        graphs.append((gr, fn, out))
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(T, V, device=DEV, generator=g))
            h.copy_(torch.randn(T, d, device=DEV, generator=g))
            tok.copy_(torch.randint(0, 900, (T,), device=DEV, generator=g))
        for gr, fn, out in graphs:
            gr.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in out] for _, _, out in graphs]
        for (gr, fn, _), have in zip(graphs, got):
            want = fn()
            torch.cuda.synchronize()
            for a, b in zip(have, want):
                assert torch.equal(a, b), f"replay {i} of {fn.__name__}"


# ----------------------------------------------------------------------------- students limited to the list

@pytest.mark.parametrize("V,repeat", [(40, 1), (3000, 1), (9001, 1), (70001, 1), (40, 256), (2000, 256)])
def test_distill_nothing_outside_the_list(H, V, repeat):
    """Only listed columns are possible: the others have probability 0 and gradient 0, in rows with one such column
    and in rows with all of them."""
    g = gen(V, 21)
    x = torch.full((4, V), -math.inf, device=DEV)
    ids = torch.stack([torch.randperm(V, device=DEV, generator=g)[:7] for _ in range(4)])
    x.scatter_(1, ids, torch.randn(4, 7, device=DEV, generator=g))
    x[1, ids[1, 1:]] = -math.inf
    tl = torch.randn(4, 7, device=DEV, generator=g)
    tl[1, 1:] = -math.inf
    many = lambda v: v.repeat(repeat, 1)
    check_distill(H, many(x), many(ids), many(tl), 1.0, False, g)
    check_distill(H, many(x).bfloat16(), many(ids), many(tl), 2.0, False, g)


# ----------------------------------------------------------------------------- enough rows for one range each

@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("T,V,n_top", [(513, 131072, 5), (520, 131071, 128), (513, 140001, 33), (700, 8193, 100)])
def test_longest_single_range(H, T, V, n_top, dtype):
    """One workgroup's whole room for a row, all but a column of it, and a second range; ties in the last columns, in one
    lane's and everywhere."""
    g = gen(T, V, dtype, 22)
    x = torch.randn(T, V, device=DEV, generator=g).to(DT[dtype])
    x[1, -3:] = 9.0
    x[2, 64:V:8192] = 7.0
    x[3, ::2] = 6.0
    x[4] = 1.0
    x[5, : V - 2] = -math.inf
    tok = torch.randint(0, V, (T,), device=DEV, generator=g)
    tok[:6] = V - 1
    check_logprobs(H, x, tok, n_top, 1.0, g)


@pytest.mark.parametrize("V", [131072, 140001])
def test_distill_longest_single_range(H, V):
    """520 rows take one range each (two past 131072 columns), eight of them many short ones: the same results, within
    the tolerances of both."""
    g = gen(V, 23)
    x = torch.randn(8, V, device=DEV, generator=g) * 2
    ids, tl = teacher(x, 100, 1.0, True, g)
    ids[0, 0], ids[1, 5] = V - 1, ids[1, 9]
    check_distill(H, x, ids, tl, 1.0, True, g)
    leaf = x.detach().requires_grad_()
    few = H.topk_distill(leaf, ids, tl, tail=True)
    (d_few,) = torch.autograd.grad(few.sum(), leaf)
    many = x.repeat(65, 1).requires_grad_()
    loss = H.topk_distill(many, ids.repeat(65, 1), tl.repeat(65, 1), tail=True)
    (dx,) = torch.autograd.grad(loss.sum(), many)
    c = ulps(V, 2 * 12.0)
    near(loss.view(65, 8), few.expand(65, 8), 2 * (2 * c + 2.0 ** -22 * few.detach().double().abs()), "loss")
    q = torch.softmax(x.double(), 1)
    p = torch.zeros_like(q).scatter_(1, ids, tl.double().exp())
    tol = 2 * (8 * c * (2 * q + p) + 2.0 ** -21 * q) + 1e-37
    near(dx.view(65, 8, V), d_few.expand(65, 8, V), tol.expand(65, 8, V), "gradient")
