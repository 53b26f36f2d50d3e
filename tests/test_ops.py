"""The public operators (lsdm_amd/ops.py) against their definitions in 64 bits, element by element, with bounds that are added up from the roundings of
the evaluation: u = 2^-24 for an fp32 operation, half a step of the result's type for the one rounding at the end, and the stated steps of what is kept
for the backward pass.  Sums: a contraction of K terms is a chain of K fp32 additions in the worst order (2 K u sum |terms|); a row sum of the norm is
at most 16 additions per lane and 10 across lanes and waves (32 u sum |terms|)."""
import copy
import ctypes as C
import math
import pickle

import pytest
import torch

from lsdm_amd import _lib, ops
from lsdm_amd.text import LayerNorm, Linear, use_kernels

gpu = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(autouse=True)
def _grad_mode():
    with torch.enable_grad():       # (other modules of the suite switch it off at import)
        yield


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps       # half the spacing of subnormals is below this


def within(got, want, tol, what=""):
    got, want = got.double(), want.double()
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), "%s: %d of %d out of bounds, worst excess %.3g (got %.6g, want %.6g)" % (
        what, int(bad.sum()), bad.numel(), float(((got - want).abs() - tol)[bad].max()), float(got[bad][0]), float(want[bad][0]))


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def act64(name, z):
    s = lambda v: torch.special.expit(v)
    phi = lambda v: torch.special.ndtr(v)
    if name == "none":
        return z.clone(), torch.ones_like(z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "gelu":
        return z * phi(z), phi(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name in ("quick_gelu", "silu"):
        c = 1.702 if name == "quick_gelu" else 1.0
        return z * s(c * z), s(c * z) * (1 + c * z * s(-c * z))
    if name == "sigmoid":
        return s(z), s(z) * s(-z)
    return torch.tanh(z), 1 / torch.cosh(z) ** 2


def pow2(e):
    """2^e exactly (torch.ldexp's power is a last bit off on the device)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def stored8(v):
    """What the 8-bit checkpoint of v (rows, D) stands for."""
    out = torch.empty_like(v)
    for lo in range(0, v.shape[1], 32):
        g = v[:, lo:lo + 32]
        m = g.abs().amax(dim=1, keepdim=True)
        e = (torch.frexp(m)[1] - 7).clamp(min=-126)
        out[:, lo:lo + 32] = torch.round(g * pow2(-e)).clamp(-127, 127) * pow2(e)
    return out


def step8(v):
    """The step of every element's group."""
    out = torch.empty_like(v)
    for lo in range(0, v.shape[1], 32):
        g = v[:, lo:lo + 32]
        e = (torch.frexp(g.abs().amax(dim=1, keepdim=True))[1] - 7).clamp(min=-126)
        out[:, lo:lo + 32] = pow2(e)
    return out


def linear_case(M, K, N, dt, seed, bias=True, residual=True, bias_f32=False):
    gen = torch.Generator().manual_seed(seed)
    t = DT[dt]
    x = torch.randn(M, K, generator=gen).to(t)
    w = (torch.randn(N, K, generator=gen) / math.sqrt(K)).to(t)
    b = (0.5 * torch.randn(N, generator=gen)).to(torch.float32 if bias_f32 else t) if bias else None
    r = torch.randn(M, N, generator=gen).to(t) if residual else None
    dy = torch.randn(M, N, generator=gen).to(t)
    return [v.to(DEV) if v is not None else None for v in (x, w, b, r, dy)]


def linear_check(x, w, b, r, dy, act, y, grads=None, checkpoint8=False):
    """y and (dx, dw, db) of the operator against the definition.  x (M,K), w (N,K)."""
    t = x.dtype
    M, K = x.shape
    N = w.shape[0]
    x64, w64 = x.detach().double(), w.detach().double()
    z = x64 @ w64.T
    mag = x64.abs() @ w64.abs().T
    if b is not None:
        z = z + b.detach().double()
        mag = mag + b.detach().double().abs()
    ez = 2 * (K + 1) * U * mag                                     # fp32 sums
    a, d = act64(act, z)
    # the activation: slope at most 1.13; its own evaluation is off by at most 4e-7 (1 + |z|) (16 bits) or a few fp32 roundings
    ea = 1.13 * ez + (4e-7 if t != torch.float32 else 8 * U) * (1 + z.abs()) * (act != "none")
    want = a + (r.detach().double() if r is not None else 0)
    out = half_step(t)
    within(y, want, (ea + 4 * U * want.abs()) * (1 + out) + out * want.abs() + tiny(t), "y")
    if grads is None:
        return
    dy64 = dy.double()
    # a'(z): second derivatives are at most 1.2 (quick_gelu 1.702 x that); relu jumps where z is not sure of its sign
    ed = 2.1 * ez + (1.2e-6 if t != torch.float32 else 16 * U) * (1 + z.abs()) * (act != "none")
    if act == "relu":
        ed = (z.abs() <= ez).double()
    if act == "none":
        ed = torch.zeros_like(z)
    if checkpoint8:
        x64 = stored8(x64)
    if checkpoint8 and t != torch.float32 and act != "none":
        frac = (192 * d - torch.floor(192 * d) - 0.5).abs()
        flip = (frac <= 192 * ed).double() if act != "relu" else ed * 192
        ed = flip / 192
        d = torch.round(192 * d) / 192
    elif t != torch.float32 and act != "none":
        ed = ed + 2.0 ** -13 * d.abs() + 2.0 ** -19
    dz = dy64 * d
    edz = dy64.abs() * ed + 2 * U * dz.abs()
    edz_r = edz + half_step(t) * (dz.abs() + edz) + tiny(t)        # rounded to the operand's type in front of the products
    dx, dw, db = grads
    if dx is not None:
        want = dz @ w64
        within(dx, want, edz_r @ w64.abs() + 2 * (N + 1) * U * (dz.abs() + edz_r) @ w64.abs() + 2 * out * want.abs() + tiny(t) + 1e-30, "dx")
    if dw is not None:
        want = dz.T @ x64
        within(dw, want, edz_r.T @ x64.abs() + 2 * (M + 34) * U * (dz.abs() + edz_r).T @ x64.abs() + 2 * out * want.abs() + tiny(t) + 1e-30, "dw")
    if db is not None:
        want = dz.sum(0)
        within(db, want, edz.sum(0) + 2 * (M + 2) * U * (dz.abs() + edz).sum(0) + 2 * half_step(db.dtype) * want.abs() + tiny(t) + 1e-30, "db")


def run_linear(x, w, b, r, dy, act, **kw):
    leaves = [v.requires_grad_(True) for v in (x, w, b, r) if v is not None]
    y = ops.linear(x, w, b, act, r, **kw)
    g = list(torch.autograd.grad(y, leaves, dy))
    dx, dw = g[0], g[1]
    db = g[2] if b is not None else None
    if r is not None:
        assert torch.equal(g[-1], dy)
    return y.detach(), (dx, dw, db)


# sizes: single rows and columns, both sides of the few-rows kernel's limit and of its 16-row blocks, tiles cut on every side, contraction tails,
# widths that no 16-byte load divides, long contractions (split and joined)
LINEAR_SIZES = [(1, 1, 1), (1, 512, 256), (2, 7, 3), (16, 64, 33), (17, 100, 8), (48, 33, 50), (64, 129, 64), (65, 64, 64), (66, 1, 9), (100, 72, 1),
                (129, 520, 136), (257, 65, 131), (300, 515, 70), (77, 768, 512), (512, 48, 640), (70, 5000, 24), (2100, 40, 24), (1030, 256, 520)]


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("i", range(len(LINEAR_SIZES)), ids=["x".join(map(str, s)) for s in LINEAR_SIZES])
def test_linear_forward_and_gradients(dt, i):
    M, K, N = LINEAR_SIZES[i]
    acts = list(ops.ACTIVATIONS)
    act = acts[(i + 2 * list(DT).index(dt)) % len(acts)]
    x, w, b, r, dy = linear_case(M, K, N, dt, i, bias=i % 4 != 1, residual=i % 3 != 2, bias_f32=i % 5 == 0)
    y, g = run_linear(x, w, b, r, dy, act)
    linear_check(x, w, b, r, dy, act, y, g)
    with torch.no_grad():
        assert torch.equal(ops.linear(x, w, b, act, r), y)             # inference evaluates the same thing
    y, g = run_linear(x, w, b, r, dy, act, checkpoint8=True)
    linear_check(x, w, b, r, dy, act, y, g, checkpoint8=True)


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("act", list(ops.ACTIVATIONS))
def test_linear_every_activation(dt, act):
    x, w, b, r, dy = linear_case(130, 96, 72, dt, 5)
    x.mul_(3.0)                                                         # saturated tails too
    y, g = run_linear(x, w, b, r, dy, act)
    linear_check(x, w, b, r, dy, act, y, g)


@gpu
@pytest.mark.parametrize("dt,M,K,N", [("bf16", 2304, 256, 2048), ("f16", 1100, 1024, 1536), ("bf16", 768, 4096, 640), ("f32", 1200, 640, 1152)])
def test_linear_large_tiles(dt, M, K, N):
    """Sizes that the 256- and 128-wide tiles and the split contraction take."""
    x, w, b, r, dy = linear_case(M, K, N, dt, 9)
    y, g = run_linear(x, w, b, r, dy, "gelu")
    linear_check(x, w, b, r, dy, "gelu", y, g)


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("M,K,N", [(2828, 2846, 2987), (5509, 666, 5667), (2089, 2099, 2028), (4762, 392, 2952), (1794, 1839, 1671), (1044, 1060, 2942)])
def test_linear_every_tile(dt, M, K, N):
    """Ragged sizes at which y, dx and dW are evaluated by the 256 x 256 tile (whole and split), the 128 x 128 one (whole; split) and the 64 x 128 one
    (whole; dx split) in 16 bits, and by fp32's large tile."""
    x, w, b, r, dy = linear_case(M, K, N, dt, 21, bias_f32=True)
    y, g = run_linear(x, w, b, r, dy, "quick_gelu")
    linear_check(x, w, b, r, dy, "quick_gelu", y, g)


@gpu
def test_linear_gradient_against_differences():
    gen = torch.Generator().manual_seed(3)
    x, w, b = (torch.randn(*s, generator=gen).to(DEV) for s in ((9, 12), (7, 12), (7,)))
    for act in ops.ACTIVATIONS:
        if act == "relu":
            continue
        leaves = [v.clone().requires_grad_(True) for v in (x, w, b)]
        c = torch.randn(9, 7, generator=gen).to(DEV)
        g = torch.autograd.grad((ops.linear(*leaves, act) * c).sum(), leaves)
        for k in range(3):
            v = torch.randn(leaves[k].shape, generator=gen).to(DEV)
            h = 2.0 ** -7

            def f(s):
                args = [t.detach() for t in leaves]
                args[k] = args[k] + s * v
                return float((ops.linear(*args, act).double() * c.double()).sum())
            # truncation: h^2 / 6 times a third derivative summed over 63 outputs; rounding: fp32 outputs over 2 h
            assert abs((f(h) - f(-h)) / (2 * h) - float((g[k].double() * v.double()).sum())) <= 0.03 * (1 + float((g[k] * v).abs().sum())), (act, k)


@gpu
def test_linear_layouts_and_leading_axes():
    x, w, b, r, dy = linear_case(6 * 35, 96, 80, "bf16", 11)
    want = ops.linear(x, w, b, "silu", r)
    assert torch.equal(ops.linear(x.view(6, 35, 96), w, b, "silu", r.view(6, 35, 80)).view(-1, 80), want)
    wide = torch.zeros(210, 200, device=DEV, dtype=torch.bfloat16)
    wide[:, 16:112] = x
    assert torch.equal(ops.linear(wide[:, 16:112], w, b, "silu", r), want)                    # a row stride
    wide[:, 3:99] = x
    assert torch.equal(ops.linear(wide[:, 3:99], w, b, "silu", r), want)                      # unaligned rows
    assert torch.equal(ops.linear(x.t().contiguous().t(), w, b, "silu", r), want)             # columns outermost
    assert torch.equal(ops.linear(x, w.t().contiguous().t(), b, "silu", r), want)
    rr = r[:1].expand(210, 80)
    assert torch.equal(ops.linear(x, w, b, "silu", rr), ops.linear(x, w, b, "silu", rr.contiguous()))
    bb = torch.zeros(160, device=DEV, dtype=torch.bfloat16)
    bb[::2] = b
    assert torch.equal(ops.linear(x, w, bb[::2], "silu", r), want)
    # gradients of broadcast inputs and of expanded upstream gradients
    base = r[:1].clone().requires_grad_(True)
    xg, wg = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    ops.linear(xg, wg, b, "silu", base.expand(210, 80)).float().sum().backward()
    within(base.grad, torch.full((1, 80), 210.0, device=DEV), half_step(torch.bfloat16) * 210, "residual's gradient")
    one = torch.ones(210, 80, device=DEV, dtype=torch.bfloat16)
    linear_check(x, w, b, None, one, "silu", ops.linear(x, w, b, "silu"), (xg.grad, wg.grad, None))
    # the same tensor as input and residual
    sq = linear_case(70, 64, 64, "f32", 2)
    xs = sq[0].clone().requires_grad_(True)
    (g,) = torch.autograd.grad(ops.linear(xs, sq[1], sq[2], "none", xs), [xs], sq[4])
    within(g, sq[4].double() + sq[4].double() @ sq[1].double(), 1e-4, "x as its own residual")


@gpu
def test_lazily_negated_views():
    """torch keeps a conjugate's imaginary part as a view with a negation still to be done."""
    x, w, b, r, dy = (t.contiguous() for t in linear_case(70, 40, 24, "f32", 3))
    neg = torch._neg_view
    assert neg(x).is_neg()
    assert torch.equal(ops.linear(neg(x), neg(w), neg(b), "gelu", neg(r)), ops.linear(-x, -w, -b, "gelu", -r))
    assert torch.equal(ops.layer_norm(neg(x), neg(w[0]), neg(w[1])), ops.layer_norm(-x, -w[0], -w[1]))
    assert torch.equal(ops.checkpoint8(neg(x)).restore(), ops.checkpoint8(-x).restore())
    for f in (lambda t: ops.linear(t, w, b, "gelu"), lambda t: ops.layer_norm(t)):
        t = x.clone().requires_grad_()
        y = f(t)
        g = dy if y.shape == dy.shape else x
        want, got = torch.autograd.grad(y, t, -g, retain_graph=True)[0], torch.autograd.grad(y, t, neg(g))[0]
        assert torch.equal(got, want)


@gpu
def test_linear_subsets_of_gradients():
    x, w, b, r, dy = linear_case(90, 40, 24, "bf16", 4)
    for need in ((1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (1, 0, 1, 0), (0, 1, 0, 1)):
        ins = [v.clone().requires_grad_(bool(n)) for v, n in zip((x, w, b, r), need)]
        y = ops.linear(*ins[:3], "gelu", ins[3])
        got = iter(torch.autograd.grad(y, [v for v in ins if v.requires_grad], dy))
        dx, dw, db = (next(got) if n else None for n in need[:3])
        linear_check(x, w, b, r, dy, "gelu", y.detach(), (dx, dw, db))
        if need[3]:
            assert torch.equal(next(got), dy)


@gpu
def test_empty_sizes():
    w, b = torch.randn(5, 8, device=DEV, requires_grad=True), torch.randn(5, device=DEV, requires_grad=True)
    x = torch.zeros(0, 8, device=DEV, requires_grad=True)
    y = ops.linear(x, w, b, "gelu")
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], torch.zeros(0, 5, device=DEV))
    assert y.shape == (0, 5) and gx.shape == (0, 8) and not gw.any() and not gb.any()
    assert ops.linear(torch.zeros(3, 0, 8, device=DEV), w.detach(), b.detach()).shape == (3, 0, 5)
    assert ops.linear(torch.zeros(3, 8, device=DEV), torch.zeros(0, 8, device=DEV)).shape == (3, 0)
    xg = torch.zeros(3, 8, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(ops.linear(xg, torch.zeros(0, 8, device=DEV)), [xg], torch.zeros(3, 0, device=DEV))
    assert not g.any() and g.shape == (3, 8)
    n = torch.zeros(0, 12, device=DEV, requires_grad=True)
    lw = torch.ones(12, device=DEV, requires_grad=True)
    gn, gl = torch.autograd.grad(ops.layer_norm(n, lw), [n, lw], torch.zeros(0, 12, device=DEV))
    assert gn.shape == (0, 12) and not gl.any()
    for shape in ((0, 7), (4, 0), (0, 0), (2, 0, 5)):
        assert ops.checkpoint8(torch.zeros(shape, device=DEV)).restore().shape == shape


@gpu
def test_not_finite_inputs_stay_in_their_rows():
    for dt in DT:
        for M in (40, 200):
            x, w, b, _, dy = linear_case(M, 96, 72, dt, 6, residual=False)
            clean = ops.linear(x, w, b, "gelu")
            x[7, 3], x[11, 5] = float("nan"), float("inf")
            y = ops.linear(x, w, b, "relu")
            assert bool(y[7].isnan().all())
            y = ops.linear(x, w, b, "gelu")
            keep = torch.ones(M, dtype=torch.bool)
            keep[[7, 11]] = False
            assert torch.equal(y[keep], clean[keep]) and bool(y[7].isnan().all())
        n = torch.randn(30, 100, device=DEV).to(DT[dt])
        clean = ops.layer_norm(n)
        n[4, 9], n[8, 0] = float("nan"), -float("inf")
        y = ops.layer_norm(n)
        keep = torch.ones(30, dtype=torch.bool)
        keep[[4, 8]] = False
        assert torch.equal(y[keep], clean[keep]) and bool(y[4].isnan().all()) and bool(y[8].isnan().all())


# ------------------------------------------------------------------------------------------------ layer norm
NORM_SIZES = [(1, 1), (3, 2), (5, 31), (9, 64), (33, 65), (257, 128), (70, 100), (70, 256), (40, 257), (77, 512), (50, 771), (60, 1024), (40, 1025), (33, 2048),
              (20, 4096), (19, 4100), (12, 8192), (7, 5001), (5, 16384), (3000, 48), (1500, 768)]


def norm_check(x, w, b, dy, eps, y, grads, checkpoint8=False):
    t = x.dtype
    rows, D = x.shape
    x64 = x.detach().double()
    w64 = w.detach().double() if w is not None else torch.ones(D, device=x.device, dtype=torch.float64)
    b64 = b.detach().double() if b is not None else torch.zeros(D, device=x.device, dtype=torch.float64)
    mu = x64.mean(1, keepdim=True)
    var = ((x64 - mu) ** 2).mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    h = (x64 - mu) * rstd
    emu = 34 * U * x64.abs().mean(1, keepdim=True)
    ec = emu + U * (x64 - mu).abs() + U * (x64.abs() + mu.abs())
    # relative error of var + eps: the centred values' errors, the sum, eps itself as fp32
    erel = (2 * (ec * (x64 - mu).abs()).mean(1, keepdim=True) + (ec ** 2).mean(1, keepdim=True)) * rstd ** 2 + 36 * U
    eh = ec * rstd + h.abs() * (erel + 4 * U)
    out = half_step(t)
    want = h * w64 + b64
    within(y, want, (eh * w64.abs() + 3 * U * (h * w64).abs() + 3 * U * want.abs()) * (1 + out) + out * want.abs() + tiny(t), "y")
    if grads is None:
        return
    hs = h
    if checkpoint8:
        # the code of a value within eh of a tie may be either neighbour; where the group's largest value is within eh of a power of two, the step may differ too
        step = step8(h)
        hs = stored8(h)
        frac = (h / step - torch.floor(h / step) - 0.5).abs()
        eh = torch.where(frac * step <= eh, step, torch.zeros_like(step)) + 0.0 * eh
        m = torch.empty_like(h)
        for lo in range(0, D, 32):
            m[:, lo:lo + 32] = h[:, lo:lo + 32].abs().amax(1, keepdim=True)
        near = torch.minimum((m / torch.exp2(torch.floor(torch.log2(m.clamp(min=1e-30)))) - 1).abs(), (m / torch.exp2(torch.ceil(torch.log2(m.clamp(min=1e-30)))) - 1).abs()) <= 1e-4
        eh = torch.where(near, 2 * step, eh)
    dy64 = dy.double()
    g = dy64 * w64
    c1, c2 = g.mean(1, keepdim=True), (g * hs).mean(1, keepdim=True)
    e1 = 36 * U * g.abs().mean(1, keepdim=True)
    e2 = (g.abs() * eh).mean(1, keepdim=True) + 36 * U * (g * hs).abs().mean(1, keepdim=True)
    dx, dw, db = grads
    want = rstd * (g - c1 - hs * c2)
    scale = g.abs() + c1.abs() + (hs * c2).abs()
    tol = rstd * (e1 + hs.abs() * e2 + eh * c2.abs() + eh * e2 + 6 * U * scale) + want.abs() * 0 + rstd * scale * (erel + 4 * U)
    within(dx, want, tol * (1 + out) + out * want.abs() + tiny(t), "dx")
    if dw is not None:
        want = (dy64 * hs).sum(0)
        within(dw, want, (dy64.abs() * eh).sum(0) + 2 * (rows + 20) * U * (dy64.abs() * (hs.abs() + eh)).sum(0) + 2 * half_step(dw.dtype) * want.abs() + tiny(t), "dw")
    if db is not None:
        want = dy64.sum(0)
        within(db, want, 2 * (rows + 20) * U * dy64.abs().sum(0) + 2 * half_step(db.dtype) * want.abs() + tiny(t), "db")


def norm_case(rows, D, dt, seed, affine="same"):
    gen = torch.Generator().manual_seed(seed)
    t = DT[dt]
    x = (torch.randn(rows, D, generator=gen) * (0.5 + torch.rand(rows, 1, generator=gen)) + torch.randn(rows, 1, generator=gen)).to(t)
    pt = torch.float32 if affine == "f32" else t
    w = (1 + 0.3 * torch.randn(D, generator=gen)).to(pt) if affine not in ("none", "bias") else None
    b = (0.3 * torch.randn(D, generator=gen)).to(pt) if affine not in ("none", "weight") else None
    dy = torch.randn(rows, D, generator=gen).to(t)
    return [v.to(DEV) if v is not None else None for v in (x, w, b, dy)]


def run_norm(x, w, b, dy, eps, **kw):
    leaves = [v.requires_grad_(True) for v in (x, w, b) if v is not None]
    y = ops.layer_norm(x, w, b, eps, **kw)
    g = iter(torch.autograd.grad(y, leaves, dy))
    return y.detach(), tuple(next(g) if v is not None else None for v in (x, w, b))


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("i", range(len(NORM_SIZES)), ids=["x".join(map(str, s)) for s in NORM_SIZES])
def test_layer_norm_forward_and_gradients(dt, i):
    rows, D = NORM_SIZES[i]
    affine = ("same", "f32", "none", "weight", "bias")[i % 5]
    eps = (1e-5, 1e-12, 1e-3)[i % 3] if D > 2 else 1e-3
    x, w, b, dy = norm_case(rows, D, dt, i, affine)
    y, g = run_norm(x, w, b, dy, eps)
    norm_check(x, w, b, dy, eps, y, g)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b, eps), y)
    if dt != "f32":
        y8, g8 = run_norm(x, w, b, dy, eps, checkpoint8=True)
        assert torch.equal(y8, y)
        norm_check(x, w, b, dy, eps, y8, g8, checkpoint8=True)


@gpu
def test_layer_norm_constant_rows_and_layouts():
    x = torch.full((4, 96), 3.0, device=DEV)
    b = torch.randn(96, device=DEV)
    assert torch.equal(ops.layer_norm(x, None, b), b.expand(4, 96))                            # no spread: h = 0
    x, w, b, dy = norm_case(36, 160, "f16", 3)
    want = ops.layer_norm(x, w, b)
    wide = torch.zeros(36, 200, device=DEV, dtype=torch.float16)
    for lo in (8, 5):
        wide[:, lo:lo + 160] = x
        got = ops.layer_norm(wide[:, lo:lo + 160], w, b)
        norm_check(x, w, b, None, 1e-5, got, None)
        if lo == 8:
            assert torch.equal(got, want)
    assert torch.equal(ops.layer_norm(x.view(4, 9, 160), w, b).view(36, 160), want)
    norm_check(x, w, b, None, 1e-5, ops.layer_norm(x.t().contiguous().t(), w, b), None)
    xg = x.clone().requires_grad_(True)
    ops.layer_norm(xg, w, b).sum().backward()                                                   # an expanded upstream gradient
    one = torch.ones(36, 160, device=DEV, dtype=torch.float16)
    norm_check(x, w, b, one, 1e-5, want, (xg.grad, None, None))


# ------------------------------------------------------------------------------------------------ 8-bit checkpoints
@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 31), (5, 32), (9, 33), (64, 96), (77, 512), (10, 1000), (1, 4099)])
def test_checkpoint8_values_are_the_definition(dt, rows, D):
    gen = torch.Generator().manual_seed(rows + D)
    x = torch.randn(rows, D, generator=gen) * torch.exp2(torch.randint(-20, 12, (rows, D), generator=gen).float())
    x[torch.rand(rows, D, generator=gen) < 0.3] = 0.0
    x[0] = 0.0 if rows > 1 else x[0]                                   # a row of zeros
    x = x.to(DT[dt]).to(DEV)
    c = ops.checkpoint8(x)
    assert c.codes.shape == (rows, D) and c.exps.shape == (rows, (D + 31) // 32) and c.codes.dtype == torch.int8 and c.exps.dtype == torch.uint8
    want = stored8(x.double())
    assert c.restore().dtype == x.dtype and torch.equal(c.restore().double(), want)
    assert torch.equal(c.restore(torch.float32).double(), want)
    within(want, x.double(), step8(x.double()) * (0.5 + 0.5 * (x.double().abs() > 127.5 * step8(x.double()))), "half a step")


@gpu
@pytest.mark.parametrize("dt", list(DT))
def test_checkpoint8_extremes(dt):
    t = DT[dt]
    big, small = torch.finfo(t).max, torch.finfo(t).smallest_normal * torch.finfo(t).eps
    for D in (64, 45):
        x = torch.ones(4, D, device=DEV, dtype=t)
        x[0, 0], x[1, 2], x[2, 40] = float("inf"), float("nan"), -float("inf")
        v = ops.checkpoint8(x).restore()
        assert bool(v[0, :32].isnan().all()) and bool(v[1, :32].isnan().all()) and bool(v[2, 32:].isnan().all())
        assert torch.equal(v[0, 32:], x[0, 32:]) and torch.equal(v[2, :32], x[2, :32]) and torch.equal(v[3], x[3])
        x = torch.full((2, D), big, device=DEV, dtype=t)
        x[1] = small
        v = ops.checkpoint8(x).restore()
        assert torch.equal(v.double(), stored8(x.double())) and bool(v.isfinite().all())
        assert torch.equal(v[1], x[1]) or t != torch.float16               # (fp16's subnormals are exact; below 2^-133 fp32 and bf16 round to 0)
    x = torch.randn(6, 7, 40, device=DEV).to(t)
    assert torch.equal(ops.checkpoint8(x).restore(), ops.checkpoint8(x.reshape(42, 40)).restore().view(6, 7, 40))
    assert torch.equal(ops.checkpoint8(x.transpose(0, 1)).restore(), ops.checkpoint8(x).restore().transpose(0, 1))
    assert torch.equal(ops.checkpoint8(x[..., 3:35]).restore(), ops.checkpoint8(x[..., 3:35].contiguous()).restore())


@gpu
def test_checkpoint8_poisons_the_weight_gradient():
    """An overflowed activation must not disappear in 8 bits: the weight gradient of its group is NaN."""
    x, w, b, r, dy = linear_case(80, 64, 16, "f16", 1)
    x[3, 40] = float("inf")
    w.requires_grad_(True)
    (g,) = torch.autograd.grad(ops.linear(x, w, b, checkpoint8=True), [w], dy)
    assert bool(g[:, 32:].isnan().all()) and bool(g[:, :32].isfinite().all())


# ------------------------------------------------------------------------------------------------ together, streams, graphs
def block(x, p, c8=False):
    """A residual block as a tower runs it: norm, widening product with activation, narrowing product onto the residual stream, norm."""
    h = ops.layer_norm(x, p["n1w"], p["n1b"], checkpoint8=c8)
    h = ops.linear(h, p["w1"], p["b1"], "gelu", checkpoint8=c8)
    y = ops.linear(h, p["w2"], p["b2"], residual=x, checkpoint8=c8)
    return ops.layer_norm(y, p["n2w"], p["n2b"], checkpoint8=c8)


def block_params(D, F, dt, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    p = {"n1w": 1 + 0.1 * r(D), "n1b": 0.1 * r(D), "w1": r(F, D) / D ** 0.5, "b1": 0.1 * r(F), "w2": r(D, F) / F ** 0.5, "b2": 0.1 * r(D), "n2w": 1 + 0.1 * r(D),
         "n2b": 0.1 * r(D)}
    return {k: v.to(DEV, DT[dt]).requires_grad_(True) for k, v in p.items()}


def block64(x, p):
    ln = lambda v, w, b: torch.nn.functional.layer_norm(v, (v.shape[-1],), w, b, 1e-5)
    h = torch.nn.functional.gelu(ln(x, p["n1w"], p["n1b"]) @ p["w1"].T + p["b1"])
    return ln(h @ p["w2"].T + p["b2"] + x, p["n2w"], p["n2b"])


@gpu
@pytest.mark.parametrize("dt,c8,bound", [("f32", False, 1e-4), ("bf16", False, 0.03), ("f16", False, 0.004), ("bf16", True, 0.06), ("f16", True, 0.05)])
def test_a_block_and_its_gradients_against_64_bits(dt, c8, bound):
    """Relative 2-norms.  A gradient passes about ten roundings: of the type (2^-9 and 2^-12 rms below half a step each), and with 8 bits of 1/384 in a' and
    up to 1/128 of a group's maximum in what is stored, a percent or two of a typical value each."""
    D, F, M = 160, 416, 231
    p = block_params(D, F, dt)
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(3, M // 3, D, generator=gen).to(DEV, DT[dt]).requires_grad_(True)
    dy = torch.randn(3, M // 3, D, generator=gen).to(DEV, DT[dt])
    y = block(x, p, c8)
    got = torch.autograd.grad(y, [x, *p.values()], dy)
    x64 = x.detach().double().requires_grad_(True)
    p64 = {k: v.detach().double().requires_grad_(True) for k, v in p.items()}
    y64 = block64(x64, p64)
    want = torch.autograd.grad(y64, [x64, *p64.values()], dy.double())
    for name, a, b in zip(["y", "x", *p], [y, *got], [y64, *want]):
        rel = float((a.detach().double() - b.detach()).norm() / b.detach().norm())
        assert rel <= bound, (name, rel)


@gpu
def test_same_bits_again_and_on_another_stream():
    p = block_params(128, 320, "bf16")
    x = torch.randn(700, 128, device=DEV).bfloat16().requires_grad_(True)
    dy = torch.randn(700, 128, device=DEV).bfloat16()
    run = lambda: [t.detach().clone() for t in (lambda y: (y, *torch.autograd.grad(y, [x, *p.values()], dy)))(block(x, p, True))]
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = run()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(first, other))


@gpu
def test_captured_forward_and_backward_replays():
    p = block_params(96, 200, "f16", 3)
    x = torch.randn(150, 96, device=DEV).half().requires_grad_(True)
    dy = torch.randn(150, 96, device=DEV).half()
    leaves = [x, *p.values()]

    def step():
        y = block(x, p)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                                  # two graphs of the same work: no scratch memory is shared
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(150, 96, device=DEV, generator=torch.Generator(device=DEV).manual_seed(k)))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for g, outs in graphs if k % 2 else reversed(graphs):
            g.replay()
        torch.cuda.synchronize()
        for g, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want)), k


@gpu
def test_capture_with_a_live_eager_graph_is_refused():
    """Autograd would have to join the default stream, on which the leaf's gradient node lives, to the capture."""
    w = torch.randn(8, 16, device=DEV, requires_grad=True)
    x = torch.randn(70, 16, device=DEV)
    alive = ops.linear(x, w)                                            # built on the default stream
    g = torch.cuda.CUDAGraph()
    n = torch.ones(16, device=DEV, requires_grad=True)
    alive_n = ops.layer_norm(x, n)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    refused = []
    with torch.cuda.graph(g, stream=s):
        for f in (lambda: ops.linear(x, w), lambda: ops.layer_norm(x, n)):
            try:
                f()
            except _lib.LsdmError as e:
                refused.append(str(e))
        with torch.no_grad():
            y = ops.linear(x, w)                                        # inference takes no part in autograd
    assert len(refused) == 2 and all("live autograd graph" in r for r in refused)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, alive.detach())
    torch.autograd.grad(alive, [w], torch.ones_like(alive))             # the eager graph is as it was
    torch.autograd.grad(alive_n, [n], torch.ones_like(alive_n))


@gpu
def test_differentiable_once():
    w = torch.randn(8, 16, device=DEV, requires_grad=True)
    x = torch.randn(70, 16, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(ops.linear(x, w, None, "gelu").sum(), [x], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


@gpu
def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the first and the last rows against the same rows alone."""
    rows, D = 140000, 16384
    x = torch.empty(rows, D, device=DEV, dtype=torch.bfloat16)
    x[:2].normal_()
    x[-2:].normal_()
    x[2:-2].zero_()
    y = ops.layer_norm(x)
    assert torch.equal(y[-2:], ops.layer_norm(x[-2:].clone())) and torch.equal(y[:2], ops.layer_norm(x[:2].clone()))
    del y
    c = ops.checkpoint8(x)
    v = c.restore()
    assert torch.equal(v[-2:], ops.checkpoint8(x[-2:].clone()).restore()) and not bool(v[2].any())
    del c, v, x
    M, K, N = 1 << 20, 64, 2056
    x = torch.zeros(M, K, device=DEV, dtype=torch.bfloat16)
    x[-300:].normal_()
    w, b = torch.randn(N, K, device=DEV, dtype=torch.bfloat16), torch.randn(N, device=DEV, dtype=torch.bfloat16)
    y = ops.linear(x, w, b, "relu")
    linear_check(x[-300:], w, b, None, None, "relu", y[-300:])
    assert torch.equal(y[0], ops.linear(x[:1], w, b, "relu")[0])


@gpu
def test_c_entries_write_their_outputs_only():
    """The C entry points on odd sizes inside larger buffers: what lies behind the outputs (and the scratch memory) stays as it was."""
    lib = _lib.load()
    M, K, N = 83, 37, 45
    es = 2
    buf = lambda n, dt: torch.full((n + 64,), 77 if dt == torch.uint8 else 7.0, device=DEV, dtype=dt)
    x, w, b, r, dy = (t.contiguous() for t in linear_case(M, K, N, "bf16", 8))
    y, d = buf(M * N, torch.bfloat16), buf(M * N, torch.bfloat16)
    need = lib.lsdm_linear_workspace(1, 256 | 512, M, N, K)
    ws = buf(need, torch.uint8)
    st = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()
    assert lib.lsdm_linear(0, 1, 2, 0, M, N, K, p(x), K, p(w), K, p(b), p(r), N, p(y), p(d), p(ws), need, st) == 0
    linear_check(x, w, b, r, dy, "gelu", y[:M * N].view(M, N))
    assert bool((y[M * N:] == 7).all()) and bool((d[M * N:] == 7).all()) and bool((ws[need:] == 77).all())
    flags = 4 | 8 | 16 | 32 | 64
    need = lib.lsdm_linear_workspace(1, flags | 256 | 512 | 1024, M, N, K)
    ws = buf(need, torch.uint8)
    dx, dw, db = buf(M * K, torch.bfloat16), buf(N * K, torch.bfloat16), buf(N, torch.bfloat16)
    assert lib.lsdm_linear_backward(0, 1, 0, M, N, K, p(dy), N, p(d), p(x), K, None, None, p(w), K, p(dx), p(dw), p(db), p(ws), need, st) == 0
    linear_check(x, w, b, r, dy, "gelu", y[:M * N].view(M, N), (dx[:M * K].view(M, K), dw[:N * K].view(N, K), db[:N]))
    for t, n in ((dx, M * K), (dw, N * K), (db, N)):
        assert bool((t[n:] == 7).all())
    assert bool((ws[need:] == 77).all())
    assert lib.lsdm_linear_backward(0, 1, 0, M, N, K, p(dy), N, p(d), p(x), K, None, None, p(w), K, p(dx), p(dw), p(db), p(ws), need - 1, st) == -1
    assert b"workspace" in lib.lsdm_last_error(None)
    rows, D = 29, 83
    n, nw, nb, ndy = (t.contiguous() for t in norm_case(rows, D, "f16", 2))
    y, mean, rstd = buf(rows * D, torch.float16), buf(rows, torch.float32), buf(rows, torch.float32)
    codes, exps = buf(rows * D, torch.uint8), buf(rows * 3, torch.uint8)
    assert lib.lsdm_layer_norm(0, 2, 0, rows, D, p(n), D, p(nw), p(nb), 1e-5, p(y), p(mean), p(rstd), p(codes), p(exps), st) == 0
    need = lib.lsdm_layer_norm_workspace(rows, D)
    ws, dx, dw, db = buf(need, torch.uint8), buf(rows * D, torch.float16), buf(D, torch.float16), buf(D, torch.float16)
    assert lib.lsdm_layer_norm_backward(0, 2, 0, rows, D, p(ndy), D, p(n), D, None, None, p(nw), p(mean), p(rstd), p(dx), p(dw), p(db), p(ws), need, st) == 0
    norm_check(n, nw, nb, ndy, 1e-5, y[:rows * D].view(rows, D), (dx[:rows * D].view(rows, D), dw[:D], db[:D]))
    for t, k, v in ((y, rows * D, 7), (mean, rows, 7), (rstd, rows, 7), (codes, rows * D, 77), (exps, rows * 3, 77), (dx, rows * D, 7), (dw, D, 7), (db, D, 7), (ws, need, 77)):
        assert bool((t[k:] == v).all())
    assert lib.lsdm_pack8(0, 2, rows, D, p(n), D, p(codes), p(exps), st) == 0 and lib.lsdm_unpack8(0, 2, rows, D, p(codes), p(exps), p(y), st) == 0
    assert torch.equal(y[:rows * D].view(rows, D).double(), stored8(n.double())) and bool((y[rows * D:] == 7).all()) and bool((codes[rows * D:] == 77).all())


# ------------------------------------------------------------------------------------------------ refusals
def test_host_tensors_and_bad_arguments_are_refused_without_a_device():
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    for f in (lambda: ops.linear(x, w), lambda: ops.layer_norm(x), lambda: ops.checkpoint8(x), lambda: ops.Checkpoint8(x.to(torch.int8), x, x.shape, x.dtype).restore()):
        with pytest.raises(_lib.LsdmError, match="HIP device"):
            f()
    with pytest.raises(ValueError, match="activation"):
        ops.linear(x, w, activation="swish")
    with pytest.raises(TypeError):
        ops.linear([1.0], w)


def test_c_entries_refuse_bad_arguments_before_they_touch_a_device():
    lib = _lib.load()
    P = C.c_void_p(4096)                    # never dereferenced: every call below fails its checks first
    bad = lambda rc, word: (rc == -1 and word in lib.lsdm_last_error(None).decode()) or pytest.fail("%d %s" % (rc, lib.lsdm_last_error(None)))
    lin = lambda dt=1, act=0, M=8, N=8, K=8, x=P, ldx=8, w=P, ldw=8, r=None, ldr=0, y=P, ws=None, n=0: lib.lsdm_linear(0, dt, act, 0, M, N, K, x, ldx, w, ldw, None, r, ldr, y, None, ws, n, None)
    bad(lin(dt=3), "dtype")
    bad(lin(act=7), "activation")
    bad(lin(act=-1), "activation")
    bad(lin(M=0), "sizes")
    bad(lin(K=(1 << 30) + 1), "sizes")
    bad(lin(x=None), "NULL")
    bad(lin(y=None), "NULL")
    bad(lin(ldx=7), "row stride")
    bad(lin(ldw=7), "row stride")
    bad(lin(r=P, ldr=7), "row stride")
    bad(lin(M=100, K=7, ldx=7, ldw=7), "workspace")
    back = lambda M=8, dy=P, lddy=8, x=P, ldx=8, codes=None, exps=None, w=P, ldw=8, dx=P, dw=P, n=0: lib.lsdm_linear_backward(
        0, 1, 0, M, 8, 8, dy, lddy, None, x, ldx, codes, exps, w, ldw, dx, dw, None, None, n, None)
    bad(back(dy=None), "dy")
    bad(back(lddy=4), "dy")
    bad(back(w=None), "needs w")
    bad(back(x=None), "needs x")
    bad(back(x=None, codes=P), "needs x")
    bad(back(x=None, codes=P, exps=P), "workspace")
    norm = lambda D=8, x=P, ldx=8, y=P, eps=1e-5, codes=None: lib.lsdm_layer_norm(0, 1, 0, 4, D, x, ldx, None, None, eps, y, None, None, codes, None, None)
    bad(norm(D=0), "width")
    bad(norm(D=16385, ldx=20000), "width")
    bad(norm(x=None), "NULL")
    bad(norm(ldx=3), "NULL")
    bad(norm(eps=-1.0), "eps")
    bad(norm(eps=float("nan")), "eps")
    bad(norm(codes=P), "together")
    bad(lib.lsdm_layer_norm_backward(0, 1, 0, 4, 8, P, 8, None, 8, None, None, None, P, P, P, None, None, None, 0, None), "needed")
    bad(lib.lsdm_layer_norm_backward(0, 1, 0, 4, 8, P, 8, P, 8, None, None, None, P, P, P, P, None, None, 0, None), "workspace")
    bad(lib.lsdm_pack8(0, 1, 0, 8, P, 8, P, P, None), "pack8")
    bad(lib.lsdm_unpack8(0, 5, 1, 8, P, P, P, None), "unpack8")
    bad(lin(N=(1 << 25) + 1, r=P, ldr=1 << 26), "sizes")
    bad(lib.lsdm_pack8(0, 1, 1 << 31, 32, P, 32, P, P, None), "pack8")
    bad(lib.lsdm_unpack8(0, 1, 1 << 31, 32, P, P, P, None), "unpack8")
    # sizes whose tiles are more threads than a launch takes choose a larger tile, or are refused
    assert lib.lsdm_linear_workspace(0, 0, 1 << 30, 1, 8) == 0
    bad(lin(dt=0, M=1 << 30, N=1 << 20, ldw=8), "tiles")
    assert lib.lsdm_linear_workspace(1, 0, 0, 8, 8) == -1 and lib.lsdm_layer_norm_workspace(4, 0) == -1
    assert lib.lsdm_linear_workspace(1, 0, 64, 8, 7) == 0 and lib.lsdm_linear_workspace(1, 0, 1000, 512, 512) >= 0


@gpu
def test_refusals_on_the_device():
    x, w = torch.zeros(2, 4, device=DEV), torch.zeros(3, 4, device=DEV)
    cases = [(lambda: ops.linear(x, w.t()), "expected x"), (lambda: ops.linear(x, w.half()), "dtype"), (lambda: ops.linear(x.int(), w), "dtype"),
             (lambda: ops.linear(x.double(), w.double()), "dtype"), (lambda: ops.linear(x, w, torch.zeros(4, device=DEV)), "bias"),
             (lambda: ops.linear(x, w, torch.zeros(3, device=DEV, dtype=torch.float16)), "bias"), (lambda: ops.linear(x, w, residual=torch.zeros(2, 4, device=DEV)), "residual"),
             (lambda: ops.linear(x, w, residual=torch.zeros(3, device=DEV)), "residual"), (lambda: ops.linear(x, w, residual=torch.zeros(2, 3, device=DEV).half()), "dtype"),
             (lambda: ops.linear(torch.zeros(2, 0, device=DEV), torch.zeros(3, 0, device=DEV)), "columns"), (lambda: ops.linear(x, w[0]), "expected x"),
             (lambda: ops.layer_norm(x, torch.ones(3, device=DEV)), "weight"), (lambda: ops.layer_norm(x, eps=-1.0), "eps"), (lambda: ops.layer_norm(x, checkpoint8=True), "checkpoint8"),
             (lambda: ops.layer_norm(torch.zeros(2, 16385, device=DEV)), "last axis"), (lambda: ops.layer_norm(torch.zeros(2, 0, device=DEV)), "last axis"),
             (lambda: ops.layer_norm(x.half(), torch.ones(4, device=DEV), torch.ones(4, device=DEV).half()), "same dtype"), (lambda: ops.checkpoint8(x.long()), "dtype"),
             (lambda: ops.checkpoint8(torch.zeros((), device=DEV)), "axis"), (lambda: ops.checkpoint8(x).restore(torch.int8), "dtype")]
    for f, word in cases:
        with pytest.raises(ValueError, match=word):
            f()
    for f in (lambda: ops.linear(x, w.cpu()), lambda: ops.linear(x, w, torch.zeros(3)), lambda: ops.layer_norm(x, torch.ones(4))):
        with pytest.raises(_lib.LsdmError, match="is on"):
            f()


# ------------------------------------------------------------------------------------------------ the text towers
def bert(layers=2, hidden=96, heads=4, inner=200, dropout=0.0):
    transformers = pytest.importorskip("transformers")
    cfg = transformers.BertConfig(vocab_size=40, hidden_size=hidden, num_hidden_layers=layers, num_attention_heads=heads, intermediate_size=inner,
                                  hidden_dropout_prob=dropout, attention_probs_dropout_prob=0.0, attn_implementation="eager")
    torch.manual_seed(0)
    return transformers.BertModel(cfg)


def clip_block():
    """A residual block of the structure the CLIP package publishes (its LayerNorm evaluates in its parameters' type whatever comes in)."""
    import torch.nn as nn

    class NormClip(nn.LayerNorm):
        def forward(self, x):
            return super().forward(x.to(self.weight.dtype)).to(x.dtype)
    NormClip.__module__ = "clip.model"

    class QuickGELU(nn.Module):
        def forward(self, x):
            return x * torch.sigmoid(1.702 * x)

    class ResidualAttentionBlock(nn.Module):
        def __init__(self, d, heads):
            super().__init__()
            from collections import OrderedDict
            self.attn = nn.MultiheadAttention(d, heads)
            self.ln_1, self.ln_2 = NormClip(d), NormClip(d)
            self.mlp = nn.Sequential(OrderedDict([("c_fc", nn.Linear(d, 4 * d)), ("gelu", QuickGELU()), ("c_proj", nn.Linear(4 * d, d))]))

        def attention(self, x):
            return self.attn(x, x, x, need_weights=False)[0]

        def forward(self, x):
            x = x + self.attention(self.ln_1(x))
            return x + self.mlp(self.ln_2(x))
    torch.manual_seed(1)
    return ResidualAttentionBlock(64, 4)


def test_use_kernels_replaces_layers_in_place():
    m = bert()
    before = {k: v.clone() for k, v in m.state_dict().items()}
    assert use_kernels(m) is m and use_kernels(m, checkpoint8=True) is m
    kinds = [type(v) for v in m.modules()]
    assert torch.nn.Linear not in kinds and torch.nn.LayerNorm not in kinds and kinds.count(Linear) == 2 * 6 + 1 and kinds.count(LayerNorm) == 1 + 2 * 2
    assert all(v.checkpoint8 for v in m.modules() if isinstance(v, (Linear, LayerNorm)))
    assert list(m.state_dict()) == list(before) and all(torch.equal(v, before[k]) for k, v in m.state_dict().items())
    b = use_kernels(clip_block())
    assert type(b.ln_1) is LayerNorm and type(b.mlp.c_fc) is Linear and b._kernel_activation == "quick_gelu" and type(b.attn.out_proj) is not Linear
    with pytest.raises(ValueError, match="no Linear"):
        use_kernels(torch.nn.ReLU())
    with pytest.raises(_lib.LsdmError, match="HIP device"):
        m(torch.zeros(1, 3, dtype=torch.long))
    kept = torch.nn.Sequential(torch.nn.LayerNorm([3, 4]), torch.nn.Linear(4, 4))
    use_kernels(kept)
    assert type(kept[0]) is torch.nn.LayerNorm                           # a norm over several axes is not the operator


class Scaled(torch.nn.Linear):
    """A dense layer of a user's own kind (adapters, quantised layers)."""
    def forward(self, x):
        return 2.0 * super().forward(x)


def test_blocks_that_are_not_the_fused_pattern_keep_their_forward():
    m = bert(layers=1)
    layer = m.encoder.layer[0]
    layer.intermediate.dense.__class__ = Scaled
    layer.output.dense.__class__ = Scaled
    m.pooler.extra = torch.nn.Identity()
    use_kernels(m)
    assert "forward" in vars(layer.attention.output) and type(layer.intermediate.dense) is Scaled
    assert not any("forward" in vars(b) for b in (layer.intermediate, layer.output, m.pooler))
    b = clip_block()
    b.ls_1 = torch.nn.Identity()                                         # a scale on a branch
    c = clip_block()
    c.mlp.c_proj.__class__ = Scaled
    d = clip_block()
    d.mlp.add_module("drop", torch.nn.Dropout(0.5))
    assert not any("forward" in vars(use_kernels(v)) for v in (b, c, d)) and "forward" in vars(use_kernels(clip_block()))


def test_a_tower_on_the_operators_can_be_copied_and_pickled():
    m = use_kernels(bert(layers=1))
    for other in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        block, own = m.encoder.layer[0].intermediate, other.encoder.layer[0].intermediate
        assert type(own.dense) is Linear and own.dense is not block.dense and own.forward.args[0] is own and torch.equal(own.dense.weight, block.dense.weight)


@gpu
def test_bert_tower_on_the_operators():
    """Padded prompts of different lengths; relative 2-norms: two layers of about ten operations, each off by a few fp32 steps of a typical sum."""
    ids = torch.randint(1, 40, (3, 17), generator=torch.Generator().manual_seed(2))
    mask = torch.ones(3, 17, dtype=torch.long)
    mask[1, 9:] = 0
    mask[2, 1:] = 0
    ref = bert().eval().double()
    with torch.no_grad():
        want = ref(input_ids=ids, attention_mask=mask)
        m = use_kernels(bert().eval().to(DEV))
        got = m(input_ids=ids.to(DEV), attention_mask=mask.to(DEV))
    rel = lambda a, b: float((a.cpu().double() - b).norm() / b.norm())
    assert rel(got.pooler_output, want.pooler_output) <= 1e-5 and rel(got.last_hidden_state, want.last_hidden_state) <= 1e-5
    # training: gradients of every parameter, with dropout's branch taken where the module asks for it
    for dt, c8, bound in (("f32", False, 1e-4), ("bf16", True, 0.15)):
        ref, m = bert().train().double(), use_kernels(bert().train().to(DEV, DT[dt]), checkpoint8=False if dt == "f32" else c8)
        ref(input_ids=ids, attention_mask=mask).pooler_output.square().sum().backward()
        m(input_ids=ids.to(DEV), attention_mask=mask.to(DEV)).pooler_output.square().sum().backward()
        num = den = 0.0
        for (name, a), (_, b) in zip(m.named_parameters(), ref.named_parameters()):
            assert (a.grad is None) == (b.grad is None), name
            if b.grad is not None:
                num += float((a.grad.cpu().double() - b.grad).square().sum())
                den += float(b.grad.square().sum())
        assert math.sqrt(num / den) <= bound, (dt, math.sqrt(num / den))
    m = use_kernels(bert(dropout=0.5).train().to(DEV))
    assert bool(m(input_ids=ids.to(DEV), attention_mask=mask.to(DEV)).pooler_output.isfinite().all())


@gpu
def test_clip_block_on_the_operators():
    x = torch.randn(11, 5, 64, generator=torch.Generator().manual_seed(4))
    ref = clip_block().eval()
    with torch.no_grad():
        want = ref.double()(x.double())
        got = use_kernels(clip_block().eval()).to(DEV)(x.to(DEV))
        rel = lambda a: float((a.cpu().double() - want).norm() / want.norm())
        assert rel(got) <= 1e-5
        half = clip_block().eval().to(DEV).half()
        for n in (half.ln_1, half.ln_2):
            n.float()                                                    # (the package keeps the norms' parameters in fp32)
        assert rel(use_kernels(half)(x.to(DEV).half())) <= 4e-3          # a dozen roundings of 2^-11


@gpu
def test_the_models_text_hook_runs_on_the_operators(tmp_path, monkeypatch):
    """SceneDiffusionModel(text_kernels=True): the same prompts through the same (randomly initialised, locally saved) tower, eager and on the operators."""
    transformers = pytest.importorskip("transformers")
    monkeypatch.setenv("HF_HUB_OFFLINE", "1")
    monkeypatch.chdir(tmp_path)
    d = tmp_path / "bert-base-uncased"
    d.mkdir()
    vocab = ["[PAD]", "[UNK]", "[CLS]", "[SEP]", "[MASK]"] + "a the chair table sofa bed sit on in next to person lying ##s walk near".split()
    (d / "vocab.txt").write_text("\n".join(vocab) + "\n")
    torch.manual_seed(0)
    transformers.BertModel(transformers.BertConfig(vocab_size=len(vocab), hidden_size=768, num_hidden_layers=2, num_attention_heads=12,
                                                   intermediate_size=1024)).save_pretrained(str(d))
    from lsdm_amd.model.sdm import SceneDiffusionModel
    texts = ["a person near the chair", "lying in bed", "walk"]
    feats = []
    for kernels in (False, True):
        m = SceneDiffusionModel(clip_dim=768, pcd_dim=3, text_encoder_type="BERT", text_kernels=kernels)
        feats.append(m._encode_text(texts, 3, torch.device(DEV)))
    a, b = feats
    assert a.shape == b.shape == (3, 768) and float((a - b).norm() / a.norm()) <= 2e-5
