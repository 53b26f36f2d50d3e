"""The public operators where values are far from one: saturated activations and their derivatives, rows whose squares leave the range of fp32.
Every bound is added up from the roundings of the evaluation, relative to the value itself: u = 2^-24 for an fp32 operation."""
import math

import pytest
import torch

import test_ops as base
from lsdm_amd import ops

gpu = pytest.mark.gpu
DEV, U, DT = base.DEV, base.U, base.DT
half_step, within = base.half_step, base.within


@pytest.fixture(autouse=True)
def _grad_mode():
    with torch.enable_grad():
        yield


def through(act, z, dt, checkpoint8=False):
    """y = a(z) and a'(z) as the operator has them: z comes in as an fp32 bias under an input of zeros, one row, and a'(z) out as the bias' gradient, which is
    summed in fp32 and not rounded to the operands' type."""
    t = DT[dt]
    x, w = torch.zeros(1, 1, device=DEV, dtype=t), torch.ones(z.numel(), 1, device=DEV, dtype=t)
    b = z.to(DEV, torch.float32).clone().requires_grad_(True)
    y = ops.linear(x, w, b, act, checkpoint8=checkpoint8)
    (d,) = torch.autograd.grad(y, [b], torch.ones_like(y))
    return y.detach().view(-1), d


def phi64(z):
    """The normal distribution function through erfc (torch's ndtr is 1 + erf, which is 0 from z = -8.3 on)."""
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))


def act64(act, z):
    if act == "gelu":
        return z * phi64(z), phi64(z) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return base.act64(act, z)


def grid(lo, hi, n=4001):
    return torch.linspace(lo, hi, n).float()


# fp32: y and a' relative to the value.  exp of an exact argument and a division are off by a few u; where the argument itself is a rounded product p
# (gelu: z / sqrt(2), z^2 / 2), its rounding costs |p|' s change of the logarithm, 2 u z^2 for both of gelu's factors.  The two terms of a'(z) may cancel, so
# its bound goes by their magnitudes.
@gpu
@pytest.mark.parametrize("act,lo,hi", [("gelu", -9.0, -2.0), ("gelu", 2.0, 9.0), ("sigmoid", -60.0, -3.0), ("sigmoid", 3.0, 60.0), ("tanh", -30.0, -1.0), ("tanh", 1.0, 30.0),
                                       ("silu", -60.0, -3.0), ("silu", 3.0, 60.0), ("quick_gelu", -40.0, -2.0), ("quick_gelu", 2.0, 40.0)])
def test_tails_in_fp32(act, lo, hi):
    z = grid(lo, hi)
    y, d = through(act, z, "f32")
    z = z.to(DEV).double()
    want_y, want_d = act64(act, z)
    if act == "gelu":
        pdf = z.abs() * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        phi = phi64(z)
        ry, sd = 2 * z * z + 16, (2 * z * z + 16) * (phi + pdf)
    elif act in ("silu", "quick_gelu"):
        c = 1.702 if act == "quick_gelu" else 1.0
        s = torch.special.expit(c * z)
        ry = 16 + 2 * c * z.abs()                          # (1.702 z is a rounded product)
        sd = ry * s * (1 + c * z.abs() * torch.special.expit(-c * z))
    else:
        ry = torch.full_like(z, 16.0)
        sd = ry * want_d
    within(y, want_y, ry * U * want_y.abs(), "y")
    within(d, want_d, sd * U, "a'")


# 16 bits: a'(z) is kept in a form that is never coarser than half a step of bf16 (2^-8 of the value) down to 2^-23, and 2^-6 down to 2^-31.7; the functions
# themselves are good to 1e-4 of their terms over these ranges (gelu: 7.1.26's polynomial far out; the others: exp2 of a rounded product).
@gpu
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("act,lo,hi", [("gelu", -5.6, -0.9), ("sigmoid", -22.0, 0.0), ("sigmoid", 0.0, 22.0), ("tanh", -11.0, 0.0), ("tanh", 0.0, 11.0), ("silu", -25.0, -1.5),
                                       ("quick_gelu", -15.0, -1.0)])
def test_small_derivatives_in_16_bits(act, lo, hi, dt):
    z = grid(lo, hi)
    _, d = through(act, z, dt)
    z = z.to(DEV).double()
    _, want = act64(act, z)
    terms = want.abs()
    if act == "gelu":
        terms = phi64(z) + z.abs() * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    elif act in ("silu", "quick_gelu"):
        c = 1.702 if act == "quick_gelu" else 1.0
        terms = torch.special.expit(c * z) * (1 + c * z.abs())
    rel = torch.where(want.abs() >= 2.0 ** -23, 2.0 ** -8, 2.0 ** -6)
    within(d, want, rel * want.abs() + 1e-4 * terms + 2.0 ** -40, "a'")
    assert bool((d != 0).all() | (want.abs() < 2.0 ** -40).any())


@gpu
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_kept_derivatives_near_one(dt):
    """... and a'(z) itself keeps 2^-13 of the value from 1/32 up, 0 and 1 exactly, and NaN."""
    for act in ("gelu", "quick_gelu", "silu", "sigmoid", "tanh"):
        z = grid(-1.5, 4.0)
        _, d = through(act, z, dt)
        _, want = act64(act, z.to(DEV).double())
        big = want.abs() >= 1.0 / 32
        within(d[big], want[big], 2.0 ** -13 * want[big].abs() + 1.2e-6 * (1 + z.to(DEV).double()[big].abs()), act)
    _, d = through("relu", torch.tensor([-3.0, -0.0, 0.0, 1e-30, 5.0, float("inf"), -float("inf")]), dt)
    assert d.tolist() == [0, 0, 0, 1, 1, 1, 0]
    for act in ("gelu", "quick_gelu", "silu", "sigmoid", "tanh"):
        _, d = through(act, torch.tensor([float("nan"), 1.0]), dt)
        assert bool(d[0].isnan()) and bool(d[1].isfinite())
    for act, ends in (("sigmoid", [0, 0]), ("tanh", [0, 0])):
        for inf in (float("inf"), 1e30):
            y, d = through(act, torch.tensor([-inf, inf]), dt)
            assert d.tolist() == ends and y[1] == 1


# ------------------------------------------------------------------------------------------------ layer norm: squares beyond fp32's range
WIDTHS = [3, 8, 40, 64, 100, 256, 300, 512, 771, 1024, 1500, 2048, 2051, 4096, 5001, 8192, 16384]


def rows_of_scales(D, dt, scales, seed):
    """Rows of standard normal values times 2^k for every k of `scales`, in turn, between rows of ordinary ones."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(len(scales), D, generator=gen) + 0.5 * torch.randn(len(scales), 1, generator=gen)
    x = x.double() * torch.tensor([2.0 ** k for k in scales], dtype=torch.float64)[:, None]
    return x.to(DT[dt]).to(DEV)


@gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("D", WIDTHS)
def test_layer_norm_of_very_large_rows(D, dt):
    x = rows_of_scales(D, dt, [0, 90, 0, 62, 64, 1, 100, 110, 118, 0, 0, 75, 118], D)
    gen = torch.Generator().manual_seed(1)
    w, b = (torch.randn(D, generator=gen).to(DEV, DT[dt]) for _ in range(2))
    dy = torch.randn(x.shape, generator=gen).to(DEV, DT[dt])
    for c8 in (False, True)[:1 if dt == "f32" else 2]:
        y, g = base.run_norm(x.clone(), w.clone(), b.clone(), dy, 1e-5, checkpoint8=c8)
        base.norm_check(x, w, b, dy, 1e-5, y, g, checkpoint8=c8)


@gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("D", [5, 64, 300, 1500, 2051, 9000])
def test_layer_norm_at_the_ends_of_the_range(D, dt):
    """The type's largest values, alone and in rows of both signs; what stands in the other rows stays as it is; rows without spread give h = 0."""
    big = torch.finfo(DT[dt]).max
    x = rows_of_scales(D, dt, [0] * 6, 3)
    clean = ops.layer_norm(x)
    x[1] = big
    x[3, ::2], x[3, 1::2] = big, -big
    x[4, D // 2] = -big
    y = ops.layer_norm(x)
    assert torch.equal(y[[0, 2, 5]], clean[[0, 2, 5]])
    assert not y[1].any()
    for k in (3, 4):
        base.norm_check(x[k:k + 1], None, None, None, 1e-5, y[k:k + 1], None)
    x[4, 0] = float("inf")
    x[3, D - 1] = float("nan")
    y = ops.layer_norm(x)
    assert bool(y[3].isnan().all()) and bool(y[4].isnan().all()) and torch.equal(y[[0, 2, 5]], clean[[0, 2, 5]])


@gpu
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("D", [5, 64, 300, 1500, 2051, 9000])
def test_layer_norm_of_very_small_rows_without_eps(D, dt):
    """eps = 0 (and far below the rows' variance): the squares of such rows leave the range at its lower end."""
    x = rows_of_scales(D, dt, [0, -60, -80, -100, 0, -110, -45], 5)
    dy = torch.randn(x.shape, generator=torch.Generator().manual_seed(2)).to(DEV, DT[dt])
    for eps in (0.0, 2.0 ** -130):
        y, g = base.run_norm(x.clone(), None, None, 2.0 ** -20 * dy, eps)
        base.norm_check(x, None, None, 2.0 ** -20 * dy, eps, y, g)
    # eps far above such rows' variance: h is next to nothing
    y = ops.layer_norm(x[[1, 3, 5]], eps=1e-5)
    base.norm_check(x[[1, 3, 5]], None, None, None, 1e-5, y, None)


# ------------------------------------------------------------------------------------------------ 8-bit checkpoints read back in other types
@gpu
@pytest.mark.parametrize("dt", list(DT))
def test_checkpoints_are_exact_in_their_own_type_and_the_wide_ones(dt):
    lo, hi = (-24, 14) if dt == "f16" else (-130, 126)
    x = rows_of_scales(70, dt, range(lo, hi, 3), 7)
    x = torch.where(x.isfinite(), x, torch.ones_like(x))
    c = ops.checkpoint8(x)
    want = base.stored8(x.double())
    for t in {DT[dt], torch.float32, torch.bfloat16}:
        assert torch.equal(c.restore(t).double(), want)
    assert torch.equal(c.restore(torch.float16), want.half())                # elsewhere: the value in that type (an infinity beyond its range)
