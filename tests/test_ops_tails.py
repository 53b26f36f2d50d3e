"""The public operators where values are far from one: rows whose squares leave the range of fp32."""
import pytest
import torch

import test_ops as base
from lsdm_amd import ops

gpu = pytest.mark.gpu
DEV, DT = base.DEV, base.DT


@pytest.fixture(autouse=True)
def _grad_mode():
    with torch.enable_grad():
        yield


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
