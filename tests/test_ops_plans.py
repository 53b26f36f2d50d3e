"""Every variant of the dense layer's kernels on sizes that are shown to choose it, the kernel of few rows over long contractions, and gradients against
differences of the definition in 64 bits."""
import pytest
import torch

import test_ops as base
from lsdm_amd import _lib, ops

gpu = pytest.mark.gpu
DEV, DT = base.DEV, base.DT
CODE = {"f32": 0, "bf16": 1, "f16": 2}


@pytest.fixture(autouse=True)
def _grad_mode():
    with torch.enable_grad():
        yield


# M, K, N: odd sizes, so that every tile is cut and every row padded; the contractions that count have more than two steps
SIZES = {"f32": [(7001, 389, 439), (389, 433, 7349), (421, 7407, 405), (4261, 67, 3363), (3421, 4343, 65), (3137, 65, 4741)],
         "bf16": [(387, 301, 7217), (7839, 3109, 19), (4127, 1435, 303), (4099, 325, 1415), (385, 7055, 323), (309, 415, 7059), (3097, 65, 4895), (69, 5073, 3123),
                  (303, 1225, 4911), (6191, 4543, 67), (4935, 6201, 67), (5729, 69, 5525), (1347, 321, 7687), (325, 1541, 6727), (4299, 2397, 331), (5521, 685, 5445),
                  (653, 5145, 6105)]}
SIZES["f16"] = SIZES["bf16"]
TILES = {"f32": [(128, 128), (64, 64)], "bf16": [(256, 256), (128, 128), (64, 128), (64, 64)]}
TILES["f16"] = TILES["bf16"]


def plans(dt, M, K, N):
    """(operand layout, tile, whether the contraction is split) of y, dx and dw, of those with at least three steps of 128 bytes."""
    lib, found = _lib.load(), []
    for what, a, b, c in (("y", M, N, K), ("dx", M, K, N), ("dw", N, K, M)):
        v = lib.lsdm_linear_plan(CODE[dt], a, b, c)
        assert v > 0
        if c >= (150 if dt == "f32" else 300):
            found.append((what, (v >> 32, v >> 16 & 0xffff), (v & 0xffff) > 1))
    return found


@pytest.mark.parametrize("dt", list(DT))
def test_the_sizes_below_take_every_tile_in_every_layout_whole_and_split(dt):
    taken = {p for s in SIZES[dt] for p in plans(dt, *s)}
    assert taken == {(what, tile, split) for what in ("y", "dx", "dw") for tile in TILES[dt] for split in (False, True)}


def test_plan_refuses_what_the_layer_refuses():
    lib = _lib.load()
    assert lib.lsdm_linear_plan(3, 8, 8, 8) == -1 and lib.lsdm_linear_plan(1, 0, 8, 8) == -1 and lib.lsdm_linear_plan(1, 8, (1 << 25) + 1, 8) == -1
    assert lib.lsdm_linear_plan(0, 1 << 30, 1 << 20, 8) == 0             # more tiles than a launch holds


@gpu
@pytest.mark.parametrize("dt,M,K,N", [(dt, *s) for dt in DT for s in SIZES[dt]])
def test_every_tile_layout_and_split(dt, M, K, N):
    acts = list(ops.ACTIVATIONS)
    x, w, b, r, dy = base.linear_case(M, K, N, dt, M + N, bias_f32=M % 2 == 0)
    act = acts[(M + K) % len(acts)]
    y, g = base.run_linear(x, w, b, r, dy, act)
    base.linear_check(x, w, b, r, dy, act, y, g)


# up to 64 rows: 1 .. 16 waves (8 from 33 rows on) that split the contraction, one and more rounds of loads each, ragged ends
@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("M,K,N", [(1, 1100, 70), (1, 2816, 70), (16, 4100, 33), (7, 9001, 40), (17, 1030, 24), (20, 2300, 48), (32, 5000, 17), (33, 530, 40), (33, 1500, 40),
                                   (48, 4097, 33), (64, 2950, 20), (64, 8192, 130)])
def test_few_rows_over_long_contractions(dt, M, K, N):
    acts = list(ops.ACTIVATIONS)
    x, w, b, r, dy = base.linear_case(M, K, N, dt, K, bias=M % 3 != 0, residual=M % 2 == 0)
    act = acts[(M + K + N) % len(acts)]
    y, g = base.run_linear(x, w, b, r, dy, act)
    base.linear_check(x, w, b, r, dy, act, y, g)
    wide = torch.zeros(M, K + 9, device=DEV, dtype=x.dtype)
    wide[:, 5:5 + K] = x.detach()
    with torch.no_grad():
        assert torch.equal(ops.linear(wide[:, 5:5 + K], w, b, act, r), y)      # rows at any address


# A gradient g against the definition's change along sign(g), which is sum |g|: any uniform error of g shows in full.  Central differences of the definition in
# 64 bits at h = 2^-14: z moves by at most 15 h, so the truncation is below (15 h)^2 = 1e-6 of the slope; g itself carries its type's roundings (three
# at most: dz, the sum's operands are exact, the result), half_step each, and fp32's sums.
def against_differences(f, leaves, g, dt):
    for k, v in enumerate(g):
        s = torch.sign(v.double())
        args = [t.detach().double() for t in leaves]
        h = 2.0 ** -14
        up, down = ([a + sg * h * s if i == k else a for i, a in enumerate(args)] for sg in (1, -1))
        slope, want = float((f(*up) - f(*down)) / (2 * h)), float(v.double().abs().sum())
        assert abs(slope - want) <= (1e-5 + 3 * base.half_step(DT[dt])) * want, (k, slope, want)


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("act", list(ops.ACTIVATIONS))
def test_linear_gradients_against_differences_of_the_definition(act, dt):
    gen = torch.Generator().manual_seed(3)
    leaves = [torch.randn(*s, generator=gen).to(DEV, DT[dt]).requires_grad_(True) for s in ((9, 12), (7, 12), (7,), (9, 7))]
    c = torch.randn(9, 7, generator=gen).to(DEV, DT[dt])
    z = leaves[0].detach().double() @ leaves[1].detach().double().T + leaves[2].detach().double()
    if act == "relu":
        assert float(z.abs().min()) > 2e-3                                # no kink within the step
    g = torch.autograd.grad(ops.linear(leaves[0], leaves[1], leaves[2], act, leaves[3]), leaves, c)
    against_differences(lambda x, w, b, r: ((base.act64(act, x @ w.T + b)[0] + r) * c.double()).sum(), leaves, g, dt)


@gpu
@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("D", [7, 40, 200])
def test_layer_norm_gradients_against_differences_of_the_definition(D, dt):
    gen = torch.Generator().manual_seed(D)
    leaves = [torch.randn(*s, generator=gen).to(DEV, DT[dt]).requires_grad_(True) for s in ((11, D), (D,), (D,))]
    c = torch.randn(11, D, generator=gen).to(DEV, DT[dt])

    def f(x, w, b):
        m = x.mean(1, keepdim=True)
        return (((x - m) / torch.sqrt(((x - m) ** 2).mean(1, keepdim=True) + 1e-3) * w + b) * c.double()).sum()
    g = torch.autograd.grad(ops.layer_norm(*leaves, 1e-3), leaves, c)
    against_differences(f, leaves, g, dt)
