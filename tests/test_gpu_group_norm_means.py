"""Group norm of values far from zero beside their spread, through every kernel.

A mean of n float32 values is off by at most the longest chain of additions
(DEPTH) units of 2^-24 of it; what it is off by is itself found from the
differences, with DEPTH units of that.  A group of one value, whose every
difference is the mean's error, comes out as its bias up to the square of this."""

import pytest
import torch

import mlx_vision_mamba_amd as mvm
from tests import group_norm_reference as ref

pytestmark = pytest.mark.gpu

DEPTH = 128  # a lane's or thread's 64 values at the most, 6 steps over lanes, the waves, the quotient
SHAPES = {  # (x's shape, groups)
    "rows": ((7, 1020), 1), "rows of heads": ((9, 12 * 100), 12), "rows value by value": ((5, 3 * 333), 3),
    "wide row": ((2, 2052), 1), "tile": ((3, 1020, 64), 8), "full tile": ((2, 64, 256), 1), "tile of few": ((2, 5, 40), 2),
    "map": ((2, 9000, 32), 4), "map value by value": ((1, 2900, 3), 1)}


@pytest.mark.parametrize("value", [3.0, 10.1, 100.1, 1000.1, -77.7])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_groups_of_one_value(cuda, shape, value):
    (shape, groups), eps = SHAPES[shape], 1e-5
    x = torch.full(shape, value)
    bias = torch.randn(shape[-1], generator=torch.Generator().manual_seed(1))
    weight = 1 + 0.1 * torch.randn(shape[-1], generator=torch.Generator().manual_seed(2))
    y = mvm.group_norm(x.to(cuda), groups, weight.to(cuda), bias.to(cuda), eps).cpu()
    each = (DEPTH * 2.0 ** -24) ** 2 * abs(value) / eps ** 0.5 * weight.abs() + 2.0 ** -24 * bias.abs()
    err = (y - bias).abs()
    assert bool((err <= each).all()), f"off by {float(err.max()):.3g}"


@pytest.mark.parametrize("mean", [4096.1, -1000.3])
@pytest.mark.parametrize("shape", ["rows", "rows of heads", "rows value by value", "tile", "full tile", "tile of few"])
def test_values_around_a_far_mean(cuda, shape, mean):
    """Groups that fit in registers: the output has the digits of the differences, not of the mean."""
    shape, groups = SHAPES[shape]
    x = mean + torch.randn(shape, generator=torch.Generator().manual_seed(3))
    y = mvm.group_norm(x.to(cuda), groups).cpu().double()
    want = ref.group_norm(x, groups)["y"].v
    err = float((y - want).norm() / want.norm())
    assert err <= 4 * DEPTH * 2.0 ** -24, f"off by {err:.3g}"
