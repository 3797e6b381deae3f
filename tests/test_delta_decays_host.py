"""The float64 reference of the gates' gradients (test_gpu_delta_decays.py)
against torch's autograd of the recurrence, and against differences."""

import pytest
import torch

from tests import delta_reference as ref
from tests.test_gpu_delta import _inputs, _off
from tests.test_gpu_delta_decays import _gates


def _case(gate):
    lens = [9, 0, 1, 6]
    a, init, do, df = _inputs(lens, 1, 2, 5, 4, torch.float32, 44)
    a["g"][:, 1] = gate * (1 + 0.1 * torch.rand(sum(lens), generator=torch.Generator().manual_seed(45)))
    return _off(lens), {n: x.double() for n, x in a.items()}, init.double(), do.double(), df.double()


def _loss(off, a, init, do, df):
    o, final = ref.rule(off, *a.values(), qk_l2norm=True, initial=init)
    return (o * do).sum() + (final * df).sum()


@pytest.mark.parametrize("gate", [-0.5, -8.0, -20.0])
def test_reference_agrees_with_autograd(gate):
    off, a, init, do, df = _case(gate)
    a["g"].requires_grad_(True)
    (want,) = torch.autograd.grad(_loss(off, a, init, do, df), a["g"])
    got, mag = _gates(off, **{n: x.detach() for n, x in a.items()}, initial=init, do=do, dfinal=df)
    assert bool(((got - want).abs() <= 1e-12 * mag).all()) and bool((got.abs() <= mag * (1 + 1e-12)).all())


def test_reference_agrees_with_differences():
    off, a, init, do, df = _case(-2.0)
    got, _ = _gates(off, **a, initial=init, do=do, dfinal=df)
    h = 1e-5
    for t, head in ((0, 0), (3, 1), (8, 0), (9, 1), (12, 1), (15, 0)):
        ends = []
        for s in (h, -h):
            g = a["g"].clone()
            g[t, head] += s
            ends.append(_loss(off, {**a, "g": g}, init, do, df))
        assert abs(float(ends[0] - ends[1]) / (2 * h) - float(got[t, head])) <= 1e-7 * max(1.0, abs(float(got[t, head])))
