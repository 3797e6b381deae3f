"""Gradients of the gated delta rule's gates where the gates let little through.

Every term of dg_t has exp(g_t) as a factor, so it has as many digits where the
factor is 1e-9 as where it is 1.  The tolerance is delta_reference.py's with the
magnitude of these terms alone, taken for every head and every token by itself:
sum |D_t| |exp(g_t) S_{t-1}| over the state, D_t being the gradient that reaches
it.  Heads are small, so that this sum is not far above the value's own size.
"""

import pytest
import torch

from tests import delta_reference as ref
from tests.test_gpu_delta import TYPES, _call, _inputs, _off

pytestmark = pytest.mark.gpu


def _gates(off, q, k, v, g, beta, initial, do, dfinal):
    """dg and the magnitude of its terms, in float64 (keys and queries normalised, default scale)."""
    q, k, v, g, beta, initial, do, dfinal = (x.double() for x in (q, k, v, g, beta, initial, do, dfinal))
    r = v.shape[1] // q.shape[1]
    q, k = (ref.unit(x, True).repeat_interleave(r, 1) for x in (q, k))
    scale = q.shape[-1] ** -0.5
    dg, mag = torch.zeros_like(g), torch.zeros_like(g)
    for i in range(len(off) - 1):
        h, top, before = initial[i], initial[i].abs(), []
        for t in range(off[i], off[i + 1]):
            a = g[t].clamp(min=-1e4).exp()[:, None, None]
            p = a * h
            before.append((p, a * top))
            d = beta[t][:, None] * (v[t] - (p * k[t][:, :, None]).sum(1))
            h = p + k[t][:, :, None] * d[:, None, :]
            top = torch.maximum(a * top, h.abs())
        D, mD = dfinal[i], dfinal[i].abs()
        for t in reversed(range(off[i], off[i + 1])):
            D = D + scale * q[t][:, :, None] * do[t][:, None, :]
            mD = torch.maximum(mD, D.abs())
            D = D - beta[t][:, None, None] * k[t][:, :, None] * (D * k[t][:, :, None]).sum(1)[:, None, :]
            p, mp = before.pop()
            dg[t], mag[t] = (D * p).sum((1, 2)), (mD * mp).sum((1, 2))
            a = g[t].clamp(min=-1e4).exp()[:, None, None]
            D, mD = a * D, a * mD
    return dg, mag


@pytest.mark.parametrize("gate", [-0.5, -2.0, -8.0, -14.0, -20.0, -40.0])
@pytest.mark.parametrize("HK,HV,DK,DV", [(2, 2, 8, 8), (1, 3, 8, 4), (2, 2, 40, 8), (1, 2, 128, 16)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_gates_that_let_little_through(cuda, dtype, HK, HV, DK, DV, gate):
    """Every gate of the last head near one value, the others' between 0 and -1."""
    lens = [100, 1, 64, 30]
    a, init, do, df = _inputs(lens, HK, HV, DK, DV, TYPES[dtype], 40)
    a["g"][:, -1] = gate * (1 + 0.1 * torch.rand(sum(lens), generator=torch.Generator().manual_seed(41)))
    got = _call(cuda, lens, a, init, do, df)["dg"].double().cpu()
    want, mag = _gates(_off(lens), **a, initial=init, do=do, dfinal=df)
    _, factor = ref.reference(_off(lens), **a, qk_l2norm=True, initial=init)
    tol = 10 * factor
    for h in range(HV):
        err = (got[:, h] - want[:, h]).abs()
        assert float(err.norm()) <= tol * float(mag[:, h].norm()), f"head {h}: {float(err.norm() / want[:, h].norm()):.3g} of dg"
        worst = int((err / mag[:, h]).argmax())
        assert bool((err <= 8 * tol * mag[:, h]).all()), f"head {h}, token {worst}: {got[worst, h]!r}, ref {want[worst, h]!r}"


@pytest.mark.parametrize("HK,DK", [(1, 16), (2, 100)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_gates_below_the_least(cuda, dtype, HK, DK):
    """Gates below -10000 are taken as that: their gradient is zero, exactly."""
    lens = [90, 40]
    a, init, do, df = _inputs(lens, HK, 2, DK, 16, TYPES[dtype], 42)
    a["g"][:, 0] = -2e4
    a["g"][[5, 64, 70, 95], 1] = torch.tensor([-1.5e4, -1e30, float("-inf"), -2e4])
    got = _call(cuda, lens, a, init, do, df)["dg"].cpu()
    assert bool((got[:, 0] == 0).all()) and bool((got[[5, 64, 70, 95], 1] == 0).all())
    want, mag = _gates(_off(lens), **a, initial=init, do=do, dfinal=df)
    _, factor = ref.reference(_off(lens), **{**a, "g": a["g"].clamp(min=-1e4)}, qk_l2norm=True, initial=init)
    assert bool(((got.double() - want).abs() <= 80 * factor * mag)[:, 1].all())


@pytest.mark.parametrize("tokens", [1, 64, 70])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_decays_have_the_digits_of_their_type(cuda, dtype, tokens):
    """Nothing is written (beta 0): states and their gradients are multiplied by the decay alone, of a chunk at a time.
    An exponential is off by a unit of 2^-23, its argument's fraction by 2^-26, a product by 2^-24: less than 2^-22 a chunk."""
    total = torch.tensor([-0.01, -1.0, -5.0, -16.0, -33.0, -60.0, -80.0])
    S = len(total)
    lens = [tokens] * S
    a, init, do, df = _inputs(lens, 1, 2, 16, 24, TYPES[dtype], 43)
    a["g"][:] = (total / tokens).repeat_interleave(tokens)[:, None]
    a["beta"].zero_()
    got = _call(cuda, lens, a, init, 0 * do, df)
    decay = a["g"].double().view(S, tokens, 2).sum(1).exp()[:, :, None, None]
    for name, x in (("final", init), ("dinitial", df)):
        want = decay * x.double()
        err = ((got[name].detach().double().cpu() - want) / want).abs()
        assert float(err.max()) <= 2.0 ** -22 * -(-tokens // 64), f"{name}: off by {float(err.max()):.3g} of the value"
