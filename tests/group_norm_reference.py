"""Group norm with an activation in float64, channels last, with the bound of a
float32 evaluation's errors (the running error analysis of seq_reference.py).

A sum whose longest chain of additions is d is off by at most d units of its
terms' magnitudes.  Rows (one position): a lane adds up to 32 values, 6 steps join
64 lanes: 40.  Maps of the tests' sizes: 8 values a thread, up to 256 threads of
a column one after the other, up to 64 partial results a lane and 6 steps: 340;
each join of two means and sums of squares rounds six times where an addition
does once, and pivots are taken off and added again: 8 units each.  The channels'
gradients: 512 rows or partial rows of 340 at the most, and the same again.
"""

import torch

from tests.seq_reference import E, add1, check, dbl, one_minus, sigmoid  # noqa: F401  (check: the tests')


def _sum(x, dims, depth):
    n = 1
    for d in dims:
        n *= x.v.shape[d]
    return E(x.v.sum(dims, keepdim=True), x.e.sum(dims, keepdim=True) + min(n, depth) * x.v.abs().sum(dims, keepdim=True))


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, silu=False, z=None, dy=None):
    """{name: E}: y and, with dy, the gradients."""
    shape, C = x.shape, x.shape[-1]
    rows = (shape[0], -1, groups, C // groups)
    P = x.numel() // max(1, shape[0] * C)
    depth = 40 if P == 1 and C // groups <= 2048 else 8 * 340
    X = dbl(x.reshape(rows))
    m = P * (C // groups)
    w = dbl((weight if weight is not None else torch.ones(C)).reshape(rows[2:]))
    b = dbl((bias if bias is not None else torch.zeros(C)).reshape(rows[2:]))
    mean = _sum(X, (1, 3), depth) * (1.0 / m)
    c = X + -mean
    var = _sum(c * c, (1, 3), depth) * (1.0 / m)
    # (as floats: eps is one on both sides)
    ve = E(var.v + float(torch.tensor(eps)), var.e + (var.v + eps))
    r = ve.v.rsqrt()
    rstd = E(r, r * (0.5 * ve.e / ve.v + 3))
    xh = c * rstd
    n = xh * w + b
    sn = sigmoid(n)
    a = n * sn if silu else n
    y = a
    if z is not None:
        Z = dbl(z.reshape(rows))
        sz = sigmoid(Z)
        y = a * Z * sz
    back = lambda t: E(t.v.reshape(shape), t.e.reshape(shape))
    out = {"y": back(y)}
    if dy is None:
        return out
    d = dbl(dy.reshape(rows))
    if z is not None:
        out["dz"] = back(d * a * sz * add1(Z * one_minus(sz)))
        d = d * (Z * sz)
    if silu:
        d = d * (sn * add1(n * one_minus(sn)))
    h = d * w
    m1, m2 = _sum(h * xh, (1, 3), depth) * (1.0 / m), _sum(h, (1, 3), depth) * (1.0 / m)
    out["dx"] = back(rstd * (h + -m2 + -(xh * m1)))
    flat = lambda t: E(t.v.reshape(C), t.e.reshape(C))
    out["dweight"], out["dbias"] = flat(_sum(d * xh, (0, 1), 900)), flat(_sum(d, (0, 1), 900))
    return out
