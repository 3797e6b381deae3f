"""The packed scan and conv in float64, one token after the other, each value
with a bound of the error that a float32 evaluation can have (running error
analysis, to first order).

An ``E`` holds a value and its error bound in units of U = 2^-24, the largest
relative rounding error of float32.  Every operation adds what it propagates
from its operands and one unit of its result; a sum of n terms adds n units of
the terms' magnitudes, whatever its order.  The kernels' own functions:

* exp(x) as exp2 of x log2(e): the rounded product is off by 2 units of |x|
  (log2(e) is rounded too), the exponential by one ulp (2 units);
* softplus: 30 ulp (60 units) of the result over [-30, 20];
* sigmoid(x) = 1 / (1 + exp(-x)): the exponential's error, one unit of the sum
  and one ulp of the reciprocal.
"""

import torch

U = 2.0 ** -24


class E:
    def __init__(self, v, e=None):
        self.v = v
        self.e = torch.zeros_like(v) if e is None else e

    def __add__(self, o):
        v = self.v + o.v
        return E(v, self.e + o.e + v.abs())

    def __mul__(self, o):
        if not isinstance(o, E):
            o = E(torch.as_tensor(o, dtype=torch.float64))
        v = self.v * o.v
        return E(v, self.v.abs() * o.e + o.v.abs() * self.e + v.abs())

    def __neg__(self):
        return E(-self.v, self.e)

    def __getitem__(self, i):
        return E(self.v[i], self.e[i])

    def sum(self, dim):
        n = self.v.shape[dim]
        return E(self.v.sum(dim), self.e.sum(dim) + n * self.v.abs().sum(dim))


def exp(x):
    v = x.v.exp()
    return E(v, v * (x.e + 2 * x.v.abs() + 2))


def sigmoid(x):
    v = torch.sigmoid(x.v)
    return E(v, v * (1 - v) * (x.e + 2 * x.v.abs() + 2) + 4 * v)


def softplus(x):
    v = torch.nn.functional.softplus(x.v, threshold=300)
    return E(v, torch.sigmoid(x.v) * x.e + 60 * v)


def one_minus(x):
    return E(1 - x.v, x.e + (1 - x.v).abs())


def add1(x):
    return E(1 + x.v, x.e + (1 + x.v).abs())


def stack(xs):
    return E(torch.stack([x.v for x in xs]), torch.stack([x.e for x in xs]))


def dbl(t):
    return E(t.detach().double().cpu())


def scan(off, u, delta, A, B, C, D, z=None, delta_bias=None, delta_softplus=False, a_is_log=False, initial=None,
         dy=None, dfinal=None):
    """{name: E} of y, final and, with dy (and dfinal), the gradients of every
    argument.  Rows of no sequence are zero."""
    T, Dn = u.shape
    N = A.shape[1]
    u, delta, Ain, B, C, D = (dbl(t) for t in (u, delta, A, B, C, D))
    Am = -exp(Ain) if a_is_log else Ain
    raw = delta + dbl(delta_bias) if delta_bias is not None else delta
    dl = softplus(raw) if delta_softplus else raw
    if z is not None:
        z = dbl(z)
        sg = sigmoid(z)
        silu = z * sg
    S = len(off) - 1
    h0 = dbl(initial) if initial is not None else E(torch.zeros(S, Dn, N, dtype=torch.float64))
    zero = E(torch.zeros(Dn, dtype=torch.float64))
    y = [zero] * T
    r = [zero] * T
    final, hs, bs, as_ = [], {}, {}, {}
    for i in range(S):
        h = h0[i]
        for t in range(off[i], off[i + 1]):
            a = exp(dl[t][:, None] * Am)
            bs[t], as_[t] = h, a
            h = a * h + (dl[t] * u[t])[:, None] * B[t][None, :]
            hs[t] = h
            r[t] = (h * C[t][None, :]).sum(-1) + D * u[t]
            y[t] = r[t] * silu[t] if z is not None else r[t]
        final.append(h)
    out = {"y": stack(y) if T else E(torch.zeros(0, Dn, dtype=torch.float64)),
           "final": stack(final) if S else E(torch.zeros(0, Dn, N, dtype=torch.float64))}
    if dy is None:
        return out
    dy = dbl(dy)
    rows = {k: [E(torch.zeros(n, dtype=torch.float64))] * T for k, n in
            (("du", Dn), ("ddelta", Dn), ("dz", Dn), ("dB", N), ("dC", N))}
    dA_t, dD_t, dh0 = [], [], []
    for i in range(S):
        c = dbl(dfinal)[i] if dfinal is not None else E(torch.zeros(Dn, N, dtype=torch.float64))
        for t in reversed(range(off[i], off[i + 1])):
            dr = dy[t] * silu[t] if z is not None else dy[t]
            dh = C[t][None, :] * dr[:, None] + c
            du_ = dl[t] * u[t]
            rows["dB"][t] = (dh * du_[:, None]).sum(0)
            rows["dC"][t] = (hs[t] * dr[:, None]).sum(0)
            q = (dh * B[t][None, :]).sum(-1)
            x = dh * (as_[t] * bs[t])
            dd = (x * Am).sum(-1) * 1.0 + q * u[t]
            if delta_softplus:
                dd = dd * sigmoid(raw[t])
            rows["du"][t] = q * dl[t] + D * dr
            rows["ddelta"][t] = dd
            if z is not None:
                rows["dz"][t] = dy[t] * r[t] * sg[t] * add1(z[t] * one_minus(sg[t]))
            dA_t.append(x * dl[t][:, None])
            dD_t.append(dr * u[t])
            c = as_[t] * dh
        dh0.append(c)
    for k, v in rows.items():
        out[k] = stack(v) if T else E(torch.zeros(0, v and v[0].v.shape[0] or Dn, dtype=torch.float64))
    none = E(torch.zeros(1, Dn, N, dtype=torch.float64))
    dA = (stack(dA_t) if dA_t else none).sum(0)
    out["dA"] = dA * Am if a_is_log else dA
    out["dD"] = (stack(dD_t) if dD_t else E(torch.zeros(1, Dn, dtype=torch.float64))).sum(0)
    out["ddelta_bias"] = out["ddelta"].sum(0)
    out["dinitial"] = stack(dh0) if S else E(torch.zeros(0, Dn, N, dtype=torch.float64))
    if z is None:
        del out["dz"]
    return out


def conv(off, x, weight, bias=None, initial=None, dy=None, dfinal=None):
    """{name: E} of y, final and the gradients."""
    T, Dn = x.shape
    W = weight.shape[1]
    x, w = dbl(x), dbl(weight)
    b = dbl(bias) if bias is not None else E(torch.zeros(Dn, dtype=torch.float64))
    S = len(off) - 1
    c0 = dbl(initial) if initial is not None else E(torch.zeros(S, W - 1, Dn, dtype=torch.float64))
    zero = E(torch.zeros(Dn, dtype=torch.float64))
    y, dx = [zero] * T, [zero] * T
    final, dc0, dw_t, db_t = [], [], [], []
    for i in range(S):
        n = off[i + 1] - off[i]
        xt = [c0[i][r] for r in range(W - 1)] + [x[off[i] + t] for t in range(n)]
        final += xt[n:n + W - 1]
        g = [zero] * (n + W - 1)
        if dfinal is not None:
            for r in range(W - 1):
                g[n + r] = g[n + r] + dbl(dfinal)[i, r]
        for t in range(n):
            pre = b
            for j in range(W):
                pre = pre + w[:, j] * xt[t + j]
            s = sigmoid(pre)
            y[off[i] + t] = pre * s
            if dy is not None:
                dpre = dbl(dy)[off[i] + t] * s * add1(pre * one_minus(s))
                for j in range(W):
                    g[t + j] = g[t + j] + w[:, j] * dpre
                dw_t.append(stack([dpre * xt[t + j] for j in range(W)]))
                db_t.append(dpre)
        dc0 += g[:W - 1]
        for t in range(n):
            dx[off[i] + t] = g[W - 1 + t]

    def rows(v, *shape):
        r = stack(v) if v else E(torch.zeros(0, Dn, dtype=torch.float64))
        return E(r.v.reshape(*shape), r.e.reshape(*shape))

    out = {"y": rows(y, T, Dn), "final": rows(final, S, W - 1, Dn)}
    if dy is not None:
        out["dx"], out["dinitial"] = rows(dx, T, Dn), rows(dc0, S, W - 1, Dn)
        dw = (stack(dw_t) if dw_t else E(torch.zeros(1, W, Dn, dtype=torch.float64))).sum(0)
        out["dweight"] = E(dw.v.t(), dw.e.t())
        out["dbias"] = (stack(db_t) if db_t else E(torch.zeros(1, Dn, dtype=torch.float64))).sum(0)
    return out


def check(name, got, ref):
    """|got - ref| within the float32 bound, and half a step of got's own type."""
    assert tuple(got.shape) == tuple(ref.v.shape), (name, got.shape, ref.v.shape)
    g = got.detach().double().cpu()
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    lim = ref.e * U
    # (float32's and bf16's smallest normal, where exponentials flush to zero)
    lim = lim + half * (ref.v.abs() + lim) + 2.0 ** -126
    err = (g - ref.v).abs()
    if err.numel() and not bool((err <= lim).all()):
        k = int((torch.nan_to_num(err - lim, nan=float("inf"))).argmax())
        raise AssertionError(f"{name}: element {k}: got {float(g.flatten()[k])!r}, ref {float(ref.v.flatten()[k])!r}, "
                             f"off {float(err.flatten()[k]):.3g} > {float(lim.flatten()[k]):.3g}")
