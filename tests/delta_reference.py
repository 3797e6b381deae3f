"""The gated delta rule in float64, one token after the other, its adjoint, and
for every output the magnitude of the terms that the kernels sum for it.

Tolerances.  Products in float32 (whose operands are exact sums of bf16 parts)
round at 2^-24 a term; the errors of a sum of n terms are independent of each
other, so that with overwhelming probability the sum is off by less than LAMBDA
sqrt(n) 2^-24 of its terms' root of squares (Higham and Mary, "A new approach to
probabilistic rounding error analysis", 2019), LAMBDA = 4.  Here n <= 192: at
most 128 key values and 64 tokens.  An output is a chain of such products: 5
forward (S^T k, the triangle's inverse, its product, the outer product, S^T q)
and as many again behind them for the gradients.  Errors of the inverse T and of
what it is applied to grow by at most the 2-norm of |T|, KAPPA below, formed
from the inputs.  Along a sequence errors do not grow: for |k| <= 1 and 0 <=
beta <= 1 every step a (I - beta k k^T) is a contraction, and errors of the
chunks add up as the root of their number; a gate above 0 grows them by as much
as the magnitudes below.  So

    |got - ref| <= LAMBDA sqrt(192) 2^-24 STAGES KAPPA sqrt(chunks) mag + half a step of the type

with mag the terms' magnitudes: over all of an output in the 2-norm, and 8 times
that for any one element.
"""

import torch

LAMBDA = 4
STAGES = {"o": 5, "final": 5}  # the gradients: 10
CHUNK = 64
EPS = 1e-6


def unit(x, on):
    return x / (x.square().sum(-1, keepdim=True) + EPS).sqrt() if on else x


def rule(off, q, k, v, g, beta, scale=None, qk_l2norm=False, initial=None):
    """o and final states by torch operations (differentiable); float64."""
    T, HV, DV = v.shape
    r = HV // q.shape[1]
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    q, k = (unit(x, qk_l2norm).repeat_interleave(r, 1) for x in (q, k))
    rows, final = [torch.zeros(HV, DV, dtype=v.dtype)] * T, []
    for i in range(len(off) - 1):
        h = initial[i] if initial is not None else torch.zeros(HV, q.shape[-1], DV, dtype=v.dtype)
        for t in range(off[i], off[i + 1]):
            h = g[t].exp()[:, None, None] * h
            d = beta[t][:, None] * (v[t] - torch.einsum("hkv,hk->hv", h, k[t]))
            h = h + k[t][:, :, None] * d[:, None, :]
            rows[t] = scale * torch.einsum("hkv,hk->hv", h, q[t])
        final.append(h)
    o = torch.stack(rows) if T else torch.zeros(0, HV, DV, dtype=v.dtype)
    return o, torch.stack(final) if final else torch.zeros(0, HV, q.shape[-1], DV, dtype=v.dtype)


def kappa(off, k, g, beta, qk_l2norm):
    """The largest 2-norm of |T| over the chunks and heads."""
    worst, r = 1.0, g.shape[1] // k.shape[1]
    k = unit(k, qk_l2norm).repeat_interleave(r, 1)
    for i in range(len(off) - 1):
        for t in range(off[i], off[i + 1], CHUNK):
            s = slice(t, min(t + CHUNK, off[i + 1]))
            G = g[s].clamp(min=-1e4).cumsum(0).t()
            D = torch.tril(G[:, :, None] - G[:, None, :], -1)  # (gates above 0 grow)
            A = torch.einsum("ihk,jhk->hij", k[s], k[s]) * D.exp()
            A = torch.tril(A * beta[s].t()[:, :, None], -1)
            T = torch.linalg.inv(torch.eye(A.shape[-1], dtype=A.dtype) + A)
            worst = max(worst, float(torch.linalg.matrix_norm(T.abs(), 2).max()))
    return worst


def reference(off, q, k, v, g, beta, scale=None, qk_l2norm=False, initial=None, do=None, dfinal=None):
    """{name: (value, magnitude)} and the factor of the tolerance."""
    q, k, v, g, beta = (x.detach().double().cpu() for x in (q, k, v, g, beta))
    initial = initial.detach().double().cpu() if initial is not None else None
    T, HV, DV = v.shape
    HK, DK = q.shape[1:]
    r, S = HV // HK, len(off) - 1
    scale = DK ** -0.5 if scale is None else scale
    qn, kn = (unit(x, qk_l2norm).repeat_interleave(r, 1) for x in (q, k))
    z = lambda *s: torch.zeros(*s, dtype=torch.float64)
    o, mo, final, mf = z(T, HV, DV), z(T, HV, DV), z(S, HV, DK, DV), z(S, HV, DK, DV)
    names = ("q", "k", "v", "g", "beta")
    out = {n: z(T, HV, *((DK,) if n in "qk" else (DV,) if n == "v" else ())) for n in names}
    mag = {n: torch.zeros_like(x) for n, x in out.items()}
    dinit, mi = z(S, HV, DK, DV), z(S, HV, DK, DV)
    for i in range(S):
        h = initial[i] if initial is not None else z(HV, DK, DV)
        hs, ps, ds, top = [h], [], [], h.abs()
        for t in range(off[i], off[i + 1]):
            p = g[t].exp()[:, None, None] * h
            d = beta[t][:, None] * (v[t] - torch.einsum("hkv,hk->hv", p, kn[t]))
            h = p + kn[t][:, :, None] * d[:, None, :]
            top = torch.maximum(g[t].exp()[:, None, None] * top, h.abs()) + (kn[t][:, :, None] * v[t][:, None, :]).abs() * 0.1
            o[t] = scale * torch.einsum("hkv,hk->hv", h, qn[t])
            mo[t] = abs(scale) * torch.einsum("hkv,hk->hv", top, qn[t].abs())
            hs.append(h), ps.append(p), ds.append(d)
        final[i], mf[i] = h, top
        if do is None:
            continue
        D = dfinal[i].double().cpu() if dfinal is not None else z(HV, DK, DV)
        mD, dgs = D.abs(), 0
        for t in reversed(range(off[i], off[i + 1])):
            n = t - off[i]
            dot = scale * do[t].double().cpu()
            D = D + qn[t][:, :, None] * dot[:, None, :]
            mD = torch.maximum(mD, D.abs())
            dd = torch.einsum("hkv,hk->hv", D, kn[t])
            mdd = torch.einsum("hkv,hk->hv", mD, kn[t].abs())
            b = beta[t][:, None]
            out["q"][t] = torch.einsum("hkv,hv->hk", hs[n + 1], dot)
            mag["q"][t] = torch.einsum("hkv,hv->hk", hs[n + 1].abs() + ps[n].abs(), dot.abs())
            out["k"][t] = torch.einsum("hkv,hv->hk", D, ds[n]) - b * torch.einsum("hkv,hv->hk", ps[n], dd)
            mag["k"][t] = torch.einsum("hkv,hv->hk", mD, ds[n].abs()) + b * torch.einsum("hkv,hv->hk", ps[n].abs(), mdd)
            out["v"][t], mag["v"][t] = b * dd, b * mdd
            err = v[t] - torch.einsum("hkv,hk->hv", ps[n], kn[t])
            out["beta"][t] = (dd * err).sum(-1)
            mag["beta"][t] = (mdd * (v[t].abs() + torch.einsum("hkv,hk->hv", ps[n].abs(), kn[t].abs()))).sum(-1)
            D = D - kn[t][:, :, None] * (b * dd)[:, None, :]
            out["g"][t] = (D * ps[n]).sum((-1, -2))
            # the kernels sum the tokens' parts over a chunk, and take what cancels with the sum over all of it
            dgs = dgs + (qn[t] * out["q"][t]).abs().sum(-1) + 3 * (kn[t] * out["k"][t]).abs().sum(-1)
            mag["g"][t] = (mD * ps[n].abs()).sum((-1, -2)) + dgs
            D = g[t].exp()[:, None, None] * D
            mD = g[t].exp()[:, None, None] * mD
            if n % CHUNK == 0:
                mag["g"][t:t + CHUNK] = mag["g"][t:min(t + CHUNK, off[i + 1])].max(0).values
                dgs = 0
        dinit[i], mi[i] = D, mD
    res = {"o": (o, mo), "final": (final, mf)}
    if do is not None:
        for n, x in (("q", q), ("k", k)):
            d, m = (y[n].view(T, HK, r, DK).sum(2) for y in (out, mag))
            if qk_l2norm:
                rn = (x.square().sum(-1, keepdim=True) + EPS).rsqrt()
                u = x * rn
                d, m = rn * (d - u * (u * d).sum(-1, keepdim=True)), rn * (m + u.abs() * (u.abs() * m).sum(-1, keepdim=True))
            out[n], mag[n] = d, m
        res.update({"d" + n: (out[n], mag[n]) for n in names})
        res["dinitial"] = (dinit, mi)
    longest = max([b - a for a, b in zip(off, off[1:])] + [1])
    factor = LAMBDA * 192 ** 0.5 * 2.0 ** -24 * kappa(off, k, g, beta, qk_l2norm) * (-(-longest // CHUNK)) ** 0.5
    return res, factor


def check(name, got, ref, factor):
    value, mag = ref
    assert tuple(got.shape) == tuple(value.shape), (name, got.shape, value.shape)
    if not value.numel():
        return
    g = got.detach().double().cpu()
    tol = factor * STAGES.get(name, 10)
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    err, rms = (g - value).abs(), mag.square().mean().sqrt()
    lim = tol * mag.norm() + half * value.norm()
    assert float(err.norm()) <= float(lim) + 1e-37, f"{name}: off {float(err.norm()):.3g} > {float(lim):.3g} in the 2-norm"
    each = 8 * tol * (mag + rms) + half * value.abs() + 1e-37
    if not bool((err <= each).all()):
        j = int((torch.nan_to_num(err - each, nan=float("inf"))).argmax())
        raise AssertionError(f"{name}: element {j}: got {float(g.flatten()[j])!r}, ref {float(value.flatten()[j])!r}, "
                             f"off {float(err.flatten()[j]):.3g} > {float(each.flatten()[j]):.3g}")
