"""Blocks in bfloat16 on packed and served sequences, against a float64 evaluation
that rounds to bf16 where the block does, forward and backward; and the example
in bfloat16.

The block's values and the oracle's are rounded at the same places.  What is left
between them are float32 sums in another order, off by some 2^-24 of their terms,
which move a value across a border between two bf16 numbers seldom (about one in
2^16 times the terms of the sum), and then by one step of 2^-7.  Were every element
of an output off by half a step, it would be off by 2^-8 in norm: that is the limit."""

import importlib.util
import os

import pytest
import torch
import torch.nn.functional as F

import mlx_vision_mamba_amd as mvm

pytestmark = pytest.mark.gpu

LIMIT = 2.0 ** -8


def _bf16(x):
    return x.bfloat16().to(x.dtype)


class _Stored(torch.autograd.Function):
    """A tensor that is held in bf16, its gradient too."""

    @staticmethod
    def forward(ctx, x):
        return _bf16(x)

    @staticmethod
    def backward(ctx, g):
        return _bf16(g)


class _Used(torch.autograd.Function):
    """One use of such a tensor: this use's share of its gradient is bf16."""

    @staticmethod
    def forward(ctx, x):
        return x.view_as(x)

    @staticmethod
    def backward(ctx, g):
        return _bf16(g)


stored, used = _Stored.apply, _Used.apply


def _linear(x, w):
    return stored(used(x) @ used(w).t())


def _block(p, x, n, off, conv0, scan0):
    """MambaBlock in float64 with its roundings: y, the conv's and the scan's states."""
    Din, W = p["conv1d.weight"].shape[0], p["conv1d.weight"].shape[-1]
    R = p["dt_proj.weight"].shape[1]
    xz = _linear(x, p["in_proj.weight"])
    cw, cb = used(p["conv1d.weight"]).reshape(Din, W), used(p["conv1d.bias"])
    xb, z = used(xz[:, :Din]), used(xz[:, Din:])
    xc, conv1 = [], []
    for i, (a, b) in enumerate(zip(off, off[1:])):
        xt = torch.cat([conv0[i], xb[a:b]])
        conv1.append(xt[b - a:])
        if b > a:
            xc.append(F.silu(sum(cw[:, j] * xt[j:j + b - a] for j in range(W)) + cb))
    xc = stored(torch.cat(xc))
    dbc = _linear(xc, p["x_proj.weight"])
    delta = _linear(used(dbc[:, :R]), p["dt_proj.weight"])
    u, dl, Bm, Cm = used(xc), used(delta), used(dbc[:, R:R + n]), used(dbc[:, R + n:])
    dl = F.softplus(dl + used(p["dt_proj.bias"]))
    A, D = -torch.exp(used(p["A_log"])), used(p["D"])
    ys, scan1 = [], []
    for i, (a, b) in enumerate(zip(off, off[1:])):
        h = scan0[i]
        for t in range(a, b):
            h = torch.exp(dl[t][:, None] * A) * h + (dl[t] * u[t])[:, None] * Bm[t]
            ys.append((h @ Cm[t] + D * u[t]) * F.silu(z[t]))
        scan1.append(h)
    y = stored(torch.stack(ys))
    return _linear(y, p["out_proj.weight"]), torch.stack(conv1), torch.stack(scan1)


def _residual(p, x, *rest):
    """ResidualMambaBlock: the norm's output is held in bf16, and the sum."""
    m, v = used(x).mean(-1, keepdim=True), used(x).var(-1, unbiased=False, keepdim=True)
    h = stored((used(x) - m) / torch.sqrt(v + 1e-5) * used(p["norm.weight"]) + used(p["norm.bias"]))
    inner = {k[len("mamba."):]: w for k, w in p.items() if k.startswith("mamba.")}
    y, conv1, scan1 = _block(inner, h, *rest)
    return stored(used(x) + used(y)), conv1, scan1


def _make(cuda, kind, seed):
    torch.manual_seed(seed)
    blk = getattr(mvm, kind)(64, d_state=16).to(cuda).bfloat16()
    p = {k: v.detach().double().cpu().requires_grad_(True) for k, v in blk.named_parameters()}
    return blk, p, (_block if kind == "MambaBlock" else _residual)


def _close(name, got, want):
    got, want = got.detach().double().cpu(), want.detach()
    assert got.shape == want.shape, name
    err, size = float((got - want).norm()), float(want.norm())
    assert err <= LIMIT * size, (name, err / size)


@pytest.mark.parametrize("kind", ["MambaBlock", "ResidualMambaBlock"])
def test_packed_block(cuda, kind):
    """Outputs, states and every gradient of packed sequences that start from states."""
    blk, p, oracle = _make(cuda, kind, 0)
    off, S = [0, 19, 20, 52, 52, 59], 5
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16()  # noqa: E731
    x, dy, conv0, dconv = r(59, 64), r(59, 64), r(S, 3, 128), r(S, 3, 128)
    scan0, dscan = torch.randn(S, 128, 16, generator=g), torch.randn(S, 128, 16, generator=g)
    live = [t.to(cuda).requires_grad_(True) for t in (x, conv0, scan0)]
    y, (conv1, scan1) = blk.forward_packed(live[0], off, (live[1], live[2]), max_len=32)
    assert y.dtype == conv1.dtype == torch.bfloat16 and scan1.dtype == torch.float32
    params = dict(blk.named_parameters())
    grads = torch.autograd.grad([y, conv1, scan1], [*live, *params.values()],
                                [t.to(cuda) for t in (dy, dconv, dscan)])
    refs = [t.double().requires_grad_(True) for t in (x, conv0, scan0)]
    want = oracle(p, refs[0], 16, off, refs[1], refs[2])
    wgrads = torch.autograd.grad(want, [*refs, *p.values()], [t.double() for t in (dy, dconv, dscan)])
    for n, a, b in zip(("y", "conv's states", "scan's states"), (y, conv1, scan1), want):
        _close(n, a, b)
    for n, a, b in zip(("x", "conv0", "scan0", *params), grads, wgrads):
        assert a.dtype == (torch.float32 if n == "scan0" else torch.bfloat16)
        _close("gradient of " + n, a, b)


@pytest.mark.parametrize("kind", ["MambaBlock", "ResidualMambaBlock"])
def test_served_block(cuda, kind):
    """A prompt in two pieces and single tokens, from a cache in shuffled order."""
    blk, p, oracle = _make(cuda, kind, 2)
    x = torch.randn(2, 24, 64, generator=torch.Generator().manual_seed(3)).bfloat16()
    zero = [torch.zeros(2, 3, 128, dtype=torch.float64), torch.zeros(2, 128, 16, dtype=torch.float64)]
    with torch.no_grad():
        want, conv1, scan1 = oracle(p, x.double().reshape(48, 64), 16, [0, 24, 48], *zero)
    states = blk.init_states(4)
    assert states[0].dtype == torch.bfloat16 and states[1].dtype == torch.float32
    for s in states:
        s.fill_(float("nan"))
    slots, xc = torch.tensor([3, 1], dtype=torch.int32, device=cuda), x.to(cuda)
    got = [blk.prefill(xc[:, :13], states, slots=slots, fresh=torch.tensor([True, True], device=cuda)),
           blk.prefill(xc[:, 13:18].reshape(10, 64), states, [0, 5, 10], slots=slots).view(2, 5, 64),
           *[blk.step(xc[:, t], states, slots=slots)[:, None] for t in range(18, 24)]]
    assert all(t.dtype == torch.bfloat16 for t in got)
    _close("y", torch.cat(got, 1).reshape(48, 64), want)
    _close("conv's states", states[0][[3, 1]], conv1)
    _close("scan's states", states[1][[3, 1]], scan1)


def test_example_in_bfloat16(cuda):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "stream_tokens.py")
    spec = importlib.util.spec_from_file_location("stream_tokens", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main(["--bf16"]) > 0.9
