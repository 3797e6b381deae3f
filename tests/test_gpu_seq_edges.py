"""The packed and served scan and conv at the edges of what they accept:
caches of more rows than 32-bit products hold, traces,
grad mode, no channels, infinities in a last token,
single rows of any stride, no sequences, autocast."""

import pytest
import torch

import mlx_vision_mamba_amd as mvm
from mlx_vision_mamba_amd import gemm
from tests import seq_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def test_conv_cache_past_32_bit_products(cuda):
    """Rows of a cache of one channel whose number times the window's 7 earlier
    inputs passes 2^31: the state is read from the row that it is left in."""
    rows, W = 2 ** 31 // 7 + 64, 8
    if torch.cuda.mem_get_info()[0] < 3 * rows * 7 * 2:
        pytest.skip("not enough free memory")
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(9, 1, generator=g).bfloat16(), torch.randn(1, W, generator=g)
    states = torch.empty(rows, W - 1, 1, dtype=torch.bfloat16, device=cuda)
    slots = [rows - 1, 3]
    init = torch.randn(2, W - 1, 1, generator=g).bfloat16()
    for s, c in zip(slots, init):
        states[s] = c.to(cuda)
    y = mvm.causal_conv_silu_prefill(x.to(cuda), w.to(cuda), None, states, [0, 5, 9], slots=slots)
    want = ref.conv([0, 5, 9], x, w, initial=init)
    ref.check("y", y, want["y"])
    for i, s in enumerate(slots):
        ref.check("states", states[s], want["final"][i])
    # and the next token of both, by the step
    init = torch.stack([states[s] for s in slots]).cpu()
    x = torch.randn(2, 1, generator=g).bfloat16()
    y = mvm.causal_conv_silu_step(x.to(cuda), w.to(cuda), None, states, slots=slots)
    want = ref.conv([0, 1, 2], x, w, initial=init)
    ref.check("y", y, want["y"])
    for i, s in enumerate(slots):
        ref.check("states", states[s], want["final"][i])


class _Packed(torch.nn.Module):
    def __init__(self, kind, d_model, d_state):
        super().__init__()
        self.width = d_model
        self.block = getattr(mvm, kind)(d_model, d_state=d_state)

    def forward(self, x, offsets):
        y, (conv, scan) = self.block.forward_packed(x, offsets)
        return y, conv, scan


class _Products(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.width = 64
        self.w = torch.nn.Parameter(torch.randn(2 * 32, 64))
        self.v = torch.nn.Parameter(torch.randn(2, 24, 32))

    def forward(self, x, offsets):
        h = gemm.in_proj(x, self.w)
        return h, gemm.out_proj(h.view(-1, 2, 32), self.v)


@pytest.mark.parametrize("make", [
    # (the first one's x_proj and dt_proj are too narrow for the package's products)
    lambda: _Packed("MambaBlock", 32, 4), lambda: _Packed("MambaBlock", 64, 16),
    lambda: _Packed("ResidualMambaBlock", 64, 16), _Products], ids=["narrow", "mamba", "residual", "products"])
def test_traced_packed_blocks_compute(cuda, make):
    """A torch.jit trace runs the block again on new tokens and another cut of
    them: its outputs and gradients are the module's own."""
    torch.manual_seed(0)
    m = make().to(cuda)
    rn = lambda seed: torch.randn(40, m.width, generator=torch.Generator().manual_seed(seed)).to(cuda)  # noqa: E731
    off = lambda *o: torch.tensor(o, dtype=torch.int32, device=cuda)  # noqa: E731
    t = torch.jit.trace(m, (rn(0), off(0, 7, 40)), check_trace=False)
    x = rn(1).requires_grad_()
    for o in (off(0, 7, 40), off(0, 25, 31)):
        torch.full((1 << 20,), float("nan"), device=cuda)  # (what unwritten memory would hold)
        got, want = t(x, o), m(x, o)
        assert len(got) == len(want)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        g = [torch.randn(w.shape, generator=torch.Generator().manual_seed(2)).to(cuda) for w in want]
        ps = [x, *m.parameters()]
        for a, b in zip(torch.autograd.grad(got, ps, g), torch.autograd.grad(want, ps, g)):
            assert torch.equal(a, b)
    with torch.no_grad():
        for a, b in zip(t(x, o), m(x, o)):
            assert torch.equal(a, b) and a.grad_fn is None


@pytest.mark.parametrize("kind", ["MambaBlock", "ResidualMambaBlock"])
def test_served_blocks_build_no_graph(cuda, kind):
    """prefill and step in the default grad mode: values without a graph."""
    torch.manual_seed(0)
    blk = getattr(mvm, kind)(32, d_state=4).to(cuda)
    x = torch.randn(2, 5, 32, device=cuda, requires_grad=True)
    states, quiet = blk.init_states(2), blk.init_states(2)
    for name, arg in (("prefill", x), ("step", x[:, 0])):
        y = getattr(blk, name)(arg, states)
        assert torch.is_grad_enabled() and not y.requires_grad and y.grad_fn is None
        with torch.no_grad():
            assert torch.equal(y, getattr(blk, name)(arg, quiet))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [0, 1, 4099])
def test_gradients_of_no_channels(cuda, T, dtype):
    """Sums over no channels: B's and C's gradients are zero."""
    z = lambda *s: torch.zeros(*s, dtype=dtype, device=cuda, requires_grad=True)  # noqa: E731
    f = lambda *s: torch.zeros(*s, device=cuda, requires_grad=True)  # noqa: E731
    leaves = dict(u=z(T, 0), delta=z(T, 0), A=f(0, 13), B=z(T, 13), C=z(T, 13), D=f(0))
    y, final = mvm.selective_scan_packed(*leaves.values(), [0, T // 2, T], z=z(T, 0), delta_softplus=True)
    # what the allocator hands out again holds something else
    old = [torch.full((T * 13,), 7.0, dtype=dtype, device=cuda) for _ in range(4)]
    del old
    grads = torch.autograd.grad([y, final], list(leaves.values()), [torch.ones_like(y), torch.ones_like(final)])
    for (n, v), g in zip(leaves.items(), grads):
        assert g.shape == v.shape and g.dtype == v.dtype and not g.any(), n


def _check_kinds(name, got, want):
    """The oracle's infinities and NaN where it has them, within its bound elsewhere."""
    g, v = got.detach().double().cpu(), want.v
    assert torch.equal(torch.isnan(g), torch.isnan(v)), (name, "NaN")
    inf = torch.isinf(v)
    assert torch.equal(torch.isinf(g), inf) and torch.equal(g[inf], v[inf]), (name, "infinities")
    ok = torch.isfinite(v)
    ref.check(name, torch.where(ok.to(got.device), got, 0), ref.E(torch.where(ok, v, 0.0), torch.where(ok, want.e, 0.0)))


LAST = {"u": ("u", (4, 3)), "u negative": ("u", (15, 65)), "B": ("B", (4, 6)), "C": ("C", (15, 2)),
        "all of B": ("B", (35,)), "final's gradient": ("dfinal", (0, 9, 5)), "every one": ("u", (4, 11))}


@pytest.mark.parametrize("what", list(LAST))
@pytest.mark.parametrize("chunk", [0, 16])
@pytest.mark.parametrize("N", [8, 16])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_infinite_last_tokens(cuda, dtype, N, chunk, what):
    """A sequence ends inside a tile: what its last token makes infinite stays so,
    and nothing else turns into NaN (tokens 4, 15 and 35 are last ones)."""
    lens, D, t = [5, 8, 3, 20, 1], 70, TYPES[dtype]
    off = [0, 5, 13, 16, 36, 37]
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    a = dict(u=r(37, D).to(t), delta=(0.5 * r(37, D)).to(t), A=torch.log(torch.arange(1, N + 1).float()).repeat(D, 1),
             B=r(37, N).to(t), C=r(37, N).to(t), D=1 + 0.1 * r(D))
    k = dict(z=r(37, D).to(t), delta_bias=0.5 * r(D) - 3, initial=r(len(lens), D, N))
    dy, df = r(37, D).to(t), r(len(lens), D, N)
    name, at = LAST[what]
    (df if name == "dfinal" else a[name])[at] = float("-inf") if "negative" in what else float("inf")
    if what == "every one":
        a["B"][15, 1] = a["C"][35, 2] = df[1, 2, 3] = float("inf")
    leaves = {n: v.to(cuda).requires_grad_(True) for n, v in {**a, **k}.items()}
    y, final = mvm.selective_scan_packed(*[leaves[n] for n in a], off, z=leaves["z"], delta_bias=leaves["delta_bias"],
                                         initial_states=leaves["initial"], delta_softplus=True, a_is_log=True,
                                         chunk_len=chunk)
    grads = torch.autograd.grad([y, final], list(leaves.values()), [dy.to(cuda), df.to(cuda)])
    want = ref.scan(off, **a, **k, delta_softplus=True, a_is_log=True, dy=dy, dfinal=df)
    got = {"y": y, "final": final, **{"d" + n: v for n, v in zip(leaves, grads)}}
    for n, v in got.items():
        _check_kinds(n, v, want[n])


@pytest.mark.parametrize("dtype", list(TYPES))
def test_single_rows_of_any_stride(cuda, dtype):
    """One row has no next one: a stride that the kernels could not walk (the last
    token of a long history, say) is as good as any."""
    t, D, N = TYPES[dtype], 64, 16
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    a = dict(u=r(1, D).to(t), delta=r(1, D).to(t), A=-torch.rand(D, N, generator=g), B=r(1, N).to(t), C=r(1, N).to(t),
             D=r(D))
    z, init = r(1, D).to(t), r(1, D, N)
    want = ref.scan([0, 1], **a, z=z, initial=init, delta_softplus=True)
    far = lambda v: v.to(cuda).as_strided(v.shape, (2 ** 33 + 64, 1))  # noqa: E731
    rows = [far(v) if n in ("u", "delta", "B", "C") else v.to(cuda) for n, v in a.items()]
    states = init.to(cuda)
    y = mvm.selective_scan_step(*rows, states, z=far(z), delta_softplus=True)
    ref.check("y", y, want["y"])
    ref.check("states", states, want["final"])
    states = init.to(cuda)
    y = mvm.selective_scan_prefill(*rows, states, [0, 1], z=far(z), delta_softplus=True)
    ref.check("y", y, want["y"])
    y, final = mvm.selective_scan_packed(*rows, [0, 1], z=far(z), delta_softplus=True, initial_states=init.to(cuda))
    ref.check("y", y, want["y"])
    ref.check("final", final, want["final"])
    x, w, init = r(1, D).to(t), r(D, 4), r(1, 3, D).to(t)
    want = ref.conv([0, 1], x, w, initial=init)
    states = init.to(cuda)
    ref.check("y", mvm.causal_conv_silu_step(far(x), w.to(cuda), None, states), want["y"])
    ref.check("states", states, want["final"])
    y, final = mvm.causal_conv_silu_packed(far(x), w.to(cuda), None, [0, 1], initial_states=init.to(cuda))
    ref.check("y", y, want["y"])


def test_calls_of_no_sequences(cuda):
    """A scheduler's turn without any: empty outputs, an untouched cache."""
    D, N = 64, 16
    z = lambda *s: torch.zeros(*s, device=cuda)  # noqa: E731
    scan_ops = (z(0, D), z(0, D), -torch.ones(D, N, device=cuda), z(0, N), z(0, N), z(D))
    h, c = torch.randn(2, D, N, device=cuda), torch.randn(2, 3, D, device=cuda)
    h0, c0 = h.clone(), c.clone()
    for y in (mvm.selective_scan_step(*scan_ops, h, slots=[]), mvm.selective_scan_prefill(*scan_ops, h, [0], slots=[]),
              mvm.causal_conv_silu_step(z(0, D), z(D, 4), None, c, slots=[]),
              mvm.causal_conv_silu_prefill(z(0, D), z(D, 4), None, c, [0], slots=[])):
        assert y.shape == (0, D)
    assert torch.equal(h, h0) and torch.equal(c, c0)


@pytest.mark.parametrize("kind", ["MambaBlock", "ResidualMambaBlock"])
def test_served_under_autocast(cuda, kind):
    """The states that a block makes by default fit what it computes there: a
    prompt and single tokens give the packed form's values."""
    torch.manual_seed(3)
    blk = getattr(mvm, kind)(64).to(cuda)
    x = torch.randn(2, 12, 64, device=cuda)
    with torch.autocast("cuda", torch.bfloat16), torch.no_grad():
        want, (conv, _) = blk.forward_packed(x)
        states = blk.init_states(2)
        assert states[0].dtype == conv.dtype == torch.bfloat16 and states[1].dtype == torch.float32
        got = [blk.prefill(x[:, :9], states)] + [blk.step(x[:, t], states)[:, None] for t in range(9, 12)]
        # the same roundings to bf16 at the same places: float32 sums in another
        # order move a value across a border of half a step seldom, by one step
        got = torch.cat(got, 1)
        assert got.dtype == want.dtype and (got - want).float().norm() <= 2.0 ** -8 * want.float().norm()
    assert blk.init_states(2)[0].dtype == torch.float32
    with torch.autocast("cuda", torch.bfloat16):
        assert blk.init_states(2, dtype=torch.float32)[0].dtype == torch.float32  # what is asked for
