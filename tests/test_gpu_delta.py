"""GPU parity of the gated delta rule against the float64 recurrence of
tests/delta_reference.py, within its tolerances; states, layouts, streams,
graph replays, rows of no sequence."""

import pytest
import torch

import mlx_vision_mamba_amd as mvm
from mlx_vision_mamba_amd import _lib
from tests import delta_reference as ref

pytestmark = pytest.mark.gpu

LENS = {"one": [1], "empty": [0, 5, 0], "chunk": [63, 64, 65, 1], "long": [130, 1, 0, 67], "none": []}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
NAMES = ("q", "k", "v", "g", "beta")


def _off(lens):
    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    return off


def _inputs(lens, HK, HV, DK, DV, dtype, seed, extra=0, beta_dtype=None, l2=True):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    T, S = sum(lens) + extra, len(lens)
    k = r(T, HK, DK)
    a = dict(q=r(T, HK, DK).to(dtype), k=(k if l2 else k / (k.norm(dim=-1, keepdim=True) + 1e-3) * 0.99).to(dtype),
             v=r(T, HV, DV).to(dtype), g=-torch.rand(T, HV, generator=gen) * torch.rand(HV, generator=gen),
             beta=torch.sigmoid(r(T, HV)).to(beta_dtype or dtype))
    return a, r(S, HV, DK, DV), r(T, HV, DV).to(dtype), r(S, HV, DK, DV)


def _call(cuda, lens, a, init, do, df, l2=True, use_init=True, scale=None, **more):
    """Outputs and gradients."""
    off, leaves = _off(lens), {n: x.to(cuda).requires_grad_(True) for n, x in a.items()}
    if use_init:
        leaves["initial"] = init.to(cuda).requires_grad_(True)
    o, final = mvm.gated_delta_rule_packed(*[leaves[n] for n in NAMES], torch.tensor(off, dtype=torch.int32, device=cuda),
                                           initial_states=leaves.get("initial"), qk_l2norm=l2, scale=scale, **more)
    grads = torch.autograd.grad([o, final], list(leaves.values()), [do.to(cuda), df.to(cuda)])
    got = {"o": o, "final": final, **{"d" + n: g for n, g in zip(leaves, grads)}}
    for n, g in got.items():
        want = o.dtype if n in ("o", "dq", "dk", "dv") else a["beta"].dtype if n == "dbeta" else torch.float32
        assert g.dtype == want, n
    return got


def _run(cuda, lens, a, init, do, df, l2=True, use_init=True, scale=None, **more):
    """(outputs and gradients on the GPU, the reference's, the factor of its tolerance)"""
    off, got = _off(lens), _call(cuda, lens, a, init, do, df, l2, use_init, scale, **more)
    want, factor = ref.reference(off, **a, qk_l2norm=l2, scale=scale, initial=init if use_init else None, do=do, dfinal=df)
    return got, want, factor


def _compare(got, want, factor):
    for n, g in got.items():
        ref.check(n, g, want[n], factor)


@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_packed(cuda, dtype, lens):
    ins = _inputs(LENS[lens], 2, 2, 32, 32, TYPES[dtype], 1, extra=3)
    _compare(*_run(cuda, LENS[lens], *ins))


@pytest.mark.parametrize("DK,DV", [(1, 1), (8, 16), (17, 33), (32, 64), (40, 100), (64, 128), (65, 70), (128, 128), (100, 200)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_packed_head_sizes(cuda, dtype, DK, DV):
    ins = _inputs([70, 20], 1, 1, DK, DV, TYPES[dtype], 2)
    _compare(*_run(cuda, [70, 20], *ins))


@pytest.mark.parametrize("HK,HV", [(1, 1), (3, 3), (2, 4), (1, 3)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_packed_shared_keys(cuda, dtype, HK, HV):
    ins = _inputs([66, 9], HK, HV, 24, 40, TYPES[dtype], 3)
    _compare(*_run(cuda, [66, 9], *ins))


@pytest.mark.parametrize("split", [64, 128, 192, 6400])
@pytest.mark.parametrize("DK,DV", [(32, 32), (60, 70), (128, 128)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_packed_splits(cuda, dtype, DK, DV, split):
    """Every split of the time axis gives the same function; the lengths end inside chunks and parts."""
    lens = [300, 0, 64, 129, 1]
    ins = _inputs(lens, 1, 2, DK, DV, TYPES[dtype], 30, extra=200)
    _compare(*_run(cuda, lens, *ins, split_len=split))
    _compare(*_run(cuda, lens, *ins, split_len=split, use_init=False, max_len=70))


@pytest.mark.parametrize("split", [0, 64])
@pytest.mark.parametrize("DK,DV", [(16, 128), (64, 72), (128, 96)])
def test_packed_many_heads(cuda, DK, DV, split):
    """Chunks and heads for a full card: bfloat16 takes its wider workgroups."""
    lens = [70, 0, 64, 5, 129]
    ins = _inputs(lens, 52, 104, DK, DV, torch.bfloat16, 32, extra=3)
    _compare(*_run(cuda, lens, *ins, split_len=split))


def test_prefill_in_parts(cuda):
    """A cache that is read and written by sequences in several parts."""
    lens = [200, 70, 0, 130]
    a, init, do, df = _inputs(lens, 2, 2, 32, 32, torch.bfloat16, 31)
    states = init.to(cuda)
    slots, fresh = [2, -1, 0, 3], [False, False, False, True]
    o = mvm.gated_delta_rule_prefill(*_on(cuda, a), states, _off(lens), slots=slots, qk_l2norm=True, split_len=64,
                                     fresh=torch.tensor(fresh, device=cuda))
    start = torch.stack([torch.zeros_like(init[0]) if s < 0 or f else init[s] for s, f in zip(slots, fresh)])
    want, factor = ref.reference(_off(lens), **a, qk_l2norm=True, initial=start)
    ref.check("o", o, want["o"], factor)
    for i, s in enumerate(slots):
        if s >= 0:
            ref.check("final", states[s], tuple(x[i] for x in want["final"]), factor)
    assert torch.equal(states[1].cpu(), init[1])


@pytest.mark.parametrize("options", [dict(l2=False), dict(use_init=False), dict(scale=0.7), dict(max_len=3), dict(max_len=10 ** 6)])
def test_packed_options(cuda, options):
    ins = _inputs([40, 90], 2, 2, 32, 48, torch.float32, 4, l2=options.get("l2", True))
    _compare(*_run(cuda, [40, 90], *ins, **options))


def test_packed_beta_in_float32(cuda):
    ins = _inputs([50, 21], 2, 2, 32, 32, torch.bfloat16, 5, beta_dtype=torch.float32)
    _compare(*_run(cuda, [50, 21], *ins))


def test_repeated_keys_and_strong_writes(cuda):
    """One key throughout, beta 1, no decay: every token replaces what the last one wrote."""
    a, init, do, df = _inputs([150], 1, 1, 32, 32, torch.float32, 6)
    a["k"] = a["k"][:1].expand(150, -1, -1).contiguous()
    a["g"], a["beta"] = torch.zeros_like(a["g"]), torch.ones_like(a["beta"])
    _compare(*_run(cuda, [150], a, init, do, df))


def test_decays_from_none_to_all(cuda):
    """g of 0, of -200 and of -inf (a state that starts over)."""
    a, init, do, df = _inputs([150], 1, 2, 32, 32, torch.float32, 7)
    a["g"][10], a["g"][70], a["g"][100] = -200.0, -1e30, -1e4
    a["g"][20:60] = 0.0
    got, want, factor = _run(cuda, [150], a, init, do, df)
    _compare(got, want, factor)
    a["g"][70] = float("-inf")
    again = _call(cuda, [150], a, init, do, df)
    for n in got:
        assert torch.equal(got[n], again[n]), n


@pytest.mark.parametrize("DK", [32, 100])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_gates_that_grow(cuda, dtype, DK):
    """g above 0 as well as below: pairs of tokens whose state grew between them."""
    a, init, do, df = _inputs([70, 131], 1, 2, DK, 32, TYPES[dtype], 14)
    a["g"] = 0.1 * torch.randn(a["g"].shape, generator=torch.Generator().manual_seed(15))
    a["g"][20:30] = 0.2
    _compare(*_run(cuda, [70, 131], a, init, do, df))
    _compare(*_run(cuda, [70, 131], a, init, do, df, split_len=64))


def test_batch_form_and_strides(cuda):
    """(B, L, ...) without offsets; operands that are columns of one wide projection."""
    Bn, L, HK, HV, DK, DV = 3, 21, 2, 4, 16, 24
    a, init, do, df = _inputs([L] * Bn, HK, HV, DK, DV, torch.bfloat16, 8)
    sizes = [HK * DK, HK * DK, HV * DV, HV]
    wide = torch.randn(Bn, L, 3 + sum(sizes), generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda)
    cut, at = {}, 3
    for n, s in zip(("q", "k", "v", "beta"), sizes):
        wide[..., at:at + s] = a[n].reshape(Bn, L, s).to(cuda)
        cut[n] = (at, s)
        at += s
    wide.requires_grad_(True)
    view = lambda n, *s: wide[..., cut[n][0]:cut[n][0] + cut[n][1]].view(Bn, L, *s)
    o, final = mvm.gated_delta_rule_packed(view("q", HK, DK), view("k", HK, DK), view("v", HV, DV),
                                           a["g"].view(Bn, L, HV).to(cuda), view("beta", HV), qk_l2norm=True,
                                           initial_states=init.to(cuda))
    assert o.shape == (Bn, L, HV, DV)
    (gw,) = torch.autograd.grad([o, final], [wide], [do.view(Bn, L, HV, DV).to(cuda), df.to(cuda)])
    want, factor = ref.reference(_off([L] * Bn), **a, qk_l2norm=True, initial=init, do=do, dfinal=df)
    got = {"o": o.flatten(0, 1), "final": final}
    for n in cut:
        got["d" + n] = gw.flatten(0, 1)[:, cut[n][0]:cut[n][0] + cut[n][1]].reshape(want["d" + n][0].shape)
    _compare(got, want, factor)


def test_transposed_heads(cuda):
    """(H, T, D) tensors seen as (T, H, D), and expanded ones."""
    a, init, do, df = _inputs([80], 2, 2, 32, 32, torch.float32, 9)
    a["k"] = a["k"][:, :1].expand(-1, 2, -1)
    b = {n: x.transpose(0, 1).contiguous().transpose(0, 1) if n in ("q", "v") else x for n, x in a.items()}
    b = {n: x.to(cuda) for n, x in b.items()}
    b["k"] = a["k"][:, :1].to(cuda).expand(-1, 2, -1)
    b["beta"] = a["beta"].to(cuda).t().contiguous().t()
    o, final = mvm.gated_delta_rule_packed(*[b[n] for n in NAMES], [0, 80], qk_l2norm=True, initial_states=init.to(cuda))
    want, factor = ref.reference([0, 80], **a, qk_l2norm=True, initial=init)
    _compare({"o": o, "final": final}, want, factor)


def test_rows_of_no_sequence_are_zero(cuda):
    a, init, do, df = _inputs([20, 30], 2, 4, 16, 16, torch.bfloat16, 10, extra=90)
    for n in NAMES:  # what lies there is not looked at
        a[n][50:] = float("nan")
    leaves = {n: x.to(cuda).requires_grad_(True) for n, x in a.items()}
    o, final = mvm.gated_delta_rule_packed(*leaves.values(), [0, 20, 50], qk_l2norm=True, initial_states=init.to(cuda))
    do[50:] = float("nan")
    grads = torch.autograd.grad([o, final], list(leaves.values()), [do.to(cuda), df.to(cuda)])
    assert bool((o[50:] == 0).all()) and bool(torch.isfinite(final).all())
    for g in grads:
        assert bool((g[50:] == 0).all()) and bool(torch.isfinite(g).all())


def test_a_value_that_is_not_finite_stays_in_its_sequence(cuda):
    a, init, do, df = _inputs([70, 70, 70], 1, 1, 32, 32, torch.float32, 11)
    clean = _call(cuda, [70, 70, 70], a, init, do, df)
    a["v"][75] = float("inf")
    a["k"][80] = float("nan")
    got = _call(cuda, [70, 70, 70], a, init, do, df)
    for n in ("o", "dq", "dk", "dv", "dg", "dbeta"):
        assert torch.equal(got[n][:70], clean[n][:70]) and torch.equal(got[n][140:], clean[n][140:]), n
    for i in (0, 2):
        assert torch.equal(got["final"][i], clean["final"][i]) and torch.equal(got["dinitial"][i], clean["dinitial"][i])


def test_only_one_gradient(cuda):
    """Through o alone, through the final states alone, and of some inputs only."""
    a, init, do, df = _inputs([70, 5], 1, 2, 16, 16, torch.float32, 12)
    for which in (0, 1):
        leaves = {n: x.to(cuda).requires_grad_(n in ("k", "g")) for n, x in a.items()}
        out = mvm.gated_delta_rule_packed(*leaves.values(), [0, 70, 75], qk_l2norm=True, initial_states=init.to(cuda))
        grads = torch.autograd.grad(out[which], [leaves["k"], leaves["g"]], (do, df)[which].to(cuda))
        want, factor = ref.reference([0, 70, 75], **a, qk_l2norm=True, initial=init, do=do if which == 0 else 0 * do,
                                     dfinal=df if which else None)
        _compare({"dk": grads[0], "dg": grads[1]}, want, factor)


def test_second_derivatives_are_refused(cuda):
    a, init, do, df = _inputs([9], 1, 1, 8, 8, torch.float32, 13)
    leaves = [x.to(cuda).requires_grad_(True) for x in a.values()]
    o, _ = mvm.gated_delta_rule_packed(*leaves, [0, 9], qk_l2norm=True)
    (g,) = torch.autograd.grad(o.sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match="not twice differentiable"):
        g.sum().backward()


# ------------------------------------------------------------------- serving

def _on(cuda, a):
    return [a[n].to(cuda) for n in NAMES]


@pytest.mark.parametrize("dtype", list(TYPES))
def test_prefill(cuda, dtype):
    """Rows of a larger cache; fresh and continued sequences, one without a row, an empty one."""
    lens = [70, 0, 5, 64, 33]
    a, init, do, df = _inputs(lens, 2, 4, 32, 48, TYPES[dtype], 20, extra=2)
    cache = torch.randn(9, 4, 32, 48, generator=torch.Generator().manual_seed(3))
    slots, fresh = [7, 2, -1, 0, 5], [False, False, False, True, False]
    states = cache.to(cuda)
    o = mvm.gated_delta_rule_prefill(*_on(cuda, a), states, _off(lens), slots=slots, qk_l2norm=True,
                                     fresh=torch.tensor(fresh, device=cuda))
    start = torch.stack([torch.zeros_like(cache[0]) if s < 0 or f else cache[s] for s, f in zip(slots, fresh)])
    want, factor = ref.reference(_off(lens), **a, qk_l2norm=True, initial=start)
    ref.check("o", o, want["o"], factor)
    for i, s in enumerate(slots):
        if s >= 0:
            ref.check("final", states[s], tuple(x[i] for x in want["final"]), factor)
    for s in set(range(9)) - set(slots):
        assert torch.equal(states[s].cpu(), cache[s])


@pytest.mark.parametrize("HK,HV,DK,DV", [(1, 1, 1, 1), (2, 4, 16, 17), (2, 2, 64, 64), (1, 2, 128, 130), (3, 3, 100, 128)])
@pytest.mark.parametrize("S", [1, 5])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_step(cuda, dtype, S, HK, HV, DK, DV):
    a, init, do, df = _inputs([1] * S, HK, HV, DK, DV, TYPES[dtype], 21)
    cache = torch.randn(S + 3, HV, DK, DV, generator=torch.Generator().manual_seed(3))
    slots = torch.randperm(S + 3, generator=torch.Generator().manual_seed(4))[:S].tolist()
    states = cache.to(cuda)
    o = mvm.gated_delta_rule_step(*_on(cuda, a), states, slots=slots, qk_l2norm=True)
    want, factor = ref.reference(list(range(S + 1)), **a, qk_l2norm=True, initial=cache[slots])
    ref.check("o", o, want["o"], factor)
    ref.check("final", states[slots], want["final"], factor)
    for s in set(range(S + 3)) - set(slots):
        assert torch.equal(states[s].cpu(), cache[s])


def test_step_many_sequences(cuda):
    """As many as take the variant for full cards; padding rows; without normalisation."""
    S, HK, HV, DK, DV = 300, 2, 2, 32, 64
    a, init, do, df = _inputs([1] * S, HK, HV, DK, DV, torch.bfloat16, 22, l2=False)
    slots = torch.arange(S, dtype=torch.int32)
    slots[[5, 77, 299]] = torch.tensor([-1, 1000, -7], dtype=torch.int32)
    states = init.to(cuda)
    o = mvm.gated_delta_rule_step(*_on(cuda, a), states, slots=slots.to(cuda))
    want, factor = ref.reference(list(range(S + 1)), **a, initial=init)
    none = torch.zeros(S, dtype=torch.bool)
    none[[5, 77, 299]] = True
    assert bool((o.cpu()[none] == 0).all()) and torch.equal(states.cpu()[none], init[none])
    ref.check("o", o.cpu()[~none], tuple(x[~none] for x in want["o"]), factor)
    ref.check("final", states.cpu()[~none], tuple(x[~none] for x in want["final"]), factor)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_prompts_in_pieces_and_steps_agree_with_packed(cuda, dtype):
    lens = [100, 37]
    a, init, do, df = _inputs(lens, 2, 2, 32, 32, TYPES[dtype], 23)
    want, factor = ref.reference(_off(lens), **a, qk_l2norm=True)
    x = {n: torch.stack([torch.nn.functional.pad(t[:100], (0,) * (2 * t.dim() - 1) + (0,)) if i == 0 else
                         torch.cat([t[100:], torch.zeros_like(t[:63])]) for i in range(2)]) for n, t in a.items()}
    states = torch.full((2, 2, 32, 32), float("nan"), device=cuda)
    outs, at, first = [[], []], [0, 0], True
    for piece in ([1, 30], [70, 0], [0, 3]):
        part = {n: torch.cat([x[n][i, at[i]:at[i] + piece[i]] for i in range(2)]) for n in NAMES}
        o = mvm.gated_delta_rule_prefill(*_on(cuda, part), states, _off(piece), qk_l2norm=True,
                                         fresh=torch.tensor([first, first], device=cuda))
        for i, got in enumerate(o.split(piece)):
            outs[i].append(got)
            at[i] += piece[i]
        first = False
    while at[0] < 100 or at[1] < 37:
        live = [i for i in range(2) if at[i] < lens[i]]
        part = {n: torch.stack([x[n][i, min(at[i], lens[i] - 1)] for i in range(2)]) for n in NAMES}
        slots = [i if i in live else -1 for i in range(2)]
        o = mvm.gated_delta_rule_step(*_on(cuda, part), states, slots=slots, qk_l2norm=True)
        for i in live:
            outs[i].append(o[i:i + 1])
            at[i] += 1
    # (every step rounds the states once more: 66 and 4 of them)
    ref.check("o", torch.cat(outs[0] + outs[1]), want["o"], 8 * factor)
    ref.check("final", states, want["final"], 8 * factor)


def test_cache_refusals(cuda):
    a, init, do, df = _inputs([4, 4], 1, 2, 8, 8, torch.float32, 24)
    args = _on(cuda, a)
    good = torch.zeros(2, 2, 8, 8, device=cuda)
    for states in (good[:1], good.double(), good[..., :4], good.transpose(2, 3), good[0]):
        with pytest.raises(ValueError, match="states"):
            mvm.gated_delta_rule_prefill(*args, states, [0, 4, 8])
    with pytest.raises(ValueError, match="in place"):
        mvm.gated_delta_rule_prefill(*args, good.clone().requires_grad_(True), [0, 4, 8])
    with pytest.raises(ValueError, match="fresh"):
        mvm.gated_delta_rule_prefill(*args, good, [0, 4, 8], fresh=torch.zeros(3, dtype=torch.bool, device=cuda))
    with pytest.raises(ValueError, match="slots"):
        mvm.gated_delta_rule_prefill(*args, good, [0, 4, 8], slots=torch.zeros(2, dtype=torch.int64, device=cuda))
    with pytest.raises(RuntimeError, match="must be on"):
        mvm.gated_delta_rule_prefill(*args, good.cpu(), [0, 4, 8])


def test_version_counter_and_streams(cuda):
    a, init, do, df = _inputs([70], 1, 2, 32, 32, torch.bfloat16, 25)
    args, states = _on(cuda, a), init.to(cuda)
    version = states._version
    mvm.gated_delta_rule_prefill(*args, states, [0, 70], qk_l2norm=True)
    assert states._version == version + 1
    one = mvm.gated_delta_rule_packed(*args, [0, 70], qk_l2norm=True)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two = mvm.gated_delta_rule_packed(*args, [0, 70], qk_l2norm=True)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(one, two)


def test_results_are_the_same_bits(cuda):
    ins = _inputs([300, 64, 17], 2, 4, 64, 72, torch.float32, 26)
    one = _call(cuda, [300, 64, 17], *ins)
    two = _call(cuda, [300, 64, 17], *ins)
    for n in one:
        assert torch.equal(one[n], two[n]), n


def test_graph_of_a_training_step_and_a_decode_step(cuda):
    a, init, do, df = _inputs([70, 60], 1, 2, 32, 32, torch.bfloat16, 27)
    leaves = {n: x.to(cuda).requires_grad_(True) for n, x in a.items()}
    off, dog = torch.tensor([0, 70, 130], dtype=torch.int32, device=cuda), do.to(cuda)
    states, tok = init.to(cuda), [x[:2].detach().clone() for x in leaves.values()]

    def work():
        o, final = mvm.gated_delta_rule_packed(*leaves.values(), off, qk_l2norm=True)
        grads = torch.autograd.grad(o, list(leaves.values()), dog)
        return [o.detach(), final.detach(), *grads, mvm.gated_delta_rule_step(*tok, states, qk_l2norm=True)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            leaves["v"].copy_(torch.randn(130, 2, 32, generator=g).bfloat16())
        before = states.clone()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured] + [states.clone()]
        states.copy_(before)
        want = work() + [states.clone()]
        for i, (x, y) in enumerate(zip(got, want)):
            assert torch.equal(x, y), i


def test_traced(cuda):
    a, init, do, df = _inputs([20], 1, 1, 16, 16, torch.float32, 28)
    off = torch.tensor([0, 20], dtype=torch.int32, device=cuda)

    class M(torch.nn.Module):
        def forward(self, q, k, v, g, beta):
            return mvm.gated_delta_rule_packed(q, k, v, g, beta, off, qk_l2norm=True)[0]

    args = _on(cuda, a)
    traced = torch.jit.trace(M(), args)
    args[2] = args[2] * 2
    assert torch.equal(traced(*args), M()(*args))
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda q, k, v, g, b: mvm.gated_delta_rule_step(q, k, v, g, b, init.to(cuda)), [x[:1] for x in args])
