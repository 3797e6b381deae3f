"""GPU parity of the packed and served scan and conv against the float64 oracle
of tests/seq_reference.py, within its running bound of float32's errors (and
half a step of bf16 where an output is held in it); their states, layouts,
streams, graph replays and refusals."""

import pytest
import torch

import mlx_vision_mamba_amd as mvm
from mlx_vision_mamba_amd import _lib
from tests import seq_reference as ref

pytestmark = pytest.mark.gpu

LENS = {"one": [1], "empty": [0, 5, 0], "tiles": [7, 8, 9, 16, 17, 1], "long": [130, 1, 0, 67], "none": []}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _off(lens):
    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    return off


def _scan_inputs(lens, D, N, dtype, seed, extra=0, delta_dtype=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    T, S = sum(lens) + extra, len(lens)
    a = dict(u=r(T, D).to(dtype), delta=(0.5 * r(T, D)).to(delta_dtype or dtype),
             A=torch.log(torch.arange(1, N + 1).float()).repeat(D, 1) + 0.1 * r(D, N), B=r(T, N).to(dtype),
             C=r(T, N).to(dtype), D=1 + 0.1 * r(D))
    k = dict(z=r(T, D).to(dtype), delta_bias=0.5 * r(D) - 3, initial=r(S, D, N))
    return a, k, r(T, D).to(dtype), r(S, D, N)


def _run_scan(cuda, lens, a, k, dy, df, gate=True, bias=True, soft=True, init=True, a_is_log=True, **more):
    """(outputs and gradients on the GPU, the oracle's)."""
    off = _off(lens)
    k = {n: v for n, v in k.items() if {"z": gate, "delta_bias": bias, "initial": init}[n]}
    leaves = {n: v.to(cuda).requires_grad_(True) for n, v in {**a, **k}.items()}
    pos = [leaves[n] for n in a]
    kw = {("initial_states" if n == "initial" else n): leaves[n] for n in k}
    y, final = mvm.selective_scan_packed(*pos, torch.tensor(off, dtype=torch.int32, device=cuda), delta_softplus=soft,
                                         a_is_log=a_is_log, **kw, **more)
    grads = torch.autograd.grad([y, final], list(leaves.values()), [dy.to(cuda), df.to(cuda)])
    got = {"y": y, "final": final, **{"d" + n: g for n, g in zip(leaves, grads)}}
    want = ref.scan(off, **a, **k, delta_softplus=soft, a_is_log=a_is_log, dy=dy, dfinal=df)
    return got, want


def _compare(got, want):
    for n, g in got.items():
        ref.check(n, g, want[n])


@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_scan_packed(cuda, dtype, lens):
    ins = _scan_inputs(LENS[lens], 70, 16, TYPES[dtype], 1, extra=3)
    _compare(*_run_scan(cuda, LENS[lens], *ins))


@pytest.mark.parametrize("N", [1, 4, 5, 12, 15])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_scan_packed_state_sizes(cuda, dtype, N):
    ins = _scan_inputs([20, 3], 64, N, TYPES[dtype], 2)
    _compare(*_run_scan(cuda, [20, 3], *ins))


@pytest.mark.parametrize("D", [1, 63, 65, 200])
def test_scan_packed_channels(cuda, D):
    ins = _scan_inputs([33, 40], D, 16, torch.float32, 3)
    _compare(*_run_scan(cuda, [33, 40], *ins))


@pytest.mark.parametrize("chunk", [16, 32, 64, 256])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_scan_packed_chunks(cuda, dtype, chunk):
    """Every cut gives the same function; the lengths end inside tiles and chunks."""
    lens = [100, 0, 16, 32, 61, 1]
    ins = _scan_inputs(lens, 66, 16, TYPES[dtype], 4, extra=40)
    _compare(*_run_scan(cuda, lens, *ins, chunk_len=chunk))


@pytest.mark.parametrize("options", [dict(gate=False), dict(bias=False), dict(init=False),
                                     dict(soft=False, bias=False), dict(a_is_log=False),
                                     dict(gate=False, bias=False, init=False)])
def test_scan_packed_options(cuda, options):
    a, k, dy, df = _scan_inputs([40, 9], 64, 16, torch.float32, 5)
    if not options.get("soft", True):
        a["delta"] = a["delta"].abs() * 0.1
    if not options.get("a_is_log", True):
        a["A"] = -a["A"].exp()
    _compare(*_run_scan(cuda, [40, 9], a, k, dy, df, chunk_len=16, **options))


def test_scan_packed_delta_in_float32(cuda):
    ins = _scan_inputs([50, 21], 64, 16, torch.bfloat16, 6, delta_dtype=torch.float32)
    _compare(*_run_scan(cuda, [50, 21], *ins))


def test_scan_max_len_is_only_a_hint(cuda):
    ins = _scan_inputs([100, 70], 64, 16, torch.float32, 7)
    for hint in (1, 70, 100, 10 ** 6):
        _compare(*_run_scan(cuda, [100, 70], *ins, max_len=hint))


def test_scan_batch_form_and_strides(cuda):
    """(B, L, D) without offsets; operands that are columns of wider rows."""
    Bn, L, D, N = 3, 21, 64, 16
    a, k, dy, df = _scan_inputs([L] * Bn, D, N, torch.bfloat16, 8)
    wide = torch.randn(Bn, L, 2 * D + 2 * N + 8, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda)
    wide[..., 4:4 + D] = a["u"].view(Bn, L, D).to(cuda)
    wide[..., 4 + D:4 + 2 * D] = k["z"].view(Bn, L, D).to(cuda)
    wide[..., -2 * N:-N] = a["B"].view(Bn, L, N).to(cuda)
    wide[..., -N:] = a["C"].view(Bn, L, N).to(cuda)
    wide.requires_grad_(True)
    init = k["initial"].to(cuda)
    y, final = mvm.selective_scan_packed(
        wide[..., 4:4 + D], a["delta"].view(Bn, L, D).to(cuda), a["A"].to(cuda), wide[..., -2 * N:-N], wide[..., -N:],
        a["D"].to(cuda), z=wide[..., 4 + D:4 + 2 * D], delta_bias=k["delta_bias"].to(cuda), delta_softplus=True,
        a_is_log=True, initial_states=init)
    assert y.shape == (Bn, L, D)
    (g,) = torch.autograd.grad([y, final], [wide], [dy.view(Bn, L, D).to(cuda), df.to(cuda)])
    want = ref.scan(_off([L] * Bn), **a, **k, delta_softplus=True, a_is_log=True, dy=dy, dfinal=df)
    g = g.view(Bn * L, -1)
    _compare({"y": y.view(-1, D), "final": final, "du": g[:, 4:4 + D], "dz": g[:, 4 + D:4 + 2 * D],
              "dB": g[:, -2 * N:-N], "dC": g[:, -N:]}, want)


def test_scan_odd_bc_alignment(cuda):
    """bf16 B and C rows that start between 4-byte words."""
    a, k, dy, df = _scan_inputs([40], 64, 16, torch.bfloat16, 9)
    wide = torch.zeros(40, 35, dtype=torch.bfloat16, device=cuda)
    wide[:, 1:17], wide[:, 17:33] = a["B"].to(cuda), a["C"].to(cuda)
    y, _ = mvm.selective_scan_packed(a["u"].to(cuda), a["delta"].to(cuda), a["A"].to(cuda), wide[:, 1:17],
                                     wide[:, 17:33], a["D"].to(cuda), [0, 40], a_is_log=True, delta_softplus=True)
    ref.check("y", y, ref.scan([0, 40], **a, delta_softplus=True, a_is_log=True)["y"])


def test_scan_broadcast_rows(cuda):
    """Inputs expanded over the rows (stride 0), their gradients summed."""
    g = torch.Generator().manual_seed(10)
    r = lambda *s: torch.randn(*s, generator=g)
    T, D, N = 30, 64, 16
    a = dict(u=r(1, D), delta=r(1, D), A=-torch.rand(D, N, generator=g), B=r(1, N), C=r(1, N), D=r(D))
    leaves = {n: v.to(cuda).requires_grad_(True) for n, v in a.items()}
    rows = {n: (v.expand(T, -1) if v.shape[0] == 1 else v) for n, v in leaves.items()}
    y, _ = mvm.selective_scan_packed(*rows.values(), [0, 10, T], delta_softplus=True)
    dy = r(T, D)
    grads = torch.autograd.grad(y, list(leaves.values()), dy.to(cuda))
    full = {n: (v.expand(T, -1) if v.shape[0] == 1 else v) for n, v in a.items()}
    want = ref.scan([0, 10, T], **full, delta_softplus=True, dy=dy)
    for n, got in zip(leaves, grads):
        w = want["d" + n]
        ref.check(n, got, w if a[n].shape[0] != 1 else ref.E(w.sum(0).v[None], w.sum(0).e[None]))


def test_scan_decays_that_vanish(cuda):
    """A so large that nothing survives a step, and A = -inf (A_log = inf)."""
    a, k, _, _ = _scan_inputs([19], 64, 16, torch.float32, 11)
    a["A"][:, 3] = 40.0
    a["A"][:, 5] = float("inf")
    y, final = mvm.selective_scan_packed(*[v.to(cuda) for v in a.values()], [0, 19], a_is_log=True,
                                         delta_softplus=True, initial_states=k["initial"].to(cuda))
    a["A"][:, 5] = 80.0  # exp(-delta e^80) is 0 as well, without inf * 0 in the oracle's bound
    want = ref.scan([0, 19], **a, initial=k["initial"], a_is_log=True, delta_softplus=True)
    for e in want.values():
        e.e = torch.nan_to_num(e.e, nan=0.0)
    _compare({"y": y, "final": final}, want)


def test_scan_bad_values_stay_in_their_sequence(cuda):
    """NaN and infinities of one sequence, and of rows of none, reach no other."""
    a, k, dy, df = _scan_inputs([12, 20, 9], 64, 16, torch.float32, 12, extra=6)
    for n in ("u", "delta", "B", "C"):
        a[n][12:32:3] = float("nan") if n != "u" else float("inf")
        a[n][41:] = float("nan")
    k["z"][41:] = float("nan")
    dy[41:] = float("nan")
    got, _ = _run_scan(cuda, [12, 20, 9], a, k, dy, df, chunk_len=16)
    keep = torch.tensor(list(range(12)) + list(range(32, 41)))
    clean = {n: torch.nan_to_num(v[keep], 0, 0, 0) if n in ("u", "delta", "B", "C") else v for n, v in a.items()}
    want = ref.scan([0, 12, 21], **clean, z=k["z"][keep], delta_bias=k["delta_bias"], initial=k["initial"][[0, 2]],
                    delta_softplus=True, a_is_log=True, dy=dy[keep], dfinal=df[[0, 2]])
    for n in ("y", "du", "ddelta", "dz", "dB", "dC"):
        ref.check(n, got[n][keep.to(cuda)], want[n])
        assert not got[n][41:].any(), n  # rows of no sequence: zero
    ref.check("final", got["final"][[0, 2]], want["final"])
    ref.check("dinitial", got["dinitial"][[0, 2]], want["dinitial"])


def test_scan_decreasing_offsets_stay_in_bounds(cuda):
    """Offsets on the GPU are not looked at: bad ones give some values, and every
    access is clamped.  The rows beside the tensors keep theirs."""
    a, k, dy, df = _scan_inputs([64], 64, 16, torch.float32, 13)
    fence = torch.full((4, 64), 7.0, device=cuda)
    off = torch.tensor([9, 70, -5, 30, 12, 1 << 30], dtype=torch.int32, device=cuda)
    leaves = [v.to(cuda).requires_grad_(True) for v in a.values()]
    y, final = mvm.selective_scan_packed(*leaves, off, chunk_len=16, a_is_log=True, delta_softplus=True)
    torch.autograd.grad(y.sum() + final.sum(), leaves)
    assert y.shape == (64, 64) and final.shape == (5, 64, 16)
    assert bool((fence == 7.0).all())


def test_scan_repeats_bit_for_bit(cuda):
    ins = _scan_inputs([300, 41, 160], 130, 16, torch.bfloat16, 14)
    one, _ = _run_scan(cuda, [300, 41, 160], *ins)
    two, _ = _run_scan(cuda, [300, 41, 160], *ins)
    for n in one:
        assert torch.equal(one[n], two[n]), n


def test_scan_unused_outputs_and_second_derivatives(cuda):
    a, k, dy, df = _scan_inputs([10, 4], 64, 16, torch.float32, 15)
    leaves = {n: v.to(cuda).requires_grad_(True) for n, v in {**a, "initial": k["initial"]}.items()}

    def run():
        return mvm.selective_scan_packed(*list(leaves.values())[:6], [0, 10, 14], a_is_log=True, delta_softplus=True,
                                         initial_states=leaves["initial"])
    y, _ = run()
    got = torch.autograd.grad(y, list(leaves.values()), dy.to(cuda))
    want = ref.scan([0, 10, 14], **a, initial=k["initial"], delta_softplus=True, a_is_log=True, dy=dy)
    _compare({"d" + n: g for n, g in zip(leaves, got)}, want)
    _, final = run()
    got = torch.autograd.grad(final, list(leaves.values()), df.to(cuda))
    want = ref.scan([0, 10, 14], **a, initial=k["initial"], delta_softplus=True, a_is_log=True,
                    dy=torch.zeros_like(dy), dfinal=df)
    _compare({"d" + n: g for n, g in zip(leaves, got)}, want)
    y, _ = run()
    (g,) = torch.autograd.grad(y.sum(), leaves["u"], create_graph=True)
    with pytest.raises(RuntimeError, match="not twice differentiable"):
        g.sum().backward()
    with torch.no_grad():
        assert not run()[0].requires_grad


# ------------------------------------------------------------ served: cache

@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("chunk", [0, 16])
def test_scan_prefill_on_a_cache(cuda, dtype, chunk):
    """Shuffled rows, a fresh sequence, one without a row; other rows keep their values."""
    lens, D, N = [30, 0, 17, 65, 4, 0], 64, 16
    a, k, _, _ = _scan_inputs(lens, D, N, TYPES[dtype], 20)
    cache = torch.randn(9, D, N, generator=torch.Generator().manual_seed(3))
    slots, fresh = [4, 8, 0, -1, 2, 5], [False, False, True, False, True, True]
    init = torch.stack([torch.zeros(D, N) if f or s < 0 else cache[s] for s, f in zip(slots, fresh)])
    want = ref.scan(_off(lens), **a, z=k["z"], delta_bias=k["delta_bias"], initial=init, delta_softplus=True,
                    a_is_log=True)
    states = cache.to(cuda)
    before = states._version
    y = mvm.selective_scan_prefill(*[v.to(cuda) for v in a.values()], states, _off(lens),
                                   slots=torch.tensor(slots, dtype=torch.int32, device=cuda),
                                   fresh=torch.tensor(fresh, device=cuda), z=k["z"].to(cuda),
                                   delta_bias=k["delta_bias"].to(cuda), delta_softplus=True, a_is_log=True,
                                   chunk_len=chunk)
    assert states._version > before
    ref.check("y", y, want["y"])
    for i, s in enumerate(slots):
        if s >= 0:
            ref.check(f"state {s}", states[s], want["final"][i])
    for s in (1, 3, 6, 7):
        assert torch.equal(states[s].cpu(), cache[s])


@pytest.mark.parametrize("N", [16, 8, 5, 1])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("S,D", [(1, 64), (5, 70), (3, 1)])
def test_scan_step(cuda, dtype, N, S, D):
    a, k, _, _ = _scan_inputs([1] * S, D, N, TYPES[dtype], 21)
    cache = torch.randn(S + 3, D, N, generator=torch.Generator().manual_seed(4))
    slots = [(2 * i + 1) % (S + 3) if i != 1 else S + 7 for i in range(S)]  # one is padding
    slots = [s if slots.index(s) == i else -1 for i, s in enumerate(slots)]
    init = torch.stack([cache[s] if 0 <= s < S + 3 else torch.zeros(D, N) for s in slots])
    want = ref.scan(list(range(S + 1)), **a, z=k["z"], delta_bias=k["delta_bias"], initial=init, delta_softplus=True,
                    a_is_log=True)
    states = cache.to(cuda)
    y = mvm.selective_scan_step(*[v.to(cuda) for v in a.values()], states, slots=slots, z=k["z"].to(cuda),
                                delta_bias=k["delta_bias"].to(cuda), delta_softplus=True, a_is_log=True)
    used = [i for i, s in enumerate(slots) if 0 <= s < S + 3]
    ref.check("y", y[used], want["y"][used])
    for i, s in enumerate(slots):
        if i in used:
            ref.check("state", states[s], want["final"][i])
        else:
            assert not y[i].any()
    for s in set(range(S + 3)) - set(slots):
        assert torch.equal(states[s].cpu(), cache[s])


def test_scan_step_without_options_and_empty(cuda):
    a, k, _, _ = _scan_inputs([1, 1], 64, 16, torch.float32, 22)
    a["delta"], a["A"] = a["delta"].abs(), -a["A"].exp()
    states = k["initial"].to(cuda)
    y = mvm.selective_scan_step(*[v.to(cuda) for v in a.values()], states)
    want = ref.scan([0, 1, 2], **a, initial=k["initial"])
    _compare({"y": y, "final": states}, want)
    none = [v.to(cuda)[:0] if n in ("u", "delta", "B", "C") else v.to(cuda) for n, v in a.items()]
    assert mvm.selective_scan_step(*none, states).shape == (0, 64)
    ref.check("kept", states, want["final"])


def test_scan_pieces_then_steps_match_the_whole(cuda):
    """A prompt in pieces and then token by token gives the whole sequence's values."""
    a, k, _, _ = _scan_inputs([57], 64, 16, torch.bfloat16, 23)
    want = ref.scan([0, 57], **a, z=k["z"], delta_bias=k["delta_bias"], delta_softplus=True, a_is_log=True)
    d = {n: v.to(cuda) for n, v in {**a, "z": k["z"]}.items()}
    states = torch.full((1, 64, 16), float("nan"), device=cuda)
    kw = dict(delta_bias=k["delta_bias"].to(cuda), delta_softplus=True, a_is_log=True)
    ys = []
    for lo, hi in ((0, 20), (20, 50)):
        cut = lambda n: d[n][lo:hi]
        ys.append(mvm.selective_scan_prefill(cut("u"), cut("delta"), d["A"], cut("B"), cut("C"), d["D"], states,
                                             [0, hi - lo], fresh=torch.tensor([lo == 0], device=cuda), z=cut("z"), **kw))
    for t in range(50, 57):
        cut = lambda n: d[n][t:t + 1]
        ys.append(mvm.selective_scan_step(cut("u"), cut("delta"), d["A"], cut("B"), cut("C"), d["D"], states,
                                          z=cut("z"), **kw))
    _compare({"y": torch.cat(ys), "final": states}, want)


# --------------------------------------------------------------------- conv

def _conv_inputs(lens, D, W, dtype, seed, extra=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    T, S = sum(lens) + extra, len(lens)
    return (dict(x=r(T, D).to(dtype), weight=r(D, W), bias=r(D), initial=r(S, W - 1, D).to(dtype)), r(T, D).to(dtype),
            r(S, W - 1, D).to(dtype))


def _run_conv(cuda, lens, a, dy, df, drop=()):
    a = {n: v for n, v in a.items() if n not in drop}
    leaves = {n: v.to(cuda).requires_grad_(True) for n, v in a.items()}
    y, final = mvm.causal_conv_silu_packed(leaves["x"], leaves["weight"], leaves.get("bias"),
                                           torch.tensor(_off(lens), dtype=torch.int32, device=cuda),
                                           initial_states=leaves.get("initial"))
    grads = torch.autograd.grad([y, final], list(leaves.values()), [dy.to(cuda), df.to(cuda)])
    _compare({"y": y, "final": final, **{"d" + n: g for n, g in zip(leaves, grads)}},
             ref.conv(_off(lens), **a, dy=dy, dfinal=df))


@pytest.mark.parametrize("lens", list(LENS))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_conv_packed(cuda, dtype, lens):
    _run_conv(cuda, LENS[lens], *_conv_inputs(LENS[lens], 72, 4, TYPES[dtype], 30, extra=5))


@pytest.mark.parametrize("W", range(1, 9))
@pytest.mark.parametrize("dtype", list(TYPES))
def test_conv_packed_widths(cuda, dtype, W):
    lens = [3, 70, 1, 0, 18]
    _run_conv(cuda, lens, *_conv_inputs(lens, 64, W, TYPES[dtype], 31))


@pytest.mark.parametrize("D", [1, 7, 66, 516])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_conv_packed_channels(cuda, dtype, D):
    _run_conv(cuda, [20, 5], *_conv_inputs([20, 5], D, 4, TYPES[dtype], 32))


@pytest.mark.parametrize("drop", [("bias",), ("initial",), ("bias", "initial")])
def test_conv_packed_options(cuda, drop):
    _run_conv(cuda, [20, 2], *_conv_inputs([20, 2], 64, 4, torch.float32, 33), drop=drop)


def test_conv_batch_form_strides_and_alignment(cuda):
    a, dy, df = _conv_inputs([21, 21], 64, 4, torch.bfloat16, 34)
    for at in (0, 1, 8):  # columns of wider rows, on and off 16 bytes
        wide = torch.zeros(2, 21, 80, dtype=torch.bfloat16, device=cuda)
        wide[..., at:at + 64] = a["x"].view(2, 21, 64).to(cuda)
        wide.requires_grad_(True)
        y, final = mvm.causal_conv_silu_packed(wide[..., at:at + 64], a["weight"].to(cuda), a["bias"].to(cuda),
                                               initial_states=a["initial"].to(cuda))
        (g,) = torch.autograd.grad([y, final], [wide], [dy.view(2, 21, 64).to(cuda), df.to(cuda)])
        want = ref.conv([0, 21, 42], **a, dy=dy, dfinal=df)
        _compare({"y": y.reshape(42, 64), "final": final, "dx": g[..., at:at + 64].reshape(42, 64)}, want)


@pytest.mark.parametrize("W", [1, 2, 4, 8])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_conv_prefill_and_step_on_a_cache(cuda, dtype, W):
    lens, D = [30, 0, 1, 65, 2, 0, 3], 72
    a, _, _ = _conv_inputs(lens, D, W, TYPES[dtype], 35)
    cache = torch.randn(9, W - 1, D, generator=torch.Generator().manual_seed(5)).to(TYPES[dtype])
    slots, fresh = [4, 8, 0, -1, 2, 5, 7], [False, False, True, False, True, True, False]
    init = torch.stack([torch.zeros_like(cache[0]) if f or s < 0 else cache[s] for s, f in zip(slots, fresh)])
    want = ref.conv(_off(lens), a["x"], a["weight"], a["bias"], initial=init)
    states = cache.to(cuda)
    y = mvm.causal_conv_silu_prefill(a["x"].to(cuda), a["weight"].to(cuda), a["bias"].to(cuda), states, _off(lens),
                                     slots=torch.tensor(slots, dtype=torch.int32, device=cuda),
                                     fresh=torch.tensor(fresh, device=cuda))
    ref.check("y", y, want["y"])
    for i, s in enumerate(slots):
        if s >= 0:
            assert torch.equal(states[s].cpu().double(), want["final"].v[i]), s
    for s in (1, 3, 6):
        assert torch.equal(states[s].cpu(), cache[s])
    # one token more for three of them and a padding row
    x = torch.randn(4, D, generator=torch.Generator().manual_seed(6)).to(TYPES[dtype])
    now = states.cpu()
    pick = [2, 11, 4, 7]
    init = torch.stack([now[s] if s < 9 else torch.zeros_like(now[0]) for s in pick])
    want = ref.conv([0, 1, 2, 3, 4], x, a["weight"], a["bias"], initial=init)
    y = mvm.causal_conv_silu_step(x.to(cuda), a["weight"].to(cuda), a["bias"].to(cuda), states, slots=pick)
    used = [0, 2, 3]
    ref.check("y", y[used], want["y"][used])
    assert not y[1].any()
    for i in used:
        assert torch.equal(states[pick[i]].cpu().double(), want["final"].v[i])


def test_conv_repeats_bit_for_bit(cuda):
    a, dy, df = _conv_inputs([300, 41], 132, 4, torch.float32, 36)
    runs = []
    for _ in range(2):
        lv = [a[n].to(cuda).requires_grad_(True) for n in ("x", "weight", "bias")]
        y, f = mvm.causal_conv_silu_packed(*lv, [0, 300, 341])
        runs.append([y, f, *torch.autograd.grad([y, f], lv, [dy.to(cuda), df.to(cuda)])])
    for p, q in zip(*runs):
        assert torch.equal(p, q)


# ---------------------------------------------------- streams, graphs, errors

def test_other_stream(cuda):
    ins = _scan_inputs([70, 12], 64, 16, torch.float32, 40)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, want = _run_scan(cuda, [70, 12], *ins)
    torch.cuda.current_stream().wait_stream(side)
    _compare(got, want)


def test_graph_replays_of_a_serving_step(cuda):
    """A token step of conv and scan captured once and replayed, with eager work
    between the replays, against eager steps on a second cache."""
    D, N, S = 64, 16, 3
    a, k, _, _ = _scan_inputs([1] * S, D, N, torch.bfloat16, 41)
    d = {n: v.to(cuda) for n, v in {**a, **k}.items()}
    w, b = torch.randn(D, 4, device=cuda), torch.randn(D, device=cuda)
    slots = torch.tensor([2, 0, 3], dtype=torch.int32, device=cuda)

    def caches():
        return torch.zeros(4, 3, D, dtype=torch.bfloat16, device=cuda), torch.zeros(4, D, N, device=cuda)

    def step(x, conv, scan):
        xc = mvm.causal_conv_silu_step(x, w, b, conv, slots=slots)
        return mvm.selective_scan_step(xc, d["delta"], d["A"], d["B"], d["C"], d["D"], scan, slots=slots, z=d["z"],
                                       delta_bias=d["delta_bias"], delta_softplus=True, a_is_log=True)

    x = torch.zeros(S, D, dtype=torch.bfloat16, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, *caches())
    torch.cuda.current_stream().wait_stream(side)
    mine, other = caches(), caches()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(x, *mine)
    for t in (*mine, *other):
        t.zero_()
    for i in range(5):
        x.copy_(torch.randn(S, D, generator=torch.Generator().manual_seed(i)))
        want = step(x, *other)
        torch.cuda.synchronize()
        graph.replay()
        assert torch.equal(y, want), i
        for p, q in zip(mine, other):
            assert torch.equal(p, q), i


def test_graph_replays_of_a_training_step(cuda):
    lens, off = [40, 0, 23], torch.tensor([0, 40, 40, 63], dtype=torch.int32, device=cuda)
    a, k, dy, df = _scan_inputs(lens, 64, 16, torch.float32, 42)
    d = {n: v.to(cuda) for n, v in {**a, **k}.items()}
    w, b = torch.randn(64, 4, device=cuda, requires_grad=True), torch.randn(64, device=cuda, requires_grad=True)
    x = d["u"].clone().requires_grad_(True)
    dy, df = dy.to(cuda), df.to(cuda)

    def step():
        xc, c = mvm.causal_conv_silu_packed(x, w, b, off)
        y, h = mvm.selective_scan_packed(xc, d["delta"], d["A"], d["B"], d["C"], d["D"], off, z=d["z"],
                                         delta_bias=d["delta_bias"], delta_softplus=True, a_is_log=True)
        return [y.detach(), *torch.autograd.grad([y, h], [x, w, b], [dy, df])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(63, 64, generator=torch.Generator().manual_seed(50 + i)))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        for p, q in zip(out, want):
            assert torch.equal(p, q), i


def test_gpu_refusals(cuda):
    a, k, _, _ = _scan_inputs([6], 8, 4, torch.float32, 43)
    d = [v.to(cuda) for v in a.values()]
    states = torch.zeros(2, 8, 4, device=cuda)
    one = [v[:1] if i in (0, 1, 3, 4) else v for i, v in enumerate(d)]
    off = torch.tensor([0, 6], dtype=torch.int32, device=cuda)
    for bad in (states.double(), states.transpose(1, 2), states[:, :7], states.clone().requires_grad_(True),
                torch.zeros(0, 8, 4, device=cuda)):
        with pytest.raises(ValueError):
            mvm.selective_scan_step(*one, bad)
        with pytest.raises(ValueError):
            mvm.selective_scan_prefill(*d, bad, off)
    for bad in (off.long(), off.float(), off[None], off[:0]):
        with pytest.raises(ValueError):
            mvm.selective_scan_packed(*d, bad)
    for bad in (torch.zeros(2, dtype=torch.int32, device=cuda), torch.zeros(1, dtype=torch.int64, device=cuda)):
        with pytest.raises(ValueError):
            mvm.selective_scan_step(*one, states, slots=bad)
    with pytest.raises(ValueError):
        mvm.selective_scan_prefill(*d, states, off, fresh=torch.zeros(1, device=cuda))
    with pytest.raises(RuntimeError):
        mvm.selective_scan_step(*one, states.cpu())
    with pytest.raises(ValueError):
        mvm.selective_scan_packed(*d, off, initial_states=states)
    conv = torch.zeros(2, 3, 8, device=cuda)
    w = torch.zeros(8, 4, device=cuda)
    with pytest.raises(ValueError):
        mvm.causal_conv_silu_step(one[0], w, None, conv.bfloat16())
    with pytest.raises(ValueError):
        mvm.causal_conv_silu_packed(d[0], w, None, off, initial_states=conv[:1].bfloat16())
    assert not states.any()
    assert _lib.lib().mvm_abi_version() == _lib.ABI_VERSION
