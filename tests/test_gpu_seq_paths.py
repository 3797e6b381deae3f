"""The packed scan's and conv's launch variants: many sequences, many chunks,
chunks joined by the main pass or by the carry pass, several sequences a wave.
Against the float64 oracle, or bit for bit against the same work in smaller
calls, which take another variant."""

import pytest
import torch

import mlx_vision_mamba_amd as mvm
from tests import seq_reference as ref
from tests.test_gpu_seq import TYPES, _compare, _conv_inputs, _run_conv, _run_scan, _scan_inputs

pytestmark = pytest.mark.gpu


def _many(n, top, seed):
    return torch.randint(0, top, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_scan_of_many_sequences(cuda, dtype):
    """More sequences than a wave has lanes: the search for a chunk's sequence takes rounds."""
    lens = _many(150, 5, 1)
    _compare(*_run_scan(cuda, lens, *_scan_inputs(lens, 20, 4, TYPES[dtype], 60, extra=2), chunk_len=16))


def test_conv_of_many_sequences(cuda):
    lens = _many(200, 4, 2)
    _run_conv(cuda, lens, *_conv_inputs(lens, 24, 4, torch.float32, 61, extra=2))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("max_len", [100, None])
def test_scan_chunks_joined_by_either_pass(cuda, dtype, max_len):
    """Up to a few chunks a sequence the main pass joins them; without max_len
    one sequence might hold all tokens, and the carry pass does."""
    lens = [100, 0, 61, 16, 1, 97, 8, 99]
    ins = _scan_inputs(lens, 66, 16, TYPES[dtype], 62, extra=10)
    _compare(*_run_scan(cuda, lens, *ins, chunk_len=16, max_len=max_len))


def test_scan_carry_over_several_rounds(cuda):
    """More chunks of one sequence than the carry pass holds at once."""
    lens = [5, 2100, 30]
    ins = _scan_inputs(lens, 6, 3, torch.float32, 63)
    _compare(*_run_scan(cuda, lens, *ins, chunk_len=16))


@pytest.mark.parametrize("N", [16, 12])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_scan_step_of_many_sequences(cuda, dtype, N):
    """Several sequences a wave: the values of calls of one sequence a wave."""
    S, D = 4099, 260
    a, k, _, _ = _scan_inputs([1] * S, D, N, TYPES[dtype], 64)
    d = {n: v.to(cuda) for n, v in {**a, "z": k["z"]}.items()}
    slots = torch.randperm(S + 5, generator=torch.Generator().manual_seed(7))[:S].int()
    slots[17] = -1
    slots = slots.to(cuda)
    cache = torch.randn(S + 5, D, N, device=cuda)

    def run(lo, hi, states):
        cut = lambda n: d[n][lo:hi]
        return mvm.selective_scan_step(cut("u"), cut("delta"), d["A"], cut("B"), cut("C"), d["D"], states,
                                       slots=slots[lo:hi], z=cut("z"), delta_bias=k["delta_bias"].to(cuda),
                                       delta_softplus=True, a_is_log=True)

    one, many = cache.clone(), cache.clone()
    whole = run(0, S, many)
    parts = torch.cat([run(lo, min(S, lo + 500), one) for lo in range(0, S, 500)])
    assert torch.equal(whole, parts) and torch.equal(one, many) and not whole[17].any()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_conv_step_of_many_sequences(cuda, dtype):
    S, D = 1031, 1032
    x, w, b = torch.randn(S, D, device=cuda).to(TYPES[dtype]), torch.randn(D, 4, device=cuda), torch.randn(D, device=cuda)
    slots = torch.randperm(S + 3, generator=torch.Generator().manual_seed(8))[:S].int()
    slots[1030] = S + 3
    slots = slots.to(cuda)
    cache = torch.randn(S + 3, 3, D, device=cuda).to(TYPES[dtype])
    one, many = cache.clone(), cache.clone()
    whole = mvm.causal_conv_silu_step(x, w, b, many, slots=slots)
    parts = [mvm.causal_conv_silu_step(x[i:i + 100], w, b, one, slots=slots[i:i + 100]) for i in range(0, S, 100)]
    assert torch.equal(whole, torch.cat(parts)) and torch.equal(one, many) and not whole[1030].any()


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("W", [4, 8])
def test_conv_of_many_tokens(cuda, dtype, W):
    """Longer runs of positions a wave once the card is full: the values of
    calls that do not fill it."""
    lens, D = [2111, 2090, 1, 2070], 1544
    g = torch.Generator(device="cuda").manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=g, device=cuda)
    x, c0, dy = r(sum(lens), D).to(TYPES[dtype]), r(4, W - 1, D).to(TYPES[dtype]), r(sum(lens), D).to(TYPES[dtype])
    df, w, b = r(4, W - 1, D).to(TYPES[dtype]), r(D, W), r(D)

    def run(lo, hi, i, j):
        lv = [x[lo:hi].clone().requires_grad_(True), c0[i:j].clone().requires_grad_(True)]
        y, f = mvm.causal_conv_silu_packed(lv[0], w, b, [0] + torch.tensor(lens[i:j]).cumsum(0).tolist(),
                                           initial_states=lv[1])
        return [y.detach(), f.detach(), *torch.autograd.grad([y, f], lv, [dy[lo:hi], df[i:j]])]

    whole, at, parts = run(0, sum(lens), 0, 4), 0, []
    for i, n in enumerate(lens):
        parts.append(run(at, at + n, i, i + 1))
        at += n
    for p, q in zip(whole, zip(*parts)):
        assert torch.equal(p, torch.cat(q))


def test_scan_inputs_of_many_alignments(cuda):
    """States, A, B and C that do not start on 16 bytes are read four bytes at a time."""
    a, k, _, _ = _scan_inputs([1] * 6, 64, 16, torch.float32, 65)
    off = lambda t: torch.cat([torch.zeros(1), t.flatten()]).to(cuda)[1:].view(t.shape)
    init = k["initial"]
    want = ref.scan(list(range(7)), **a, initial=init, delta_softplus=True, a_is_log=True)
    states = off(init)
    y = mvm.selective_scan_step(*[off(v) for v in a.values()], states, delta_softplus=True, a_is_log=True)
    _compare({"y": y, "final": states}, want)
    want = ref.scan([0, 4, 6], **a, initial=init[:2], delta_softplus=True, a_is_log=True)
    states = off(init[:2])
    y = mvm.selective_scan_prefill(*[off(v) for v in a.values()], states, [0, 4, 6], delta_softplus=True, a_is_log=True)
    _compare({"y": y, "final": states}, want)


@pytest.mark.parametrize("gather", [False, True])
def test_prefill_in_place_is_the_same_as_apart(cuda, gather):
    """Chunks that the main pass joins, many more of them than run at once: the
    last one's final state replaces the initial state that all of them start from."""
    lens = [60 + 40 * (i % 2) for i in range(50)]
    off = [0] + torch.tensor(lens).cumsum(0).tolist()
    T, D, N, S = off[-1], 1536, 16, len(lens)
    gen = torch.Generator().manual_seed(66)
    r = lambda *s: torch.randn(*s, generator=gen).to(cuda)
    a = [r(T, D), 0.3 * r(T, D), 0.2 * r(D, N), r(T, N), r(T, N), r(D)]
    kw = dict(delta_softplus=True, a_is_log=True, max_len=100, chunk_len=16)
    init = r(S, D, N)
    y, final = mvm.selective_scan_packed(*a, off, initial_states=init, **kw)
    for _ in range(5):
        slots = torch.randperm(S, generator=gen).int().to(cuda) if gather else None
        states = init.clone() if slots is None else torch.empty_like(init).index_copy_(0, slots.long(), init)
        ys = mvm.selective_scan_prefill(*a, states, off, slots=slots, **kw)
        assert torch.equal(ys, y)
        assert torch.equal(states if slots is None else states[slots.long()], final)


@pytest.mark.parametrize("N", [4, 8, 12, 16])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_scan_step_lanes_of_a_channel(cuda, dtype, N):
    """One, two or four lanes a channel; several sequences a wave give the values of one a wave."""
    S, D = 1001, 515
    a, k, _, _ = _scan_inputs([1] * S, D, N, TYPES[dtype], 67)
    want = ref.scan(list(range(S + 1)), **a, **k, delta_softplus=True, a_is_log=True)
    d = {n: v.to(cuda) for n, v in {**a, "z": k["z"]}.items()}
    whole, parts = k["initial"].to(cuda), []
    y = mvm.selective_scan_step(*[d[n] for n in a], whole, z=d["z"], delta_bias=k["delta_bias"].to(cuda),
                                delta_softplus=True, a_is_log=True)
    _compare({"y": y, "final": whole}, want)
    cut = k["initial"].to(cuda)
    for lo in range(0, S, 90):
        rows = lambda n: d[n] if n in ("A", "D") else d[n][lo:lo + 90]
        parts.append(mvm.selective_scan_step(*[rows(n) for n in a], cut[lo:lo + 90], z=rows("z"), a_is_log=True,
                                             delta_bias=k["delta_bias"].to(cuda), delta_softplus=True))
    assert torch.equal(torch.cat(parts), y) and torch.equal(cut, whole)
