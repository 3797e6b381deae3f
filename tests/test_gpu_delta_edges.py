"""Edges of the gated delta rule and the group norm on the GPU: outputs,
checkpoints and workspaces stay inside their buffers whatever the device's
offsets say; layouts without 16-byte rows; offsets past 2^31 values; calls side
by side, captured, and beside a live eager graph."""

import ctypes
import gc

import pytest
import torch

import mlx_vision_mamba_amd as mvm
from mlx_vision_mamba_amd import _lib
from tests import delta_reference as ref
from tests import group_norm_reference as norm_ref
from tests.test_gpu_delta import NAMES, TYPES, _call, _compare, _inputs, _off, _run
from tests.test_gpu_seq_capi import CODE, OFFSETS, Fenced

pytestmark = pytest.mark.gpu


def _stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("offsets", list(OFFSETS))
@pytest.mark.parametrize("DK,DV,split", [(32, 32, 0), (33, 70, 0), (128, 128, 64), (24, 20, 64)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_delta_stays_in_its_buffers(cuda, dtype, DK, DV, split, offsets):
    T, S, HK, HV, t = 64, 5, 1, 2, TYPES[dtype]
    a, init, do, df = _inputs([T // S] * S, HK, HV, DK, DV, t, 1, extra=T - T // S * S)
    a, h0, do, df = {n: x.to(cuda) for n, x in a.items()}, init.to(cuda), do.to(cuda), df.to(cuda)
    off = torch.tensor(OFFSETS[offsets], dtype=torch.int32, device=cuda)
    d = _lib.DeltaDesc()
    d.seq.tokens, d.seq.nseq, d.seq.state_rows, d.seq.offsets = T, S, S, off.data_ptr()
    d.key_heads, d.value_heads, d.dk, d.dv = HK, HV, DK, DV
    d.q_stride = d.k_stride = HK * DK
    d.q_stride_head = d.k_stride_head = DK
    d.v_stride, d.v_stride_head, d.g_stride, d.beta_stride = HV * DV, DV, HV, HV
    d.scale, d.dtype, d.beta_dtype, d.qk_l2norm, d.split_len = DK ** -0.5, CODE[t], CODE[t], 1, split
    lib, p, buf = _lib.lib(), ctypes.byref(d), Fenced(cuda)
    ins = [a[n].data_ptr() for n in NAMES]
    ckpt = buf("ckpt", _lib.check(lib.mvm_delta_ckpt_elems(p)))
    n = _lib.check(lib.mvm_delta_workspace_bytes(p, 0))
    cells = S * HV * DK * DV
    _lib.check(lib.mvm_delta_fwd(p, *ins, h0.data_ptr(), buf("h1", cells), buf("o", T * HV * DV, t), ckpt,
                                 buf("workspace", n, torch.uint8), n, _stream()))
    buf.check()
    n = _lib.check(lib.mvm_delta_workspace_bytes(p, 1))
    outs = [buf(k, T * HK * DK, t) for k in ("dq", "dk")] + [buf("dv", T * HV * DV, t), buf("dg", T * HV),
                                                             buf("dbeta", T * HV, t), buf("dh0", cells)]
    _lib.check(lib.mvm_delta_bwd(p, *ins, ckpt, do.data_ptr(), df.data_ptr(), *outs,
                                 buf("workspace of the backward", n, torch.uint8), n, _stream()))
    buf.check()
    if offsets == "good":
        want, factor = ref.reference(OFFSETS[offsets], **a, qk_l2norm=True, initial=h0, do=do, dfinal=df)
        for name, key, shape, dt in [("o", "o", (T, HV, DV), t), ("h1", "final", (S, HV, DK, DV), None),
                                     ("dq", "dq", (T, HK, DK), t), ("dk", "dk", (T, HK, DK), t), ("dv", "dv", (T, HV, DV), t),
                                     ("dg", "dg", (T, HV), None), ("dbeta", "dbeta", (T, HV), t),
                                     ("dh0", "dinitial", (S, HV, DK, DV), None)]:
            ref.check(key, buf.value(name, *shape, dtype=dt or torch.float32), want[key], factor)


@pytest.mark.parametrize("S,HK,HV,DK,DV", [(5, 1, 2, 24, 20), (5, 1, 2, 33, 70), (300, 2, 2, 16, 64)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_delta_step_honours_fresh_and_stays_in_its_buffers(cuda, dtype, S, HK, HV, DK, DV):
    """A fresh sequence starts from zero whatever its row holds, here NaN."""
    t, rows = TYPES[dtype], S + 2
    a, _, _, _ = _inputs([1] * S, HK, HV, DK, DV, t, 2)
    g = torch.Generator().manual_seed(3)
    cache, slots, fresh = torch.randn(rows, HV, DK, DV, generator=g), torch.randperm(rows, generator=g)[:S], torch.rand(S, generator=g) < 0.5
    fresh[0] = True
    start = torch.where(fresh[:, None, None, None], 0.0, cache[slots])
    cache[slots[fresh]] = float("nan")
    buf = Fenced(cuda)
    states, o = buf("states", cache.numel()), buf("o", S * HV * DV, t)
    buf.value("states", *cache.shape).copy_(cache)
    on = {n: x.to(cuda) for n, x in a.items()}
    sl, fr = slots.int().to(cuda), fresh.to(cuda)
    d = _lib.DeltaDesc()
    d.seq.tokens, d.seq.nseq, d.seq.seqlen, d.seq.state_rows = S, S, 1, rows
    d.seq.slots, d.seq.fresh = sl.data_ptr(), fr.data_ptr()
    d.key_heads, d.value_heads, d.dk, d.dv = HK, HV, DK, DV
    d.q_stride = d.k_stride = HK * DK
    d.q_stride_head = d.k_stride_head = DK
    d.v_stride, d.v_stride_head, d.g_stride, d.beta_stride = HV * DV, DV, HV, HV
    d.scale, d.dtype, d.beta_dtype, d.qk_l2norm = DK ** -0.5, CODE[t], CODE[t], 1
    _lib.check(_lib.lib().mvm_delta_step(ctypes.byref(d), *[on[n].data_ptr() for n in NAMES], states, o, _stream()))
    buf.check()
    want, factor = ref.reference(list(range(S + 1)), **a, qk_l2norm=True, initial=start)
    got = buf.value("states", *cache.shape).cpu()
    ref.check("o", buf.value("o", S, HV, DV, dtype=t), want["o"], factor)
    ref.check("final", got[slots], want["final"], factor)
    rest = sorted(set(range(rows)) - set(slots.tolist()))
    assert torch.equal(got[rest], cache[rest])


@pytest.mark.parametrize("split", [0, 64])
@pytest.mark.parametrize("DK,DV", [(64, 300), (128, 512), (20, 257)])
def test_delta_wide_values(cuda, DK, DV, split):
    lens = [3, 130]
    _compare(*_run(cuda, lens, *_inputs(lens, 1, 1, DK, DV, torch.bfloat16, 4), split_len=split))


@pytest.mark.parametrize("shift", [1, 4])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_delta_rows_off_16_bytes(cuda, dtype, shift):
    """Columns of a wider buffer, with heads between others': forward, parts and gradients."""
    lens, HK, HV, D = [100, 45], 2, 4, 32
    a, init, do, df = _inputs(lens, HK, HV, D, D, TYPES[dtype], 5)
    want, factor = ref.reference(_off(lens), **a, qk_l2norm=True, initial=init, do=do, dfinal=df)
    for split in (0, 64):
        leaves = {}
        for n, x in a.items():
            buf = torch.full((x.shape[0], x.shape[1], 3 + 2 * (x.shape[2] if x.dim() == 3 else 1)), 9.0, dtype=x.dtype)
            view = buf[..., shift:shift + D] if x.dim() == 3 else buf[..., 1]
            view.copy_(x)
            buf = buf.to(cuda)
            leaves[n] = (buf[..., shift:shift + D] if x.dim() == 3 else buf[..., 1]).requires_grad_(True)
            assert not leaves[n].is_contiguous()
        h = init.to(cuda).requires_grad_(True)
        o, final = mvm.gated_delta_rule_packed(*leaves.values(), _off(lens), initial_states=h, qk_l2norm=True, split_len=split)
        grads = torch.autograd.grad([o, final], [*leaves.values(), h], [do.to(cuda), df.to(cuda)])
        _compare({"o": o, "final": final, **{"d" + n: g for n, g in zip([*leaves, "initial"], grads)}}, want, factor)


@pytest.mark.parametrize("split", [0, 64])
def test_delta_of_no_tokens(cuda, split):
    """Sequences without tokens hand their states and gradients through, in both forms."""
    init = torch.randn(2, 4, 8, 12, generator=torch.Generator().manual_seed(15)).to(cuda).requires_grad_(True)
    df = torch.randn(2, 4, 8, 12, generator=torch.Generator().manual_seed(16)).to(cuda)
    for lead, off in (((0,), [0, 0, 0]), ((2, 0), None)):
        r = lambda *s: torch.zeros(*lead, *s, device=cuda, requires_grad=True)  # noqa: E731
        leaves = [r(2, 8), r(2, 8), r(4, 12), r(4), r(4)]
        o, final = mvm.gated_delta_rule_packed(*leaves, off, initial_states=init, split_len=split)
        assert o.shape == (*lead, 4, 12) and torch.equal(final, init)
        grads = torch.autograd.grad([o, final], [*leaves, init], [torch.zeros_like(o), df])
        assert torch.equal(grads[-1], df) and all(g.shape == x.shape for g, x in zip(grads, leaves))
    states = init.detach().clone()
    o = mvm.gated_delta_rule_prefill(*[x.detach() for x in leaves], states, fresh=torch.tensor([True, False], device=cuda))
    assert o.shape == (2, 0, 4, 12) and not states[0].any() and torch.equal(states[1], init[1])
    o = mvm.gated_delta_rule_step(*[x.detach()[0] for x in leaves], states)
    assert o.shape == (0, 4, 12)


def test_delta_past_32_bits(cuda):
    """More than 2^31 values: the last sequence is what it is by itself, and so are its gradients."""
    HV, D, tail = 12, 128, 200
    T = 2 ** 31 // (HV * D) + 1000
    gen = torch.Generator(device=cuda).manual_seed(6)
    r = lambda *s: torch.randn(*s, generator=gen, device=cuda, dtype=torch.bfloat16)  # noqa: E731
    ins = [r(T, 1, D), r(T, 1, D), r(T, HV, D), -torch.rand(T, HV, generator=gen, device=cuda), r(T, HV).sigmoid()]
    do = r(T, HV, D)
    assert ins[2].numel() > 2 ** 31
    got = {}
    for name, cut, off in (("all", slice(None), [0, T - tail, T]), ("tail", slice(T - tail, T), [0, tail])):
        leaves = [x[cut].detach().requires_grad_(True) for x in ins]
        o, final = mvm.gated_delta_rule_packed(*leaves, off, qk_l2norm=True, split_len=64 * 512)
        grads = torch.autograd.grad(o, leaves, do[cut])
        got[name] = [x[-tail:].clone() for x in (o, *grads)] + [final[-1].clone()]
        del o, final, grads, leaves
    for i, (x, y) in enumerate(zip(got["all"], got["tail"])):
        assert torch.equal(x, y), i


@pytest.mark.parametrize("split", [0, 64])
def test_delta_rows_far_apart(cuda, split):
    """Tokens and heads as far from each other as is allowed, or nearly."""
    a, init, do, df = _inputs([67], 2, 2, 16, 16, torch.bfloat16, 13)
    leaves = {}
    for n, x in a.items():
        row = {"q": 2 ** 25 + 64, "k": 2 ** 25 + 64, "v": 2 ** 25}.get(n, 2 ** 22)
        buf = torch.zeros(67 * row, dtype=x.dtype, device=cuda)
        view = buf.as_strided(x.shape, (row, row // 2, 1)[:1] + ((row // 2, 1) if x.dim() == 3 else (1,)))
        view.copy_(x)
        leaves[n] = view.requires_grad_(True)
    o, final = mvm.gated_delta_rule_packed(*leaves.values(), [0, 67], qk_l2norm=True, split_len=split)
    grads = torch.autograd.grad([o, final], list(leaves.values()), [do.to(cuda), df.to(cuda)])
    want, factor = ref.reference([0, 67], **a, qk_l2norm=True, do=do, dfinal=df)
    _compare({"o": o, "final": final, **{"d" + n: g for n, g in zip(leaves, grads)}}, want, factor)


def test_norm_past_32_bits(cuda):
    """The last rows of more than 2^31 values, and a map of as many that repeats a small one."""
    ins = torch.randn(5, 1536, generator=torch.Generator().manual_seed(7)).bfloat16()
    x = torch.zeros(2 ** 31 // 1536 + 100, 1536, dtype=torch.bfloat16, device=cuda)
    x[-5:] = ins.to(cuda)
    y = mvm.group_norm(x, 12, torch.ones(1536, device=cuda), torch.zeros(1536, device=cuda), z=x)
    norm_ref.check("y", y[-5:], norm_ref.group_norm(x=ins, groups=12, weight=torch.ones(1536), bias=torch.zeros(1536), z=ins,
                                                    eps=1e-5)["y"])
    del x, y
    small = torch.randn(1, 4096, 64, generator=torch.Generator().manual_seed(8))
    want = norm_ref.group_norm(x=small.bfloat16(), groups=8, weight=torch.ones(64), bias=torch.zeros(64), eps=1e-5)["y"]
    big = small.bfloat16().to(cuda).repeat(1, 2 ** 19 // 64 + 1, 1)
    assert big.numel() > 2 ** 31
    y = mvm.group_norm(big, 8, torch.ones(64, device=cuda), torch.zeros(64, device=cuda))
    norm_ref.check("y", y[:, -4096:], want)


def test_delta_on_two_streams_at_once(cuda):
    lens = [150, 90]
    calls = [_inputs(lens, 1, 2, 64, 64, torch.bfloat16, s) for s in (9, 10)]
    want = [_call(cuda, lens, *c, split_len=64) for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], []
    for _ in range(3):
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(_call(cuda, lens, *c, split_len=64))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for n in g:
            assert torch.equal(g[n], want[i % 2][n]), n


@pytest.mark.parametrize("what", ["delta", "rows", "tile", "map"])
def test_captured(cuda, what):
    """Two graphs of the same leaves, replayed in turn with eager work between; a capture beside a live eager graph of
    them is refused, since the engine would draw that graph's stream into it."""
    if what == "delta":
        a, init, do, df = _inputs([130, 70], 1, 2, 32, 32, torch.bfloat16, 11)
        leaves = [x.to(cuda).requires_grad_(True) for x in a.values()]
        off, dy = torch.tensor([0, 130, 200], dtype=torch.int32, device=cuda), do.to(cuda)
        call = lambda: mvm.gated_delta_rule_packed(*leaves, off, qk_l2norm=True, split_len=64)[0]  # noqa: E731
    else:
        g = torch.Generator().manual_seed(12)
        shape = {"rows": (40, 64), "tile": (2, 30, 64), "map": (2, 3000, 64)}[what]
        x, dy = torch.randn(*shape, generator=g).to(cuda), torch.randn(*shape, generator=g).to(cuda)
        leaves = [x.requires_grad_(True), torch.ones(64, device=cuda, requires_grad=True)]
        call = lambda: mvm.group_norm(leaves[0], 4, leaves[1], activation="silu")  # noqa: E731

    def work():
        y = call()
        return [y, *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    eager = call()
    with pytest.raises(RuntimeError, match="an eager graph of its inputs is alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            work()
    first = torch.autograd.grad(eager, leaves, dy)  # (the eager graph still works)
    del eager
    gc.collect()
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append([t.detach() for t in work()])
    want = work()
    for x, y in zip(first, want[1:]):
        assert torch.equal(x, y)
    for i in (0, 1, 0, 1, 1):
        for t in outs[i]:
            t.zero_()
        graphs[i].replay()
        torch.cuda.synchronize()
        work()
        for x, y in zip(outs[i], want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("own", [True, False])
def test_captured_accumulation_beside_accumulators_of_another_stream(cuda, own):
    """backward() into .grad, with the leaves' accumulators kept alive by an eager graph of a side stream."""
    x = torch.randn(2, 30, 64, generator=torch.Generator().manual_seed(14)).to(cuda).requires_grad_(True)
    w = torch.ones(64, device=cuda, requires_grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kept = mvm.group_norm(x, 4, w)
        mvm.group_norm(x, 4, w).square().sum().backward()
    torch.cuda.current_stream().wait_stream(side)
    want = [x.grad.clone(), w.grad.clone()]
    x.grad = w.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side if own else None):
        mvm.group_norm(x, 4, w).square().sum().backward()
    del kept
    for _ in range(3):
        x.grad.zero_(), w.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for g, v in zip((x.grad, w.grad), want):
            assert torch.equal(g, v)
