"""Backwards that are captured into a graph while an eager graph of the same
leaves is alive: the autograd engine would draw that graph's stream into the
capture, which ends the process.  Every backward of the package raises instead;
after the eager graph is gone, the same capture replays to the eager bits."""

import gc

import pytest
import torch

import mlx_vision_mamba_amd as mvm
from mlx_vision_mamba_amd.norm import layer_norm

pytestmark = pytest.mark.gpu


def _make(what, cuda):
    """(the call, its leaves)"""
    g = torch.Generator().manual_seed(60)
    r = lambda *s: (0.5 * torch.randn(*s, generator=g)).to(cuda).requires_grad_(True)  # noqa: E731
    off = torch.tensor([0, 25, 40], dtype=torch.int32, device=cuda)
    if what == "scan":
        t = [r(2, 20, 32), r(2, 20, 32), r(32, 16), r(2, 20, 16), r(2, 20, 16), r(32)]
        return lambda: mvm.selective_scan(t[0], t[1].square(), -t[2].square(), *t[3:]), t
    if what == "packed scan":
        t = [r(40, 32), r(40, 32), r(32, 16), r(40, 16), r(40, 16), r(32)]
        return lambda: mvm.selective_scan_packed(*t, off, delta_softplus=True, a_is_log=True)[0], t
    if what == "packed conv":
        t = [r(40, 32), r(32, 4), r(32)]
        return lambda: mvm.causal_conv_silu_packed(*t, off)[0], t
    if what == "norm":
        norm = torch.nn.LayerNorm(32).to(cuda)
        x = r(2, 20, 32)
        return lambda: layer_norm(x, norm), [x, *norm.parameters()]
    block = {"block": mvm.MambaBlock, "bidirectional": mvm.BidirectionalMambaBlock}[what](32, 16).to(cuda)
    x = r(2, 20, 32)
    return lambda: block(x), [x, *block.parameters()]


@pytest.mark.parametrize("what", ["scan", "packed scan", "packed conv", "norm", "block", "bidirectional"])
def test_beside_a_live_eager_graph(cuda, what):
    print("case:", what, flush=True)
    call, leaves = _make(what, cuda)
    dy = torch.randn(call().shape, generator=torch.Generator().manual_seed(61)).to(cuda)

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
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [t.detach() for t in work()]
    want = work()
    for x, y in zip(first, want[1:]):
        assert torch.equal(x, y)
    for _ in range(3):
        for t in captured:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        work()
        for x, y in zip(captured, want):
            assert torch.equal(x, y)
