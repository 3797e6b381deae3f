"""Mamba blocks on packed and served sequences: each sequence's values and
gradients are those of the block's ordinary forward on it alone, from pieces
and single tokens too; and the example that runs them together."""

import importlib.util
import os

import pytest
import torch

import mlx_vision_mamba_amd as mvm

pytestmark = pytest.mark.gpu

LENS = [19, 1, 40, 0, 7]


def _block(cuda, kind, seed=0):
    torch.manual_seed(seed)
    return getattr(mvm, kind)(32, d_state=8).to(cuda)


def _offsets(lens, cuda):
    return torch.tensor([0] + lens).cumsum(0).int().to(cuda)


def _close(got, want, what):
    # two float32 evaluations of one function; sums over 64 channels and 40
    # tokens of products of order one: 2^-24 times their number, both sides
    got, want = got.detach(), want.detach()
    scale = float(want.abs().max()) if want.numel() else 0.0
    err = float((got - want).abs().max()) if want.numel() else 0.0
    assert got.shape == want.shape and err <= 2 * 64 * 40 * 2.0 ** -24 * scale, (what, err, scale)


@pytest.mark.parametrize("kind", ["MambaBlock", "ResidualMambaBlock"])
def test_packed_block_is_the_block_on_each_sequence(cuda, kind):
    blk = _block(cuda, kind)
    x = torch.randn(sum(LENS), 32, device=cuda, requires_grad=True)
    dy = torch.randn(sum(LENS), 32, device=cuda)
    off = _offsets(LENS, cuda)
    params = dict(blk.named_parameters())
    y, (conv, scan) = blk.forward_packed(x, off, max_len=max(LENS))
    grads = torch.autograd.grad(y, [x, *params.values()], dy)
    assert conv.shape == (5, 3, 64) and scan.shape == (5, 64, 8)
    parts, o = [], off.tolist()
    for a, b in zip(o, o[1:]):
        if b > a:
            parts.append(blk(x[None, a:b])[0])
    _close(y, torch.cat(parts), "y")
    want = torch.autograd.grad(torch.cat(parts), [x, *params.values()], dy)
    for n, g, w in zip(["x", *params], grads, want):
        _close(g, w, n)


@pytest.mark.parametrize("kind", ["MambaBlock", "ResidualMambaBlock"])
def test_pieces_and_tokens_are_the_whole(cuda, kind):
    blk = _block(cuda, kind, 1)
    x = torch.randn(2, 30, 32, device=cuda)
    with torch.no_grad():
        want = blk(x)
        states = blk.init_states(4)
        states[0].fill_(float("nan"))
        states[1].fill_(float("nan"))
        slots = torch.tensor([3, 1], dtype=torch.int32, device=cuda)
        fresh = torch.tensor([True, True], device=cuda)
        a = blk.prefill(x[:, :13], states, slots=slots, fresh=fresh)
        b = blk.prefill(x[:, 13:24].reshape(-1, 32), states, _offsets([11, 11], cuda), slots=slots, max_len=11)
        c = torch.stack([blk.step(x[:, t].contiguous(), states, slots=slots) for t in range(24, 30)], 1)
        _close(torch.cat([a, b.view(2, 11, 32), c], 1), want, "y")
        # states of the differentiable form, carried by the caller
        y0, st = blk.forward_packed(x[:, :13])
        y1, st = blk.forward_packed(x[:, 13:], None, st)
        _close(torch.cat([y0, y1], 1), want, "y")
        whole = blk.forward_packed(x)[1]
        for p, q in zip(st, whole):
            _close(p, q, "state")


def test_bfloat16_block(cuda):
    blk = _block(cuda, "MambaBlock", 2)
    half = _block(cuda, "MambaBlock", 2).bfloat16()
    x = torch.randn(1, 20, 32, device=cuda).bfloat16()
    y, (conv, scan) = half.forward_packed(x)
    assert y.dtype == conv.dtype == torch.bfloat16 and scan.dtype == torch.float32
    want = blk(x.float())
    # seven roundings to bf16 on the way, each 2^-8 of values of the order of
    # the largest, through products of 32 to 64 terms
    assert float((y.float() - want).detach().abs().max()) <= 7 * 8 * 2.0 ** -8 * float(want.abs().max())


def test_replaced_scan_has_no_packed_form(cuda):
    blk = _block(cuda, "MambaBlock")
    blk._scan_fn = lambda *a: a[0]
    with pytest.raises(ValueError, match="packed"):
        blk.forward_packed(torch.zeros(1, 4, 32, device=cuda))
    with pytest.raises(ValueError, match="packed"):
        blk.step(torch.zeros(1, 32, device=cuda), blk.init_states(1))


def test_example(cuda):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "stream_tokens.py")
    spec = importlib.util.spec_from_file_location("stream_tokens", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.main([]) > 0.9
