"""The packed and served entry points' handling of their arguments on the host,
at the edges.  No kernel is launched."""

import ctypes

import pytest
import torch

from mlx_vision_mamba_amd import _lib, mamba_block as block_mod, scan as scan_mod
from tests.test_seq_host import _conv_desc, _scan_desc


@pytest.mark.parametrize("far", [2 ** 32, 2 ** 32 + 2, -2 ** 63, 2 ** 63 - 1, 2 ** 31, 4, -1])
def test_slots_outside_the_cache_never_name_a_row(far):
    """A slot outside the cache is padding, whatever its low 32 bits are."""
    for slots in ([0, far, far], torch.tensor([0, far, far])):
        got = scan_mod.sequence_slots(slots, 4, "cpu")
        assert got.dtype == torch.int32 and got.tolist() == [0, -1, -1]


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16, torch.int32, torch.int64])
def test_slots_of_any_integer_type(dtype):
    assert scan_mod.sequence_slots(torch.tensor([3, 0, 100], dtype=dtype), 4, "cpu").tolist() == [3, 0, -1]


@pytest.mark.parametrize("off", [4, 16, 128])
def test_unaligned_scratch_is_refused(off):
    """A workspace off 256 bytes, checkpoints off 16: refused before a launch.
    (Every operand is the address 1 << 20, which nothing reads.)"""
    lib, some, odd = _lib.lib(), ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + off)
    d, c = _scan_desc(), _conv_desc()
    d.chunk_len = 16
    ref = ctypes.byref(d)
    assert lib.mvm_seq_scan_fwd(ref, *[some] * 12, odd, 1 << 40, None) == _lib.MVM_ERR_WORKSPACE
    assert "256-byte" in _lib.last_error()
    assert lib.mvm_seq_scan_bwd(ref, *[some] * 20, odd, 1 << 40, None) == _lib.MVM_ERR_WORKSPACE
    assert lib.mvm_seq_conv_bwd(ctypes.byref(c), *[some] * 10, odd, 1 << 40, None) == _lib.MVM_ERR_WORKSPACE
    if off % 16 != 0:
        assert lib.mvm_seq_scan_fwd(ref, *[some] * 11, odd, some, 1 << 40, None) == _lib.MVM_ERR_INVALID_ARG
        assert "ckpt" in _lib.last_error()
        assert lib.mvm_seq_scan_bwd(ref, *[some] * 8, odd, *[some] * 11, some, 1 << 40, None) == _lib.MVM_ERR_INVALID_ARG
        assert "ckpt" in _lib.last_error()


@pytest.mark.parametrize("kind", ["MambaBlock", "ResidualMambaBlock"])
def test_served_blocks_build_no_graph(monkeypatch, kind):
    """prefill and step in the default grad mode: no gradients, not some."""
    for name in ("conv_silu", "selective_scan"):
        for form in ("prefill", "step"):
            fn = f"causal_conv_silu_{form}" if name == "conv_silu" else f"selective_scan_{form}"
            monkeypatch.setattr(block_mod, fn, lambda u, *a, **k: u.detach() * 0.5)
    monkeypatch.setattr(block_mod, "layer_norm", lambda x, norm, residual=False: norm(x))
    blk = getattr(block_mod, kind)(32, d_state=4)
    x = torch.randn(2, 5, 32, requires_grad=True)
    states = blk.init_states(2)
    for y in (blk.prefill(x, states), blk.step(x[:, 0], states)):
        assert torch.is_grad_enabled() and not y.requires_grad and y.grad_fn is None


def test_no_slots_in_a_list():
    """A call of no sequences: an empty list is a list of whole numbers."""
    got = scan_mod.sequence_slots([], 4, "cpu")
    assert got.dtype == torch.int32 and got.shape == (0,)
    for bad in ([0.5], torch.zeros(0), [[]]):
        with pytest.raises(ValueError, match="whole numbers"):
            scan_mod.sequence_slots(bad, 4, "cpu")
