"""The packed and served entry points' handling of their arguments on the host,
at the edges.  No kernel is launched."""

import ctypes

import pytest
import torch

from mlx_vision_mamba_amd import _lib, scan as scan_mod
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
