"""The packed and served entry points' handling of their arguments on the host,
at the edges.  No kernel is launched."""

import pytest
import torch

from mlx_vision_mamba_amd import scan as scan_mod


@pytest.mark.parametrize("far", [2 ** 32, 2 ** 32 + 2, -2 ** 63, 2 ** 63 - 1, 2 ** 31, 4, -1])
def test_slots_outside_the_cache_never_name_a_row(far):
    """A slot outside the cache is padding, whatever its low 32 bits are."""
    for slots in ([0, far, far], torch.tensor([0, far, far])):
        got = scan_mod.sequence_slots(slots, 4, "cpu")
        assert got.dtype == torch.int32 and got.tolist() == [0, -1, -1]


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int16, torch.int32, torch.int64])
def test_slots_of_any_integer_type(dtype):
    assert scan_mod.sequence_slots(torch.tensor([3, 0, 100], dtype=dtype), 4, "cpu").tolist() == [3, 0, -1]
