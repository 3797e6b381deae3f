"""Options of the gated delta rule at the ends of their ranges."""

import pytest
import torch

import mlx_vision_mamba_amd as mvm
from mlx_vision_mamba_amd.delta import _split
from tests.test_gpu_delta import _inputs


def test_split_lengths_of_more_than_32_bits():
    """A part longer than any sequence is a whole sequence, not what 32 bits leave of its length."""
    for n in (2 ** 31, 2 ** 32, 2 ** 32 + 64, 2 ** 70):
        assert 2 ** 31 - 64 <= _split(n) < 2 ** 31 and _split(n) % 64 == 0
    assert [_split(n) for n in (0, 64, 2 ** 31 - 64)] == [0, 64, 2 ** 31 - 64]
    for n in (-64, 1, 2 ** 32 + 1):
        with pytest.raises(ValueError, match="split_len"):
            _split(n)


@pytest.mark.gpu
def test_split_lengths_past_the_sequences(cuda):
    a, init, _, _ = _inputs([130, 70], 1, 2, 16, 16, torch.float32, 50)
    call = lambda n: mvm.gated_delta_rule_packed(*[x.to(cuda) for x in a.values()], [0, 130, 200], qk_l2norm=True,  # noqa: E731
                                                 initial_states=init.to(cuda), split_len=n)
    want = call(192)
    for n in (2 ** 31 - 64, 2 ** 31, 2 ** 32 + 64, 2 ** 70):
        for x, y in zip(call(n), want):
            assert torch.equal(x, y)
