"""The packed and served scan and conv at the edges of what they accept:
caches of more rows than 32-bit products hold."""

import pytest
import torch

import mlx_vision_mamba_amd as mvm
from tests import seq_reference as ref

pytestmark = pytest.mark.gpu


def test_conv_cache_past_32_bit_products(cuda):
    """Rows of a cache of one channel whose number times the window's 7 earlier
    inputs passes 2^31: the state is read from the row that it is left in."""
    rows, W = 2 ** 31 // 7 + 64, 8
    if torch.cuda.mem_get_info()[0] < 3 * rows * 7 * 2:
        pytest.skip("not enough free memory")
    g = torch.Generator().manual_seed(1)
    x, w = torch.randn(9, 1, generator=g).bfloat16(), torch.randn(1, W, generator=g)
    states = torch.empty(rows, W - 1, 1, dtype=torch.bfloat16, device=cuda)
    slots = [rows - 1, 3]
    init = torch.randn(2, W - 1, 1, generator=g).bfloat16()
    for s, c in zip(slots, init):
        states[s] = c.to(cuda)
    y = mvm.causal_conv_silu_prefill(x.to(cuda), w.to(cuda), None, states, [0, 5, 9], slots=slots)
    want = ref.conv([0, 5, 9], x, w, initial=init)
    ref.check("y", y, want["y"])
    for i, s in enumerate(slots):
        ref.check("states", states[s], want["final"][i])
    # and the next token of both, by the step
    init = torch.stack([states[s] for s in slots]).cpu()
    x = torch.randn(2, 1, generator=g).bfloat16()
    y = mvm.causal_conv_silu_step(x.to(cuda), w.to(cuda), None, states, slots=slots)
    want = ref.conv([0, 1, 2], x, w, initial=init)
    ref.check("y", y, want["y"])
    for i, s in enumerate(slots):
        ref.check("states", states[s], want["final"][i])
