"""bfloat16 outputs of the gated delta rule are 32-bit results, rounded once.

Each output here is one product whose exact value a float32 holds, next to the
border between two bfloat16 values: it has to come out on the value's own side."""

import pytest
import torch

import mlx_vision_mamba_amd as mvm

pytestmark = pytest.mark.gpu


def _near_borders(*shape, seed):
    """float32 values a few float32 steps from the middle between two bfloat16 neighbours."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(*shape, generator=g).bfloat16().view(torch.int16).int() << 16) | 0x8000  # the middle
    off = torch.randint(1, 9, shape, generator=g) * (2 * torch.randint(0, 2, shape, generator=g) - 1)
    return (x + off.int()).view(torch.float32)


@pytest.mark.parametrize("heads", [1, 104])
@pytest.mark.parametrize("lens", [[1, 1], [70, 0, 130]])
@pytest.mark.parametrize("DK,DV", [(16, 16), (64, 128), (100, 70), (128, 128)])
def test_a_state_read_by_unit_queries(cuda, heads, lens, DK, DV):
    """o_t is a row of the initial state: nothing is written and nothing decays."""
    T, S = sum(lens), len(lens)
    init = _near_borders(S, heads, DK, DV, seed=1)
    row = torch.arange(T) * 7 % DK
    q = torch.nn.functional.one_hot(row, DK)[:, None].expand(T, heads, DK).bfloat16()
    k, v = torch.randn(T, heads, DK).bfloat16(), torch.randn(T, heads, DV).bfloat16()
    off = [sum(lens[:i]) for i in range(S + 1)]
    for split in (0, 64):
        o, final = mvm.gated_delta_rule_packed(*[x.to(cuda) for x in (q, k, v, torch.zeros(T, heads), torch.zeros(T, heads))],
                                               off, scale=1.0, initial_states=init.to(cuda), split_len=split)
        assert torch.equal(final.cpu(), init)
        seq = torch.repeat_interleave(torch.arange(S), torch.tensor(lens))
        assert torch.equal(o.cpu(), init[seq, :, row].bfloat16())


@pytest.mark.parametrize("heads", [1, 104])
@pytest.mark.parametrize("DK,DV", [(16, 16), (64, 128), (100, 70), (128, 128)])
def test_a_row_read_where_it_is_written(cuda, heads, DK, DV):
    """o_t = (q_t . k_t) beta_t v_t with unit q_t = k_t, all different within a sequence, and v_t a power of two."""
    lens = [min(DK, 70), 0, min(DK, 128)]
    T = sum(lens)
    off = [0, lens[0], lens[0], T]
    row = torch.cat([torch.arange(n) for n in lens])
    k = torch.nn.functional.one_hot(row, DK)[:, None].expand(T, heads, DK).bfloat16()
    beta = _near_borders(T, heads, seed=2)
    v = (2.0 ** torch.randint(-3, 4, (T, heads, DV), generator=torch.Generator().manual_seed(3))).bfloat16()
    for split in (0, 64):
        o, _ = mvm.gated_delta_rule_packed(*[x.to(cuda) for x in (k, k, v, torch.zeros(T, heads), beta)], off, scale=1.0,
                                           split_len=split)
        assert torch.equal(o.cpu(), (beta[..., None] * v.float()).bfloat16())
