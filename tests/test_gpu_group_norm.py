"""GPU parity of the group norm against the float64 reference of
tests/group_norm_reference.py within its running error bound; layouts, edges,
graph replays."""

import pytest
import torch

import mlx_vision_mamba_amd as mvm
from tests import group_norm_reference as ref

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _inputs(shape, dtype, seed, mean=0.5):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    C = shape[-1]
    return dict(x=(r(*shape) * (1 + 0.2 * r(C)) + mean * r(C)).to(dtype), weight=1 + 0.1 * r(C), bias=0.1 * r(C),
                z=r(*shape).to(dtype)), r(*shape).to(dtype)


def _run(cuda, groups, ins, dy, silu=False, gate=True, affine=True, eps=1e-5):
    ins = {n: t for n, t in ins.items() if (n != "z" or gate) and (affine or n in ("x", "z"))}
    leaves = {n: t.to(cuda).requires_grad_(True) for n, t in ins.items()}
    y = mvm.group_norm(leaves["x"], groups, leaves.get("weight"), leaves.get("bias"), eps, z=leaves.get("z"),
                       activation="silu" if silu else None)
    grads = torch.autograd.grad(y, list(leaves.values()), dy.to(cuda))
    got = {"y": y, **{"d" + n: g for n, g in zip(leaves, grads)}}
    for n, g in got.items():
        assert g.dtype == (torch.float32 if n in ("dweight", "dbias") else ins["x"].dtype), n
    return got, ref.group_norm(groups=groups, eps=eps, silu=silu, dy=dy, **ins)


def _compare(got, want):
    for n, g in got.items():
        ref.check(n, g, want[n])


@pytest.mark.parametrize("groups,C", [(1, 1), (1, 8), (4, 24), (12, 1536), (3, 111), (1, 513), (2, 1040), (1, 1531), (7, 7),
                                      (32, 96), (1, 2048), (1, 2052)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_rows(cuda, dtype, groups, C):
    ins, dy = _inputs((5, C), TYPES[dtype], 1)
    _compare(*_run(cuda, groups, ins, dy))


@pytest.mark.parametrize("silu,gate,affine", [(s, g, a) for s in (0, 1) for g in (0, 1) for a in (0, 1)])
@pytest.mark.parametrize("shape", [(6, 64), (3, 10, 64)])
def test_options(cuda, shape, silu, gate, affine):
    ins, dy = _inputs(shape, torch.float32, 2)
    _compare(*_run(cuda, 8, ins, dy, bool(silu), bool(gate), bool(affine)))


@pytest.mark.parametrize("shape,groups", [((2, 2, 8), 2), ((3, 7, 24), 4), ((2, 14, 14, 384), 32), ((1, 3, 1000, 37), 37),
                                          ((2, 300, 148), 4), ((1, 2900, 3), 1), ((1, 17, 4104), 2), ((40, 3, 12), 3),
                                          ((2, 1, 1, 16), 2)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_maps(cuda, dtype, shape, groups):
    ins, dy = _inputs(shape, TYPES[dtype], 3)
    _compare(*_run(cuda, groups, ins, dy, silu=True, gate=False))
    _compare(*_run(cuda, groups, ins, dy))


# groups of 256, 128 and 64 lanes, of as many rows as a workgroup's registers hold and of one more; many groups of one
# access; partial sums for four waves to join
@pytest.mark.parametrize("shape,groups", [((2, 8, 1024), 1), ((2, 9, 1024), 1), ((3, 16, 512), 1), ((3, 17, 512), 1),
                                          ((2, 33, 256), 1), ((2, 64, 96), 2), ((2100, 3, 16), 4), ((1, 20000, 32), 2),
                                          ((9, 1, 2, 2048), 1)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_tiles_and_their_borders(cuda, dtype, shape, groups):
    ins, dy = _inputs(shape, TYPES[dtype], 14)
    _compare(*_run(cuda, groups, ins, dy, silu=True, gate=True))
    _compare(*_run(cuda, groups, ins, dy, gate=False))


def test_rows_many(cuda):
    """More rows than the waves that walk them."""
    ins, dy = _inputs((9000, 48), torch.bfloat16, 4)
    _compare(*_run(cuda, 3, ins, dy))


@pytest.mark.parametrize("shape", [(4, 96), (2, 50, 96), (2, 3000, 96)])
def test_a_mean_far_from_zero(cuda, shape):
    """Means of thousands of standard deviations: what the values' own rounding leaves is kept."""
    ins, dy = _inputs(shape, torch.float32, 5)
    ins["x"] = ins["x"] + 4096.0
    got, want = _run(cuda, 4, ins, dy)
    _compare(got, want)
    # (the rounding of the mean, a few units of 4096, beside values of order one)
    assert float((got["y"].detach().cpu().double() - want["y"].v).norm() / want["y"].v.norm()) < 4096 * 2 ** -22


@pytest.mark.parametrize("shape", [(4, 32), (2, 50, 32), (2, 5000, 32)])
def test_constant_groups_and_eps(cuda, shape):
    ins, dy = _inputs(shape, torch.float32, 6)
    ins["x"][..., :8] = 3.0
    for eps in (1e-5, 1e-2):
        _compare(*_run(cuda, 4, ins, dy, eps=eps))


@pytest.mark.parametrize("shape", [(4, 32), (2, 50, 32), (2, 5000, 32)])
def test_a_value_that_is_not_finite_stays_in_its_group(cuda, shape):
    ins, dy = _inputs(shape, torch.float32, 7)
    clean, _ = _run(cuda, 4, ins, dy)
    ins["x"][(1,) + (0,) * (len(shape) - 2) + (9,)] = float("inf")
    got, _ = _run(cuda, 4, ins, dy)
    for n in ("y", "dx", "dz"):
        bad = torch.zeros(shape, dtype=torch.bool)
        bad[1, ..., 8:16] = True
        assert torch.equal(got[n].cpu()[~bad], clean[n].cpu()[~bad]), n
        assert not bool(torch.isfinite(got[n].cpu()[bad]).any()), n


@pytest.mark.parametrize("dtype", list(TYPES))
def test_strides(cuda, dtype):
    """Columns of wider rows (aligned and not), transposed maps, an expanded dy."""
    g = torch.Generator().manual_seed(8)
    for lead in (3, 8):
        wide = torch.randn(5, 6, 100, generator=g).to(TYPES[dtype]).to(cuda).requires_grad_(True)
        x, z = wide[..., lead:lead + 32], wide[..., lead + 40:lead + 72]
        y = mvm.group_norm(x, 4, z=z)
        (gw,) = torch.autograd.grad(y, wide, torch.ones((), device=cuda, dtype=y.dtype).expand(y.shape))
        want = ref.group_norm(x.detach().cpu(), 4, z=z.detach().cpu(), dy=torch.ones(y.shape, dtype=y.dtype))
        _compare({"y": y, "dx": gw[..., lead:lead + 32], "dz": gw[..., lead + 40:lead + 72]}, want)
        assert y.is_contiguous()
    x = torch.randn(2, 16, 5, 7, generator=g).to(TYPES[dtype])  # channels first in memory
    _compare({"y": mvm.group_norm(x.to(cuda).permute(0, 2, 3, 1), 4)}, ref.group_norm(x.permute(0, 2, 3, 1), 4))


@pytest.mark.parametrize("shape", [(0, 8), (3, 0, 8), (0, 4, 8)])
def test_nothing(cuda, shape):
    ins, dy = _inputs(shape, torch.float32, 9)
    leaves = {n: t.to(cuda).requires_grad_(True) for n, t in ins.items()}
    y = mvm.group_norm(leaves["x"], 2, leaves["weight"], leaves["bias"], z=leaves["z"])
    grads = torch.autograd.grad(y, list(leaves.values()), dy.to(cuda))
    assert y.shape == shape and grads[0].shape == shape
    assert bool((grads[1] == 0).all()) and bool((grads[2] == 0).all())


def test_parameters_of_other_types(cuda):
    ins, dy = _inputs((5, 32), torch.bfloat16, 10)
    leaves = {n: t.to(cuda, torch.bfloat16).requires_grad_(True) for n, t in ins.items()}
    y = mvm.group_norm(leaves["x"], 4, leaves["weight"], leaves["bias"], z=leaves["z"])
    grads = torch.autograd.grad(y, list(leaves.values()), dy.to(cuda))
    want = ref.group_norm(groups=4, dy=dy, **{n: t.detach().cpu() for n, t in leaves.items()})
    _compare({"y": y, **{"d" + n: g for n, g in zip(leaves, grads)}}, want)
    assert all(g.dtype == torch.bfloat16 for g in grads)


@pytest.mark.parametrize("shape", [(700, 96), (3, 200, 96)])
def test_same_bits_streams_and_replays(cuda, shape):
    ins, dy = _inputs(shape, torch.bfloat16, 11)
    leaves = {n: t.to(cuda).requires_grad_(True) for n, t in ins.items()}
    d = dy.to(cuda)

    def work():
        y = mvm.group_norm(leaves["x"], 3, leaves["weight"], leaves["bias"], z=leaves["z"], activation="silu")
        return [y.detach(), *torch.autograd.grad(y, list(leaves.values()), d)]

    one = work()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        two = work()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for seed in range(3):
        with torch.no_grad():
            leaves["x"].copy_(torch.randn(shape, generator=torch.Generator().manual_seed(seed)).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(got, work())), seed


def test_second_derivatives_are_refused_and_traces_keep_the_call(cuda):
    ins, dy = _inputs((5, 32), torch.float32, 12)
    leaves = {n: t.to(cuda).requires_grad_(True) for n, t in ins.items()}
    y = mvm.group_norm(leaves["x"], 4, leaves["weight"], leaves["bias"])
    (g,) = torch.autograd.grad(y.sum(), leaves["x"], create_graph=True)
    with pytest.raises(RuntimeError, match="not twice differentiable"):
        g.sum().backward()

    class M(torch.nn.Module):
        def forward(self, x, z):
            return mvm.group_norm(x, 4, z=z)

    x, z = ins["x"].to(cuda), ins["z"].to(cuda)
    traced = torch.jit.trace(M(), (x, z))
    assert torch.equal(traced(2 * x, z), M()(2 * x, z))


def test_mixer_of_heads(cuda):
    """Conv, gated delta rule and the heads' gated norm as one: packed with gradients, against prompts and steps."""
    T, H, D, lens = 100, 2, 32, [64, 36]
    g = torch.Generator().manual_seed(13)
    r = lambda *s: torch.randn(*s, generator=g).to(cuda)
    x, gate = r(T, 3 * H * D).requires_grad_(True), r(T, H * D).requires_grad_(True)
    w, b = (r(3 * H * D, 4) / 2).requires_grad_(True), (0.1 * r(3 * H * D)).requires_grad_(True)
    decay, beta = (-torch.rand(T, H, generator=g).to(cuda)).requires_grad_(True), torch.sigmoid(r(T, H)).requires_grad_(True)
    nw, off = (1 + 0.1 * r(H * D)).requires_grad_(True), torch.tensor([0, 64, 100], dtype=torch.int32, device=cuda)

    def heads(c):
        return [t.view(-1, H, D) for t in c.split(H * D, dim=1)]

    c, _ = mvm.causal_conv_silu_packed(x, w, b, off)
    o, final = mvm.gated_delta_rule_packed(*heads(c), decay, beta, off, qk_l2norm=True)
    y = mvm.group_norm(o.flatten(1), H, nw, z=gate)
    leaves = [x, gate, w, b, decay, beta, nw]
    up = r(T, H * D)
    grads = torch.autograd.grad(y, leaves, up)
    # each stage's gradient is tested by itself: here, that they are joined as the formulas are, in float64
    from tests import delta_reference
    L = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    conv = []
    for lo, hi in ((0, 64), (64, 100)):
        pad = torch.cat([torch.zeros(3, 3 * H * D, dtype=torch.float64), L[0][lo:hi]])
        conv.append(torch.nn.functional.silu(L[3] + sum(pad[j:j + hi - lo] * L[2][:, j] for j in range(4))))
    q, k, v = [t.reshape(-1, H, D) for t in torch.cat(conv).split(H * D, dim=1)]
    oo, _ = delta_reference.rule([0, 64, 100], q, k, v, L[4], L[5], qk_l2norm=True)
    n = torch.nn.functional.layer_norm(oo, (D,)).flatten(1) * L[6]
    yy = n * torch.nn.functional.silu(L[1])
    want = torch.autograd.grad(yy, L, up.double().cpu())
    # 30 stages of products and sums of at most 192 terms, with the norm's amplification of small rows
    tol = 30 * 4 * 192 ** 0.5 * 2.0 ** -24 * float((1 / oo.detach().std(-1)).max() * oo.detach().abs().max())
    for got, ref_ in zip((y, *grads), (yy.detach(), *want)):
        assert float((got.detach().double().cpu() - ref_).norm() / ref_.norm()) < tol
    # served: a prompt of 60 and 36 tokens, then four steps of the first sequence
    with torch.no_grad():
        cs, ss = torch.zeros(2, 3, 3 * H * D, device=cuda), torch.zeros(2, H, D, D, device=cuda)
        rows = torch.cat([torch.arange(60), torch.arange(64, 100)]).to(cuda)
        c = mvm.causal_conv_silu_prefill(x[rows], w, b, cs, [0, 60, 96])
        o = mvm.gated_delta_rule_prefill(*heads(c), decay[rows], beta[rows], ss, [0, 60, 96], qk_l2norm=True)
        outs = [mvm.group_norm(o.flatten(1), H, nw, z=gate[rows])]
        for t in range(60, 64):
            s = slice(t, t + 1)
            c = mvm.causal_conv_silu_step(x[s], w, b, cs, slots=[0])
            o = mvm.gated_delta_rule_step(*heads(c), decay[s], beta[s], ss, slots=[0], qk_l2norm=True)
            outs.append(mvm.group_norm(o.flatten(1), H, nw, z=gate[s]))
        served = torch.cat([outs[0][:60], *outs[1:], outs[0][60:]])
    assert float((served - y).norm() / y.norm()) < 2 * tol
    assert float((ss - final).norm() / final.norm()) < 2 * tol
