"""The packed and served scan and conv on the host: the ABI's validation, the
entry points' refusals, and the float64 oracle of their GPU tests against
torch's autograd and differences.  No kernel is launched."""

import ctypes
import os
import re

import pytest
import torch
import torch.nn.functional as F

import mlx_vision_mamba_amd as mvm
from mlx_vision_mamba_amd import _lib, scan as scan_mod
from tests import seq_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# --------------------------------------------------------------------- ABI

def test_header_and_binding_agree():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "mvm_seq.h")).read(), flags=re.S)
    arity = {n: p.count(",") + 1 for n, p in re.findall(r"\b(mvm_[a-z0-9_]+)\s*\(([^)]*)\)\s*;", text)}
    assert set(arity) == set(_lib.SEQ_SIGNATURES)
    for name, (_, args) in _lib.SEQ_SIGNATURES.items():
        assert len(args) == arity[name], name
        assert hasattr(_lib.lib(), name)


def _scan_desc(T=40, S=3, D=24, N=16):
    d = _lib.SeqScanDesc()
    d.seq.tokens, d.seq.nseq, d.seq.dim, d.seq.state_rows = T, S, D, S
    d.seq.offsets = 1 << 20  # an address: never read on the host
    d.dstate, d.bc_stride = N, N
    d.u_stride = d.delta_stride = d.y_stride = d.z_stride = D
    return d


def _conv_desc(T=40, S=3, D=24, W=4):
    d = _lib.SeqConvDesc()
    d.seq.tokens, d.seq.nseq, d.seq.dim, d.seq.state_rows = T, S, D, S
    d.seq.offsets = 1 << 20
    d.kwidth, d.x_stride, d.y_stride = W, D, D
    return d


BAD_SEQ = [("tokens", -1, _lib.MVM_ERR_INVALID_ARG), ("nseq", -1, _lib.MVM_ERR_INVALID_ARG),
           ("dim", -5, _lib.MVM_ERR_INVALID_ARG), ("seqlen", -1, _lib.MVM_ERR_INVALID_ARG),
           ("state_rows", -1, _lib.MVM_ERR_INVALID_ARG), ("state_rows", 2, _lib.MVM_ERR_INVALID_ARG),
           ("offsets", None, _lib.MVM_ERR_INVALID_ARG), ("tokens", 2 ** 31 - 1, _lib.MVM_ERR_UNSUPPORTED),
           ("nseq", 2 ** 40, _lib.MVM_ERR_UNSUPPORTED)]


@pytest.mark.parametrize("field,value,code", BAD_SEQ + [
    ("dstate", 0, _lib.MVM_ERR_UNSUPPORTED), ("dstate", 17, _lib.MVM_ERR_UNSUPPORTED),
    ("dtype", 2, _lib.MVM_ERR_UNSUPPORTED), ("delta_dtype", 1, _lib.MVM_ERR_UNSUPPORTED),
    ("u_stride", -1, _lib.MVM_ERR_INVALID_ARG), ("bc_stride", -1, _lib.MVM_ERR_INVALID_ARG),
    ("y_stride", 23, _lib.MVM_ERR_INVALID_ARG), ("chunk_len", 8, _lib.MVM_ERR_INVALID_ARG),
    ("chunk_len", 48, _lib.MVM_ERR_INVALID_ARG), ("max_len", -1, _lib.MVM_ERR_INVALID_ARG),
    ("reserved", 1, _lib.MVM_ERR_INVALID_ARG)])
def test_bad_scan_descriptors(field, value, code):
    lib, d = _lib.lib(), _scan_desc()
    assert lib.mvm_seq_scan_validate(ctypes.byref(d)) == 0
    setattr(d if hasattr(d, field) else d.seq, field, value)
    assert lib.mvm_seq_scan_validate(ctypes.byref(d)) == code
    assert _lib.last_error() != ""
    null = [None] * 12
    assert lib.mvm_seq_scan_fwd(ctypes.byref(d), *null, None, 0, None) == code
    assert lib.mvm_seq_scan_workspace_bytes(ctypes.byref(d), 0) == code
    assert lib.mvm_seq_scan_ckpt_elems(ctypes.byref(d)) == code


@pytest.mark.parametrize("field,value,code", BAD_SEQ + [
    ("kwidth", 0, _lib.MVM_ERR_UNSUPPORTED), ("kwidth", 9, _lib.MVM_ERR_UNSUPPORTED),
    ("dtype", -1, _lib.MVM_ERR_UNSUPPORTED), ("x_stride", -1, _lib.MVM_ERR_INVALID_ARG),
    ("y_stride", 23, _lib.MVM_ERR_INVALID_ARG), ("reserved", 1, _lib.MVM_ERR_INVALID_ARG)])
def test_bad_conv_descriptors(field, value, code):
    lib, d = _lib.lib(), _conv_desc()
    assert lib.mvm_seq_conv_validate(ctypes.byref(d)) == 0
    setattr(d if hasattr(d, field) else d.seq, field, value)
    assert lib.mvm_seq_conv_validate(ctypes.byref(d)) == code
    assert lib.mvm_seq_conv_workspace_bytes(ctypes.byref(d)) == code


def test_calls_refused_before_a_launch():
    """NULL operands, a small workspace, steps with offsets, backwards with slots."""
    lib, some = _lib.lib(), ctypes.c_void_p(1 << 20)
    d = _scan_desc()
    ptrs = [some] * 12
    assert lib.mvm_seq_scan_fwd(ctypes.byref(d), *[None] * 12, None, 0, None) == _lib.MVM_ERR_INVALID_ARG
    need = lib.mvm_seq_scan_workspace_bytes(ctypes.byref(d), 0)
    d.chunk_len = 16
    need = lib.mvm_seq_scan_workspace_bytes(ctypes.byref(d), 0)
    assert need > 0
    assert lib.mvm_seq_scan_fwd(ctypes.byref(d), *ptrs, some, need - 1, None) == _lib.MVM_ERR_WORKSPACE
    assert lib.mvm_seq_scan_workspace_bytes(ctypes.byref(d), 2) == _lib.MVM_ERR_INVALID_ARG
    assert lib.mvm_seq_scan_bwd(ctypes.byref(d), *[some] * 20, some, 0, None) == _lib.MVM_ERR_WORKSPACE
    assert lib.mvm_seq_scan_step(ctypes.byref(d), *[some] * 10, None) == _lib.MVM_ERR_INVALID_ARG
    d.seq.slots = 1 << 20
    assert lib.mvm_seq_scan_bwd(ctypes.byref(d), *[some] * 20, some, 1 << 40, None) == _lib.MVM_ERR_INVALID_ARG
    assert "slots" in _lib.last_error()
    c = _conv_desc()
    assert lib.mvm_seq_conv_fwd(ctypes.byref(c), *[None] * 7) == _lib.MVM_ERR_INVALID_ARG
    assert lib.mvm_seq_conv_step(ctypes.byref(c), *[some] * 6) == _lib.MVM_ERR_INVALID_ARG
    assert lib.mvm_seq_conv_bwd(ctypes.byref(c), *[some] * 10, some, 0, None) == _lib.MVM_ERR_WORKSPACE
    c.seq.fresh = 1 << 20
    assert lib.mvm_seq_conv_bwd(ctypes.byref(c), *[some] * 10, some, 1 << 40, None) == _lib.MVM_ERR_INVALID_ARG
    assert lib.mvm_seq_conv_fwd(None, *[None] * 7) == _lib.MVM_ERR_INVALID_ARG


def test_uniform_descriptor_needs_whole_sequences():
    d = _scan_desc(T=40, S=4)
    d.seq.offsets, d.seq.seqlen = None, 10
    assert _lib.lib().mvm_seq_scan_validate(ctypes.byref(d)) == 0
    d.seq.seqlen = 9
    assert _lib.lib().mvm_seq_scan_validate(ctypes.byref(d)) == _lib.MVM_ERR_INVALID_ARG
    d.seq.seqlen = 2 ** 62  # no overflow into the right product
    assert _lib.lib().mvm_seq_scan_validate(ctypes.byref(d)) == _lib.MVM_ERR_INVALID_ARG


def test_grids_that_pass_31_bits_are_refused():
    d = _scan_desc(T=2 ** 31 - 65, D=1 << 20)
    assert _lib.lib().mvm_seq_scan_validate(ctypes.byref(d)) == _lib.MVM_ERR_UNSUPPORTED
    assert "launch" in _lib.last_error()
    c = _conv_desc(T=2 ** 31 - 65, D=1 << 20)
    assert _lib.lib().mvm_seq_conv_validate(ctypes.byref(c)) == _lib.MVM_ERR_UNSUPPORTED


# ------------------------------------------------------------- entry points

def _scan_args(T=6, D=8, N=4, dtype=torch.float32):
    r = lambda *s: torch.randn(*s, dtype=torch.float32).to(dtype)
    return [r(T, D), r(T, D), -torch.rand(D, N), r(T, N), r(T, N), torch.ones(D)]


OFF = torch.tensor([0, 2, 6], dtype=torch.int32)


@pytest.mark.parametrize("offsets", [[1, 6], [0, 4, 3], [0, 7], [], [0.0, 6.0], [[0, 6]]])
def test_offsets_on_the_host_are_checked(offsets):
    with pytest.raises(ValueError):
        mvm.selective_scan_packed(*_scan_args(), offsets)
    with pytest.raises(ValueError):
        mvm.causal_conv_silu_packed(torch.randn(6, 8), torch.randn(8, 4), torch.randn(8), offsets)


def test_slots_on_the_host_are_checked():
    a = _scan_args()
    with pytest.raises(ValueError, match="share a slot"):
        mvm.selective_scan_prefill(*a, torch.zeros(5, 8, 4), OFF, slots=[3, 3])
    with pytest.raises(ValueError, match="share a slot"):
        mvm.causal_conv_silu_step(torch.randn(2, 8), torch.randn(8, 4), None, torch.zeros(5, 3, 8), slots=[1, 1])
    assert scan_mod.sequence_slots([-1, -1, 2], 5, "cpu").tolist() == [-1, -1, 2]  # padding may repeat


@pytest.mark.parametrize("change,error", [
    (lambda a, k: a.__setitem__(0, a[0].double()), "float32 or bfloat16"),
    (lambda a, k: a.__setitem__(0, a[0][None]), "with offsets"),
    (lambda a, k: a.__setitem__(1, a[1][:5]), "u's shape"),
    (lambda a, k: a.__setitem__(1, a[1].bfloat16()), "delta must be"),
    (lambda a, k: a.__setitem__(2, a[2][:7]), "A must be"),
    (lambda a, k: a.__setitem__(2, -torch.rand(8, 17)), "d_state=17"),
    (lambda a, k: a.__setitem__(3, a[3][:, :3]), "B and C"),
    (lambda a, k: a.__setitem__(4, a[4].bfloat16()), "u's type"),
    (lambda a, k: a.__setitem__(5, a[5][:7]), "D and delta_bias"),
    (lambda a, k: k.update(delta_bias=torch.zeros(9)), "D and delta_bias"),
    (lambda a, k: k.update(z=torch.zeros(6, 7)), "u's shape"),
    (lambda a, k: k.update(z=torch.zeros(6, 8).bfloat16()), "u's type"),
    (lambda a, k: k.update(chunk_len=24), "power of two"),
])
def test_packed_scan_refusals(change, error):
    a, k = _scan_args(), {}
    change(a, k)
    with pytest.raises(ValueError, match=error):
        mvm.selective_scan_packed(*a, OFF, **k)


def test_scan_refusals_of_states():
    a = _scan_args()
    with pytest.raises(ValueError, match="without offsets"):
        mvm.selective_scan_packed(*a)
    with pytest.raises(ValueError, match="one token"):
        mvm.selective_scan_step(*[t[None] if i in (0, 1, 3, 4) else t for i, t in enumerate(a)], torch.zeros(6, 8, 4))
    # CPU tensors that are otherwise right: there is no CPU fallback
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mvm.selective_scan_packed(*a, OFF)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mvm.causal_conv_silu_packed(torch.randn(6, 8), torch.randn(8, 4), None, OFF)


def test_conv_refusals():
    x, w = torch.randn(6, 8), torch.randn(8, 4)
    for args in [(x, torch.randn(8, 9), None), (x, torch.randn(7, 4), None), (x, w, torch.randn(7)),
                 (x.double(), w, None), (x[None], w, None)]:
        with pytest.raises(ValueError):
            mvm.causal_conv_silu_packed(*args, OFF)


# ------------------------------------------------------------------- oracle

@pytest.mark.parametrize("gate,soft,a_log", [(True, True, True), (False, False, False)])
def test_scan_oracle_against_autograd_and_differences(gate, soft, a_log):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    off, Dn, N = [0, 0, 3, 4, 9], 3, 2
    T = 10
    leaves = dict(u=r(T, Dn), delta=r(T, Dn) if soft else r(T, Dn).abs(), A=r(Dn, N) if a_log else -r(Dn, N).abs(),
                  B=r(T, N), C=r(T, N), D=r(Dn), z=r(T, Dn) if gate else None, delta_bias=r(Dn), initial=r(4, Dn, N))
    dy, df = r(T, Dn), r(4, Dn, N)

    def forward(lv):
        A = -lv["A"].exp() if a_log else lv["A"]
        d = lv["delta"] + lv["delta_bias"]
        d = F.softplus(d) if soft else d
        ys, hs = [], []
        for i in range(4):
            h = lv["initial"][i]
            for t in range(off[i], off[i + 1]):
                h = (d[t][:, None] * A).exp() * h + (d[t] * lv["u"][t])[:, None] * lv["B"][t]
                y = h @ lv["C"][t] + lv["D"] * lv["u"][t]
                ys.append(y * F.silu(lv["z"][t]) if gate else y)
            hs.append(h)
        return torch.cat([torch.stack(ys), torch.zeros(1, Dn, dtype=torch.float64)]), torch.stack(hs)

    live = {k: v.clone().requires_grad_(True) for k, v in leaves.items() if v is not None}
    y, h = forward({**leaves, **live})
    want = torch.autograd.grad([y, h], list(live.values()), [dy, df])
    out = ref.scan(off, delta_softplus=soft, a_is_log=a_log, dy=dy, dfinal=df, **leaves)
    assert torch.allclose(out["y"].v, y, rtol=1e-12, atol=1e-12)
    assert torch.allclose(out["final"].v, h, rtol=1e-12, atol=1e-12)
    for k, w in zip(live, want):
        assert torch.allclose(out["d" + k].v, w, rtol=1e-10, atol=1e-10), k
    # and one direction by central differences
    move = {k: r(*v.shape) for k, v in live.items()}
    f = lambda s: sum((a * b).sum() for a, b in zip(forward({**leaves, **{k: leaves[k] + s * move[k] for k in move}}), (dy, df)))
    slope = (f(1e-6) - f(-1e-6)) / 2e-6
    assert abs(float(slope - sum((out["d" + k].v * move[k]).sum() for k in move))) < 1e-6 * max(1.0, abs(float(slope)))


@pytest.mark.parametrize("W", [1, 2, 4])
def test_conv_oracle_against_autograd(W):
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    off, Dn = [0, 1, 1, 3, 10], 3
    lv = {k: v.requires_grad_(True) for k, v in
          dict(x=r(10, Dn), weight=r(Dn, W), bias=r(Dn), initial=r(4, W - 1, Dn)).items()}
    ys, cs = [], []
    for i in range(4):
        s = torch.cat([lv["initial"][i], lv["x"][off[i]:off[i + 1]]])
        n = off[i + 1] - off[i]
        if n:
            ys.append(F.silu(F.conv1d(s.t()[None], lv["weight"][:, None], lv["bias"], groups=Dn)[0].t()))
        cs.append(s[n:])
    y, c = torch.cat(ys), torch.stack(cs)
    dy, dc = r(10, Dn), r(4, W - 1, Dn)
    want = torch.autograd.grad([y, c], list(lv.values()), [dy, dc], allow_unused=True)
    out = ref.conv(off, **lv, dy=dy, dfinal=dc)
    assert torch.allclose(out["y"].v, y) and torch.allclose(out["final"].v, c)
    for k, w in zip(lv, want):
        if w is not None:
            assert torch.allclose(out["d" + k].v, w), k


def test_oracle_bound_notices_a_wrong_value():
    """The bounds are tight enough to see one dropped term."""
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g)
    args = dict(u=r(40, 4), delta=0.5 * r(40, 4), A=torch.log(torch.arange(1., 17.)).repeat(4, 1), B=r(40, 16),
                C=r(40, 16), D=torch.ones(4), z=r(40, 4), delta_bias=torch.full((4,), -4.6))
    out = ref.scan([0, 25, 40], delta_softplus=True, a_is_log=True, **args)
    ref.check("y", out["y"].v.float(), out["y"])
    wrong = ref.scan([0, 24, 40], delta_softplus=True, a_is_log=True, **args)
    with pytest.raises(AssertionError):
        ref.check("y", wrong["y"].v.float(), out["y"])


def test_long_rows_are_refused():
    """Rows are walked in steps of 32 bits."""
    lib, d = _lib.lib(), _scan_desc()
    for f in ("u_stride", "delta_stride", "bc_stride", "y_stride", "z_stride"):
        d = _scan_desc()
        setattr(d, f, 2 ** 29)
        assert lib.mvm_seq_scan_validate(ctypes.byref(d)) == _lib.MVM_ERR_UNSUPPORTED, f
        assert f in _lib.last_error()
    c = _conv_desc()
    c.x_stride = 2 ** 29
    assert lib.mvm_seq_conv_validate(ctypes.byref(c)) == _lib.MVM_ERR_UNSUPPORTED


def test_sizes_of_scratch_follow_the_cut():
    """No workspace without chunks; with them aggregates of every chunk slot."""
    lib, d = _lib.lib(), _scan_desc(T=4096, S=2, D=128)
    d.chunk_len = 4096
    assert lib.mvm_seq_scan_workspace_bytes(ctypes.byref(d), 0) == 0
    d.chunk_len = 64
    slots = 4096 // 64 + 3
    assert lib.mvm_seq_scan_workspace_bytes(ctypes.byref(d), 0) == slots * 128 * 17 * 4
    assert lib.mvm_seq_scan_ckpt_elems(ctypes.byref(d)) == (4096 // 8 + 3) * 128 * 16
    d.chunk_len, d.max_len = 0, 0
    for t in (1, 17, 1000, 70000):  # any cut that the library picks is within its own bounds
        d.seq.tokens = t
        for back in (0, 1):
            assert lib.mvm_seq_scan_workspace_bytes(ctypes.byref(d), back) >= 0
