"""The gated delta rule on the host: the ABI's validation, the entry points'
refusals, and the float64 reference of its GPU tests against torch's autograd
and differences.  No kernel is launched."""

import ctypes
import os
import re

import pytest
import torch

import mlx_vision_mamba_amd as mvm
from mlx_vision_mamba_amd import _lib
from tests import delta_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_header_and_binding_agree():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "mvm_delta.h")).read(), flags=re.S)
    arity = {n: p.count(",") + 1 for n, p in re.findall(r"\b(mvm_[a-z0-9_]+)\s*\(([^)]*)\)\s*;", text)}
    assert set(arity) == set(_lib.DELTA_SIGNATURES)
    for name, (_, args) in _lib.DELTA_SIGNATURES.items():
        assert len(args) == arity[name], name
        assert hasattr(_lib.lib(), name)


def _desc(T=40, S=3, HK=2, HV=4, DK=16, DV=24):
    d = _lib.DeltaDesc()
    d.seq.tokens, d.seq.nseq, d.seq.state_rows = T, S, S
    d.seq.offsets = 1 << 20  # an address: never read on the host
    d.key_heads, d.value_heads, d.dk, d.dv = HK, HV, DK, DV
    d.q_stride = d.k_stride = HK * DK
    d.q_stride_head = d.k_stride_head = DK
    d.v_stride, d.v_stride_head = HV * DV, DV
    d.g_stride = d.beta_stride = HV
    d.scale = 0.25
    return d


@pytest.mark.parametrize("field,value,code", [
    ("tokens", -1, _lib.MVM_ERR_INVALID_ARG), ("nseq", -1, _lib.MVM_ERR_INVALID_ARG),
    ("dim", 4, _lib.MVM_ERR_INVALID_ARG), ("seqlen", -1, _lib.MVM_ERR_INVALID_ARG),
    ("state_rows", 2, _lib.MVM_ERR_INVALID_ARG), ("offsets", None, _lib.MVM_ERR_INVALID_ARG),
    ("tokens", 2 ** 31 - 1, _lib.MVM_ERR_UNSUPPORTED), ("nseq", 2 ** 40, _lib.MVM_ERR_UNSUPPORTED),
    ("key_heads", 0, _lib.MVM_ERR_INVALID_ARG), ("value_heads", 0, _lib.MVM_ERR_INVALID_ARG),
    ("value_heads", 3, _lib.MVM_ERR_INVALID_ARG), ("value_heads", 2 ** 40, _lib.MVM_ERR_UNSUPPORTED),
    ("dk", 0, _lib.MVM_ERR_UNSUPPORTED), ("dk", 129, _lib.MVM_ERR_UNSUPPORTED), ("dv", 0, _lib.MVM_ERR_UNSUPPORTED),
    ("dv", 513, _lib.MVM_ERR_UNSUPPORTED), ("dtype", 2, _lib.MVM_ERR_UNSUPPORTED),
    ("beta_dtype", 1, _lib.MVM_ERR_UNSUPPORTED), ("qk_l2norm", 2, _lib.MVM_ERR_INVALID_ARG),
    ("reserved", 1, _lib.MVM_ERR_INVALID_ARG), ("max_len", -1, _lib.MVM_ERR_INVALID_ARG),
    ("split_len", -64, _lib.MVM_ERR_INVALID_ARG), ("split_len", 65, _lib.MVM_ERR_INVALID_ARG),
    ("q_stride", -1, _lib.MVM_ERR_INVALID_ARG), ("v_stride_head", -1, _lib.MVM_ERR_INVALID_ARG),
    ("g_stride", -1, _lib.MVM_ERR_INVALID_ARG), ("k_stride", 2 ** 31, _lib.MVM_ERR_UNSUPPORTED),
    ("v_stride", 2 ** 25 + 1, _lib.MVM_ERR_UNSUPPORTED), ("value_heads", 2 ** 20 + 2, _lib.MVM_ERR_UNSUPPORTED)])
def test_bad_descriptors(field, value, code):
    lib, d = _lib.lib(), _desc()
    assert lib.mvm_delta_validate(ctypes.byref(d)) == 0
    setattr(d if hasattr(d, field) else d.seq, field, value)
    assert lib.mvm_delta_validate(ctypes.byref(d)) == code
    assert _lib.last_error() != ""
    assert lib.mvm_delta_fwd(ctypes.byref(d), *[None] * 10, 0, None) == code
    assert lib.mvm_delta_bwd(ctypes.byref(d), *[None] * 15, 0, None) == code
    assert lib.mvm_delta_step(ctypes.byref(d), *[None] * 8) == code
    assert lib.mvm_delta_workspace_bytes(ctypes.byref(d), 0) == code
    assert lib.mvm_delta_ckpt_elems(ctypes.byref(d)) == code


def test_calls_refused_before_a_launch():
    lib, some, odd, d = _lib.lib(), ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 4), _desc()
    assert lib.mvm_delta_fwd(None, *[some] * 10, 0, None) == _lib.MVM_ERR_INVALID_ARG
    assert lib.mvm_delta_fwd(ctypes.byref(d), *[None] * 10, 0, None) == _lib.MVM_ERR_INVALID_ARG
    need = [lib.mvm_delta_workspace_bytes(ctypes.byref(d), w) for w in (0, 1)]
    assert min(need) > 0
    assert lib.mvm_delta_workspace_bytes(ctypes.byref(d), 2) == _lib.MVM_ERR_INVALID_ARG
    assert lib.mvm_delta_fwd(ctypes.byref(d), *[some] * 10, need[0] - 1, None) == _lib.MVM_ERR_WORKSPACE
    assert lib.mvm_delta_fwd(ctypes.byref(d), *[some] * 9, odd, need[0], None) == _lib.MVM_ERR_WORKSPACE
    assert lib.mvm_delta_fwd(ctypes.byref(d), *[some] * 8, odd, some, need[0], None) == _lib.MVM_ERR_INVALID_ARG
    assert lib.mvm_delta_bwd(ctypes.byref(d), *[some] * 15, need[1] - 1, None) == _lib.MVM_ERR_WORKSPACE
    assert lib.mvm_delta_step(ctypes.byref(d), *[some] * 8) == _lib.MVM_ERR_INVALID_ARG  # offsets
    d.seq.slots = 1 << 20
    assert lib.mvm_delta_bwd(ctypes.byref(d), *[some] * 15, need[1], None) == _lib.MVM_ERR_INVALID_ARG
    assert "slots" in _lib.last_error()
    big = _desc(T=2 ** 31 - 65, HV=1 << 16, DV=512)
    assert lib.mvm_delta_validate(ctypes.byref(big)) == _lib.MVM_ERR_UNSUPPORTED
    assert "launch" in _lib.last_error()


def _ops(T=6, HK=2, HV=4, DK=8, DV=5, dtype=torch.float32):
    return [torch.zeros(T, HK, DK, dtype=dtype), torch.zeros(T, HK, DK, dtype=dtype),
            torch.zeros(T, HV, DV, dtype=dtype), torch.zeros(T, HV), torch.zeros(T, HV)]


@pytest.mark.parametrize("at,bad,word", [
    (0, torch.zeros(6, 2, 8, dtype=torch.float16), "float32 or bfloat16"), (0, torch.zeros(6, 16), "q must be"),
    (1, torch.zeros(6, 1, 8), "k must have"), (1, torch.zeros(6, 2, 8).bfloat16(), "type"),
    (2, torch.zeros(6, 3, 5), "multiple"), (2, torch.zeros(5, 4, 5), "v must be"),
    (2, torch.zeros(6, 4, 513), "head sizes"), (2, torch.zeros(6, 4, 0), "head sizes"),
    (3, torch.zeros(6, 2), "g and beta"), (4, torch.zeros(6, 4, 1), "g and beta"),
    (4, torch.zeros(6, 4).bfloat16(), "beta"), (3, torch.zeros(6, 4, dtype=torch.int32), "g must be floating")])
def test_operands_refused(at, bad, word):
    args = _ops()
    args[at] = bad
    with pytest.raises(ValueError, match=word):
        mvm.gated_delta_rule_packed(*args, [0, 6])
    with pytest.raises(ValueError, match=word):
        mvm.gated_delta_rule_step(*args, torch.zeros(6, 4, 8, 5))


def test_other_refusals():
    args = _ops()
    for off, word in (([0, 7], "end at 6"), ([1, 6], "start at 0"), ([0, 4, 2], "not decrease"), ([0.0, 6.0], "whole")):
        with pytest.raises(ValueError, match=word):
            mvm.gated_delta_rule_packed(*args, off)
    with pytest.raises(ValueError, match="split_len"):
        mvm.gated_delta_rule_packed(*args, [0, 6], split_len=32)
    with pytest.raises(ValueError, match="without offsets"):
        mvm.gated_delta_rule_packed(*args)
    with pytest.raises(ValueError, match="share a slot"):
        mvm.gated_delta_rule_step(*args, torch.zeros(9, 4, 8, 5), slots=[0, 1, 2, 3, 4, 4])
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mvm.gated_delta_rule_packed(*args, [0, 6])


def _random(off, HK, HV, DK, DV, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    T, S = off[-1], len(off) - 1
    return dict(q=r(T, HK, DK), k=r(T, HK, DK), v=r(T, HV, DV), g=-torch.rand(T, HV, generator=g, dtype=torch.float64),
                beta=torch.sigmoid(r(T, HV)), initial=r(S, HV, DK, DV)), r(T, HV, DV), r(S, HV, DK, DV)


@pytest.mark.parametrize("l2", [False, True])
def test_reference_is_the_rule(l2):
    """Its outputs and adjoint against torch's autograd and differences of the recurrence."""
    off = [0, 3, 3, 8]
    ins, do, df = _random(off, 2, 4, 4, 3)
    if not l2:
        ins["k"] = ins["k"] / 4
    leaves = {n: x.requires_grad_(True) for n, x in ins.items()}
    o, final = ref.rule(off, **leaves, qk_l2norm=l2)
    grads = torch.autograd.grad([o, final], list(leaves.values()), [do, df])
    got, _ = ref.reference(off, **leaves, qk_l2norm=l2, do=do, dfinal=df)
    for n, x in {"o": o, "final": final, **{"d" + n: g for n, g in zip(leaves, grads)}}.items():
        assert torch.allclose(got[n][0], x.detach(), rtol=1e-10, atol=1e-12), n
        assert bool((got[n][1] >= 0).all()) and float(got[n][1].norm()) >= 0.3 * float(x.detach().norm()), n
    names = list(leaves)

    def loss(*xs):
        o, final = ref.rule(off, **dict(zip(names, xs)), qk_l2norm=l2)
        return (o * do).sum() + (final * df).sum()

    assert torch.autograd.gradcheck(loss, list(leaves.values()), eps=1e-6, atol=1e-6)


def test_check_sees_mistakes():
    """The comparison refuses an output with one wrong value, one wrong row, a lost low part."""
    off = [0, 70]
    ins, do, df = _random(off, 1, 1, 16, 16, 3)
    ins["k"] = ins["k"] / 8
    got, factor = ref.reference(off, **ins, do=do, dfinal=df)
    for n, (x, mag) in got.items():
        ref.check(n, x.float(), got[n], factor)
        for wrong in (x.flatten()[x.numel() // 2:x.numel() // 2 + 1], x[-1:]):
            y = x.clone()
            y.view(-1)[x.numel() // 2 if wrong.numel() == 1 else slice(-x[-1].numel(), None)] *= -1
            if float((y - x).norm()) > 1e-3 * float(mag.norm()):
                with pytest.raises(AssertionError):
                    ref.check(n, y.float(), got[n], factor)
