"""The group norm on the host: the ABI's validation, the entry point's
refusals, and the float64 reference of its GPU tests against torch's autograd
and differences.  No kernel is launched."""

import ctypes
import os
import re

import pytest
import torch

import mlx_vision_mamba_amd as mvm
from mlx_vision_mamba_amd import _lib
from tests import group_norm_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_header_and_binding_agree():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "mvm_group_norm.h")).read(), flags=re.S)
    arity = {n: p.count(",") + 1 for n, p in re.findall(r"\b(mvm_[a-z0-9_]+)\s*\(([^)]*)\)\s*;", text)}
    assert set(arity) == set(_lib.GROUP_NORM_SIGNATURES)
    for name, (_, args) in _lib.GROUP_NORM_SIGNATURES.items():
        assert len(args) == arity[name], name
        assert hasattr(_lib.lib(), name)


def _desc(N=4, P=9, C=24, G=4):
    d = _lib.GroupNormDesc()
    d.batch, d.positions, d.channels, d.groups, d.x_stride, d.eps = N, P, C, G, C, 1e-5
    return d


@pytest.mark.parametrize("field,value,code", [
    ("batch", -1, _lib.MVM_ERR_INVALID_ARG), ("positions", -1, _lib.MVM_ERR_INVALID_ARG),
    ("channels", 0, _lib.MVM_ERR_UNSUPPORTED), ("channels", 65540, _lib.MVM_ERR_UNSUPPORTED),
    ("groups", 0, _lib.MVM_ERR_INVALID_ARG), ("groups", 5, _lib.MVM_ERR_INVALID_ARG),
    ("groups", 48, _lib.MVM_ERR_INVALID_ARG), ("x_stride", -1, _lib.MVM_ERR_INVALID_ARG),
    ("z_stride", -1, _lib.MVM_ERR_INVALID_ARG), ("eps", -1.0, _lib.MVM_ERR_INVALID_ARG),
    ("eps", float("nan"), _lib.MVM_ERR_INVALID_ARG), ("dtype", 2, _lib.MVM_ERR_UNSUPPORTED),
    ("silu", 2, _lib.MVM_ERR_INVALID_ARG), ("reserved", 1, _lib.MVM_ERR_INVALID_ARG),
    ("batch", 2 ** 40, _lib.MVM_ERR_UNSUPPORTED), ("batch", 2 ** 27, _lib.MVM_ERR_UNSUPPORTED)])
def test_bad_descriptors(field, value, code):
    lib, d = _lib.lib(), _desc()
    assert lib.mvm_group_norm_validate(ctypes.byref(d)) == 0
    setattr(d, field, value)
    assert lib.mvm_group_norm_validate(ctypes.byref(d)) == code
    assert _lib.last_error() != ""
    assert lib.mvm_group_norm_fwd(ctypes.byref(d), *[None] * 7, 0, None) == code
    assert lib.mvm_group_norm_bwd(ctypes.byref(d), *[None] * 11, 0, None) == code
    assert lib.mvm_group_norm_workspace_bytes(ctypes.byref(d), 0) == code


def test_calls_refused_before_a_launch():
    lib, some, odd, d = _lib.lib(), ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + 4), _desc()
    assert lib.mvm_group_norm_fwd(None, *[some] * 7, 0, None) == _lib.MVM_ERR_INVALID_ARG
    assert lib.mvm_group_norm_fwd(ctypes.byref(d), *[None] * 7, 0, None) == _lib.MVM_ERR_INVALID_ARG
    need = [lib.mvm_group_norm_workspace_bytes(ctypes.byref(d), w) for w in (0, 1)]
    assert min(need) > 0 and lib.mvm_group_norm_workspace_bytes(ctypes.byref(d), 2) == _lib.MVM_ERR_INVALID_ARG
    assert lib.mvm_group_norm_fwd(ctypes.byref(d), *[some] * 7, need[0] - 1, None) == _lib.MVM_ERR_WORKSPACE
    assert lib.mvm_group_norm_fwd(ctypes.byref(d), *[some] * 6, odd, need[0], None) == _lib.MVM_ERR_WORKSPACE
    assert lib.mvm_group_norm_bwd(ctypes.byref(d), *[some] * 11, need[1] - 1, None) == _lib.MVM_ERR_WORKSPACE
    # a gate without room for its gradient
    assert lib.mvm_group_norm_bwd(ctypes.byref(d), *[some] * 9, None, some, need[1], None) == _lib.MVM_ERR_INVALID_ARG


@pytest.mark.parametrize("x,kw,word", [
    (torch.zeros(4, 24, dtype=torch.float16), {}, "float32 or bfloat16"), (torch.zeros(24), {}, "x must be"),
    (torch.zeros(4, 22), {}, "must divide"), (torch.zeros(4, 0), {}, "must divide"),
    (torch.zeros(4, 24), dict(weight=torch.ones(4)), "weight and bias"),
    (torch.zeros(4, 24), dict(bias=torch.ones(24, 1)), "weight and bias"),
    (torch.zeros(4, 24), dict(z=torch.ones(4, 4)), "z must have"),
    (torch.zeros(4, 24), dict(z=torch.ones(4, 24).bfloat16()), "z must have"),
    (torch.zeros(4, 24), dict(eps=-1.0), "eps"), (torch.zeros(4, 24), dict(activation="relu"), "activation")])
def test_operands_refused(x, kw, word):
    with pytest.raises(ValueError, match=word):
        mvm.group_norm(x, 4, **kw)


def test_no_cpu_fallback():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        mvm.group_norm(torch.zeros(4, 24), 4)


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("gate", [False, True])
def test_reference_is_the_norm(silu, gate):
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    ins = {"x": r(3, 5, 12), "weight": r(12), "bias": r(12)}
    if gate:
        ins["z"] = r(3, 5, 12)
    leaves = {n: t.requires_grad_(True) for n, t in ins.items()}
    dy = r(3, 5, 12)

    def call(x, weight, bias, z=None):
        n = torch.nn.functional.group_norm(x.movedim(-1, 1), 4, weight, bias, 1e-5).movedim(1, -1)
        n = torch.nn.functional.silu(n) if silu else n
        return n if z is None else n * torch.nn.functional.silu(z)

    y = call(*leaves.values())
    grads = torch.autograd.grad(y, list(leaves.values()), dy)
    got = ref.group_norm(groups=4, silu=silu, dy=dy, **leaves)
    for n, t in {"y": y, **{"d" + n: t for n, t in zip(leaves, grads)}}.items():
        assert torch.allclose(got[n].v, t.detach(), rtol=1e-7, atol=1e-9), n
    assert torch.autograd.gradcheck(call, list(leaves.values()))
