"""LayerNorm and group norm on the GPU (HIP kernels behind include/mvm_norm.h and
include/mvm_group_norm.h).

Replaces the reference's ``nn.LayerNorm(d_model)`` (MLX, eps 1e-5, affine):
the pre-norm of ResidualMambaBlock / BidirectionalMambaBlock /
MultiDirectionalMambaBlock (reference mamba_block.py:201-205, :222-227,
:401, :548) and the encoder's final norm (vision_mamba.py:192, :223).  The
modules keep their ``nn.LayerNorm`` children (same parameters and state_dict
keys); only the computation runs here.

``layer_norm(x, norm, residual=True)`` also returns x itself as a second
output for the block's residual branch ``x + f(norm(x))``.  The gradient
that reaches x through that branch then arrives in this function's backward
together with the normalised branch's, and the backward kernel adds the two
in its store, so no separate accumulation pass runs.

``group_norm`` norms groups of channels, channels last: the heads of a recurrent
mixer, or maps; an activation or a gate is part of the call.
"""

from __future__ import annotations

import torch

from . import _lib


def _norm(x, weight, bias, eps, residual):
    out = _lib.native().norm(x, weight, bias, eps, residual)
    return tuple(out) if residual else out[0]


class _LayerNormFn:
    """The LayerNorm's autograd Function (csrc/torch_ext.cpp)."""

    @staticmethod
    def apply(x, weight, bias, eps, residual):
        if _lib.is_tracing():
            return _lib.traced(_norm, x, weight, bias, eps, residual)
        return _norm(x, weight, bias, eps, residual)


def layer_norm(x, norm, residual=False):
    """``norm(x)`` for an ``nn.LayerNorm`` over the last axis, computed by the
    HIP kernels.  With ``residual=True`` returns ``(norm(x), x_alias)``;
    use ``x_alias`` (it is x) for the block's residual sum so that both
    gradients of x are combined by the norm's backward kernel."""
    if not isinstance(norm, torch.nn.LayerNorm):
        raise TypeError(f"layer_norm needs an nn.LayerNorm, got {type(norm).__name__}")
    if len(norm.normalized_shape) != 1 or not norm.elementwise_affine or norm.bias is None:
        raise ValueError("layer_norm supports an affine LayerNorm over the last axis with bias")
    return _LayerNormFn.apply(x, norm.weight, norm.bias, norm.eps, residual)


def _group_norm(*args):
    return _lib.native().group_norm(*args)


def group_norm(x, groups, weight=None, bias=None, eps=1e-5, *, activation=None, z=None):
    """Group norm with an activation, channels last: act(n) * silu(z).

    x: (N, ..., C), float32 or bfloat16; channel c belongs to group c // (C //
    groups), and a sample's group is normed over its channels and all positions
    between the first and the last dimension: of (T, C) rows, one position each,
    every head by itself; of (B, H, W, C) maps, over the map.

        n = (x - mean) / sqrt(var + eps) * weight + bias      (var biased)

    weight (default ones), bias (zeros): (C,).  activation: None or "silu".  z
    (default none): a gate of x's shape and type.  The last dimension is
    contiguous, rows a stride apart; other layouts are copied.  Returns a
    contiguous tensor of x's shape and type.  Gradients reach x, weight, bias
    and z; second derivatives are refused.
    """
    if activation not in (None, "silu"):
        raise ValueError(f"activation must be None or 'silu'; got {activation!r}")
    args = (x, int(groups), weight, bias, float(eps), activation == "silu", z)
    return _lib.traced(_group_norm, *args) if _lib.is_tracing() else _group_norm(*args)
