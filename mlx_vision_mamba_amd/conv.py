"""Causal depthwise conv1d + SiLU along scan orders, on the GPU.

Replaces MambaBlock's ``conv1d`` + ``[:, :L]`` + ``silu``
(reference mamba_block.py:129-132, :170-171) for all K directions of a
block at once: x is (B, N, K, D) in token order and position s of direction
k reads token row ``seq_to_tok[k, s]``, so no permuted copy is built.

``causal_conv_silu_packed``, ``causal_conv_silu_prefill`` and
``causal_conv_silu_step`` are the forms that start from the inputs before a
sequence and leave its last ones (the reference pads with zeros): packed
sequences, a serving loop's prompts and its single tokens.
"""

from __future__ import annotations

import torch

from . import _lib
from .scan import _no_trace, sequence_offsets, sequence_slots


def _conv_silu(x, weight, bias, tok):
    return _lib.native().conv_silu(x, weight, bias, tok)


def causal_conv_silu(x, weight, bias, seq_to_tok=None):
    """silu(causal depthwise conv) per direction.

    x: (B, N, K, D) float32 (channel stride 1, any other strides);
    weight: (K, D, d_conv); bias: (K, D); seq_to_tok: (K, N) int32 GPU
    tensor or None (identity order).  Returns (B, N, K, D) contiguous.
    """
    if weight.dim() != 3 or weight.shape[:2] != (x.shape[2], x.shape[3]):
        raise ValueError(f"weight must be (K, D, d_conv); got {tuple(weight.shape)}")
    if bias.shape != (x.shape[2], x.shape[3]):
        raise ValueError(f"bias must be (K, D); got {tuple(bias.shape)}")
    if seq_to_tok is not None:
        if seq_to_tok.dtype != torch.int32 or seq_to_tok.shape != (x.shape[2], x.shape[1]):
            raise ValueError("seq_to_tok must be int32 of shape (K, N)")
        seq_to_tok = seq_to_tok.to(x.device).contiguous()
    if _lib.is_tracing():
        return _lib.traced(_conv_silu, x, weight, bias, seq_to_tok)
    return _conv_silu(x, weight, bias, seq_to_tok)


def _packed(*args):
    return _lib.native().seq_conv(*args)


def causal_conv_silu_packed(x, weight, bias, offsets=None, *, initial_states=None):
    """silu(causal depthwise conv) of packed sequences: (y, final_states).

    x: (T, D) rows with ``offsets`` (S + 1, see ``scan.sequence_offsets``), or
    (B, L, D) without; float32 or bfloat16, any row stride.  weight: (D, d_conv)
    with d_conv 1..8; bias: (D,) or None.  initial_states (default zero) and
    final_states: (S, d_conv - 1, D) of x's type, the inputs before a sequence's
    first token and its last inputs, oldest first.  Gradients reach every
    argument; second derivatives are refused.
    """
    args = (x, weight, bias, initial_states, sequence_offsets(offsets, x))
    return tuple(_lib.traced(_packed, *args) if _lib.is_tracing() else _packed(*args))


def causal_conv_silu_prefill(x, weight, bias, states, offsets=None, *, slots=None, fresh=None):
    """``causal_conv_silu_packed`` on a cache: returns y, no gradients.
    ``states``: (rows, d_conv - 1, D) of x's type, contiguous, advanced in
    place; ``slots`` and ``fresh`` as in ``scan.selective_scan_prefill``."""
    _no_trace("causal_conv_silu_prefill")
    return _lib.native().seq_conv_prefill(x, weight, bias, states, sequence_offsets(offsets, x),
                                          sequence_slots(slots, states.shape[0], x.device), fresh)


def causal_conv_silu_step(x, weight, bias, states, *, slots=None):
    """One token for each of S sequences: y (S, D), ``states`` advanced in
    place; a row whose slot lies outside the cache is padding: its y is zero."""
    _no_trace("causal_conv_silu_step")
    return _lib.native().seq_conv_step(x, weight, bias, states, sequence_slots(slots, states.shape[0], x.device))
