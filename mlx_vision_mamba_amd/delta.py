"""The gated delta rule on packed and served sequences, on the GPU.

A recurrence with a matrix state beside the selective scan's diagonal one (the
reference has only the scan, mamba_block.py:20-74): every head keeps a map from
keys to values, decays it, and replaces what it holds under the new key.

``gated_delta_rule_packed`` trains on packed sequences that start from states
and leave them; ``gated_delta_rule_prefill`` and ``gated_delta_rule_step``
advance a cache by prompts and by single tokens.
"""

from __future__ import annotations

import torch

from . import _lib
from .scan import _no_trace, sequence_offsets, sequence_slots


def _packed(*args):
    return _lib.native().delta(*args)


def _offsets(offsets, q):
    if offsets is None or (isinstance(offsets, torch.Tensor) and offsets.is_cuda):
        return offsets
    # (looked at as the scan's rows are: (T, columns) with offsets)
    return sequence_offsets(offsets, q[:, 0] if q.dim() == 3 and q.shape[1] else q)


def _split(split_len):
    split_len = int(split_len)
    if split_len < 0 or split_len % 64:
        raise ValueError(f"split_len must be 0 or a multiple of 64; got {split_len}")
    return min(split_len, 2 ** 31 - 64)  # (of 32 bits beyond this; no sequence is longer)


def gated_delta_rule_packed(q, k, v, g, beta, offsets=None, *, scale=None, qk_l2norm=False, initial_states=None,
                            max_len=None, split_len=0):
    """Gated delta rule of packed sequences that start from states: (o, final_states).

    q, k: (T, H_k, D_k), v: (T, H_v, D_v), g, beta: (T, H_v), the rows of all
    sequences one after the other, cut by ``offsets`` as in
    ``selective_scan_packed``; without offsets (B, L, ...), one sequence a batch
    row.  H_v is a multiple of H_k: value head h reads key head h // (H_v / H_k).
    D_k 1..128, D_v 1..512.  q, k, v, o share a type, float32 or bfloat16, and
    may have any strides (v's rows up to 2^25 values apart) but a contiguous last
    dimension; beta has it too or is float32; g is taken in float32, and as at
    least -10000.

        S = exp(g_t) S;  d = beta_t (v_t - S^T k_t);  S = S + k_t d^T;  o_t = scale S^T q_t

    ``scale``: default D_k ** -0.5.  ``qk_l2norm``: q and k are first divided by
    sqrt(sum of squares + 1e-6).  initial_states (default zero) and
    final_states: (S, H_v, D_k, D_v), float32.  Gradients reach every argument,
    final_states' gradient included (g's is zero below -10000); second derivatives
    are refused.  A call with gradients keeps, a token and value head, 2.1 KiB for
    128 x 128 heads (the chunks' states) until its backward, which takes 1.5 to 1.8 more.
    ``max_len``: an upper bound of the lengths where the caller knows one; only
    the split over the time axis goes by it.  ``split_len``: 0, or a multiple of
    64 to set that split.  Values must be finite: one that is not makes its
    sequence's outputs and gradients meaningless, also up to 63 rows before it.
    """
    args = (q, k, v, g, beta, initial_states, _offsets(offsets, q), scale, bool(qk_l2norm), int(max_len or 0),
            _split(split_len))
    return tuple(_lib.traced(_packed, *args) if _lib.is_tracing() else _packed(*args))


def gated_delta_rule_prefill(q, k, v, g, beta, states, offsets=None, *, slots=None, fresh=None, scale=None,
                             qk_l2norm=False, max_len=None, split_len=0):
    """``gated_delta_rule_packed`` on a cache: returns o, no gradients.

    ``states``: (rows, H_v, D_k, D_v) float32, contiguous, advanced in place;
    ``slots`` and ``fresh`` as in ``selective_scan_prefill``."""
    _no_trace("gated_delta_rule_prefill")
    return _lib.native().delta_prefill(
        q, k, v, g, beta, states, _offsets(offsets, q), sequence_slots(slots, states.shape[0], q.device), fresh,
        scale, bool(qk_l2norm), int(max_len or 0), _split(split_len))


def gated_delta_rule_step(q, k, v, g, beta, states, *, slots=None, scale=None, qk_l2norm=False):
    """One token for each of S sequences: o (S, H_v, D_v), ``states`` advanced in
    place; a row whose slot lies outside the cache is padding: its o is zero."""
    _no_trace("gated_delta_rule_step")
    return _lib.native().delta_step(q, k, v, g, beta, states, sequence_slots(slots, states.shape[0], q.device),
                                    scale, bool(qk_l2norm))
