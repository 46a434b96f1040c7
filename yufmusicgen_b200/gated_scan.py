"""Elementwise gated recurrence on the B200 kernels, with its backward pass, a
packed form and a single-token form.  No reference counterpart.

Per channel of ``[B, T, D]``, in fp32 inside whatever the tensors' type::

    a_t = lower + (1 - lower) * sigmoid(forget_t)
    h_t = a_t * h_{t-1} + (1 - a_t) * x_t
    y_t = h_t * sigmoid(gate_t)          # y_t = h_t without a gate

* ``gated_scan(x, forget, gate, lower, state, cu_seqlens)`` -> ``(y, final_state)``,
  differentiable in ``x``, ``forget``, ``gate``, ``lower`` and ``state``, through
  ``y`` and ``final_state`` both.  The backward forms ``h`` again from one saved
  state per 16 tokens.
* ``gated_scan_step(x, forget, state, gate, lower)`` -> ``y``: one token, the
  state updated in place.

``x``, ``forget`` and ``gate`` are float32, bfloat16 or float16 and may be column
ranges of one projection (any batch and token strides).  ``lower`` and ``state``
are float32.  Calls run on the tensors' device and its current stream, and may be
captured in CUDA graphs, their backward passes too (as ever with torch, while no
eager graph of the same leaves is alive).
"""

from __future__ import annotations

from ._torch import ops


def gated_scan(x, forget, gate=None, lower=None, state=None, cu_seqlens=None):
    """Run the gated recurrence over ``x [B, T, D]``; returns ``(y, final_state)``.

    ``gate [B, T, D]``, ``lower [D]`` (retention floor in [0, 1)) and ``state
    [B, D]`` (initial state) are optional.  With ``cu_seqlens`` (int32, on the
    device, non-decreasing, from 0) ``x`` is ``[1, total, D]`` and row range
    ``cu[s] : cu[s + 1]`` is sequence ``s`` with its own state: ``state`` and the
    final state are ``[n_sequences, D]``, an empty sequence keeps its state, and
    rows behind the last sequence play no part; their ``y`` and gradients are 0.
    The contents of ``cu_seqlens`` are not checked (that would wait for the GPU).

    Raises ValueError or TypeError for what the kernels do not take.  The gradients
    cannot be differentiated again (RuntimeError where that is tried), and there are no
    forward-mode derivatives (NotImplementedError for an input with a tangent)."""
    return ops.gated_scan(x, forget, gate, lower, state, cu_seqlens)


def gated_scan_step(x, forget, state, gate=None, lower=None):
    """One token of ``B`` sequences: ``x``, ``forget``, ``gate`` ``[B, D]``; ``state
    [B, D]`` (float32, e.g. a row range of a pool of states) is updated in place; it must
    not share memory with an input, other than x or forget element by element (ValueError).
    Returns ``y [B, D]``.  Not differentiable (NotImplementedError where that is asked for)."""
    return ops.gated_scan_step(x, forget, state, gate, lower)
