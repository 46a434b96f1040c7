"""Dropout with an optional residual add on the B200 kernels; the mask is drawn
from a counter-based generator, in the backward pass again, and never stored.
No reference counterpart.

``dropout(x, p, seed, step, residual)``::

    y_i = residual_i + (w_i >= floor(p * 2**32) ? x_i / (1 - p) : 0)

with ``w_i`` word ``i % 4`` of Philox4x32-10(key = seed, counter = (i / 4, step)),
``i`` the element's row-major index.  Calls that are to draw different masks need
different ``(seed, step)`` pairs: e.g. a seed per layer and a step per training step.
"""

from __future__ import annotations

from ._torch import ops


def dropout(x, p, seed, step=0, residual=None):
    """``residual + dropout(x)`` (or ``dropout(x)``): elements dropped with
    probability ``p`` in [0, 1], the others scaled by ``1 / (1 - p)``.  Differentiable.

    ``x`` is float32, bfloat16 or float16, of any shape and strides; ``residual`` has
    its shape and either its type or float32, and gives the result's type.  ``seed``
    and ``step`` are taken modulo 2**64; ``step`` may be an int64 CUDA tensor of one
    element, read when the kernel runs (advance it between replays of a captured
    training step).  It must not change between the forward and the backward.

    Raises ValueError or TypeError for what the kernels do not take, NotImplementedError for
    an input with a forward-mode tangent."""
    return ops.dropout(x, p, seed, step, residual)
