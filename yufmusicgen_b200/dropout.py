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

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._cuda import DTYPES, call_on

_M64 = 2**64 - 1


def _row_stride(t):
    """Stride between the rows of ``t`` (its last axis), when they have one."""
    if t.shape[-1] != 1 and t.stride(-1) != 1:
        return None
    row, expect = None, None
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if row is None:
            row = stride
        elif stride != expect:
            return None
        expect = stride * size
    return t.shape[-1] if row is None else row


def _run(x, residual, p, seed, step, out_dtype):
    """The kernel call: x (and residual) of one shape, any strides; ``step`` an int or a tensor."""
    out = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    rows, cols, xs, rs = 1, x.numel(), x.numel(), x.numel()
    if x.ndim and not (x.is_contiguous() and (residual is None or residual.is_contiguous())):
        cols = x.shape[-1]
        rows = x.numel() // cols if cols else 0
        xs, rs = _row_stride(x), cols if residual is None else _row_stride(residual)
        if xs is None:
            x, xs = x.contiguous(), cols
        if rs is None:
            residual, rs = residual.contiguous(), cols
    on_device = isinstance(step, torch.Tensor)
    call_on(x.device, "yuf_dropout", x.data_ptr(), xs, DTYPES[x.dtype], _lib.ptr(residual), rs, out.data_ptr(),
            DTYPES[out_dtype], rows, cols, p, seed, 0 if on_device else step, step.data_ptr() if on_device else None)
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, step):
        ctx.args, ctx.x_dtype = (p, seed, step), x.dtype
        if isinstance(step, torch.Tensor):  # saved, so that a step changed before the backward is an error
            ctx.args = (p, seed, None)
            ctx.save_for_backward(step)
        return _run(x, residual, p, seed, step, x.dtype if residual is None else residual.dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        p, seed, step = ctx.args
        if step is None:
            (step,) = ctx.saved_tensors
        dx = _run(dy, None, p, seed, step, ctx.x_dtype) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x, p, seed, step=0, residual=None):
    """``residual + dropout(x)`` (or ``dropout(x)``): elements dropped with
    probability ``p`` in [0, 1], the others scaled by ``1 / (1 - p)``.  Differentiable.

    ``x`` is float32, bfloat16 or float16, of any shape and strides; ``residual`` has
    its shape and either its type or float32, and gives the result's type.  ``seed``
    and ``step`` are taken modulo 2**64; ``step`` may be an int64 CUDA tensor of one
    element, read when the kernel runs (advance it between replays of a captured
    training step).  It must not change between the forward and the backward."""
    if not x.is_cuda:
        raise ValueError("dropout: x must be on CUDA")
    if x.dtype not in DTYPES:
        raise TypeError(f"dropout: x must be float32, bfloat16 or float16, got {x.dtype}")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout: p must lie in [0, 1], got {p}")
    if residual is not None:
        if residual.shape != x.shape or residual.device != x.device:
            raise ValueError("dropout: residual must have x's shape and device")
        if residual.dtype != x.dtype and residual.dtype != torch.float32:
            raise TypeError("dropout: residual must have x's type or be float32")
    seed = int(seed) & _M64
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or step.numel() != 1 or step.device != x.device:
            raise ValueError("dropout: a step tensor must hold one int64 on x's device")
    else:
        step = int(step) & _M64
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return _Dropout.apply(x, residual, p, seed, step)
    return _run(x, residual, p, seed, step, x.dtype if residual is None else residual.dtype)
