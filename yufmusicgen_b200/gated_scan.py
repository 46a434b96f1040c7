"""Elementwise gated recurrence on the B200 kernels, with its backward pass, a
packed form and a single-token form.  No reference counterpart.

Per channel of ``[B, T, D]``, in fp32 inside whatever the tensors' type::

    a_t = lower + (1 - lower) * sigmoid(forget_t)
    h_t = a_t * h_{t-1} + (1 - a_t) * x_t
    y_t = h_t * sigmoid(gate_t)          # y_t = h_t without a gate

* ``gated_scan(x, forget, gate, lower, state, cu_seqlens)`` -> ``(y, final_state)``,
  differentiable in ``x``, ``forget``, ``gate``, ``lower`` and ``state``, through
  ``y`` and ``final_state`` both.  The backward forms ``h`` again from one saved
  state per 16 tokens (8 for fp32).
* ``gated_scan_step(x, forget, state, gate, lower)`` -> ``y``: one token, the
  state updated in place.

``x``, ``forget`` and ``gate`` are float32, bfloat16 or float16 and may be column
ranges of one projection (any batch and token strides).  ``lower`` and ``state``
are float32.
"""

from __future__ import annotations

import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._cuda import DTYPES, call_on, unit_rows

_Strides6 = ctypes.c_int64 * 6
_Strides8 = ctypes.c_int64 * 8
_Strides3 = ctypes.c_int64 * 3


def _check_tensors(x, forget, gate, lower, ndim):
    dtype, shape, device = x.dtype, x.shape, x.device
    if x.ndim != ndim:
        raise ValueError(f"gated scan: x must have shape {'[B, T, D]' if ndim == 3 else '[B, D]'}, got {tuple(shape)}")
    if not x.is_cuda:
        raise ValueError("gated scan inputs must be on CUDA")
    if dtype not in DTYPES:
        raise TypeError(f"gated scan: x must be float32, bfloat16 or float16, got {dtype}")
    for name, t in (("forget", forget), ("gate", gate)):
        if t is None and name == "gate":
            continue
        if t.shape != shape or t.dtype != dtype or t.device != device:
            raise ValueError(f"gated scan: {name} must have x's shape, type and device")
    if shape[-1] < 1:
        raise ValueError("gated scan: D must be at least 1")
    if lower is not None:
        if lower.dtype != torch.float32:
            raise TypeError("gated scan: lower must be float32")
        if lower.shape != shape[-1:] or lower.device != device:
            raise ValueError("gated scan: lower must be a [D] tensor on x's device")


def _check(x, forget, gate, lower, state, cu_seqlens):
    _check_tensors(x, forget, gate, lower, 3)
    rows = x.shape[0]
    if cu_seqlens is not None:
        if rows != 1:
            raise ValueError("gated scan: packed sequences need x of shape [1, total, D]")
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.ndim != 1 or cu_seqlens.numel() < 1:
            raise ValueError("gated scan: cu_seqlens must be an int32 [n_sequences + 1] tensor")
        if cu_seqlens.device != x.device or not cu_seqlens.is_contiguous():
            raise ValueError("gated scan: cu_seqlens must be contiguous and on x's device")
        rows = cu_seqlens.numel() - 1
    if state is not None:
        if state.dtype != torch.float32:
            raise TypeError("gated scan: state must be float32")
        if state.shape != (rows, x.shape[2]) or state.device != x.device:
            raise ValueError(f"gated scan: state must be a [{rows}, {x.shape[2]}] tensor on x's device")
    return rows


def _workspace(x, dtype, backward):
    """Device scratch of one call, or None where it needs none."""
    n = _lib.load().yuf_gated_scan_workspace_bytes(*x.shape, dtype, backward)
    return torch.empty(n, dtype=torch.uint8, device=x.device) if n else None


def _forward(x, forget, gate, lower, state, cu, rows, save):
    """The kernel call on checked tensors with unit rows; ``(y, final_state, checkpoints)``."""
    B, T, D = x.shape
    dtype = DTYPES[x.dtype]
    y = torch.empty((B, T, D), dtype=x.dtype, device=x.device)
    last = torch.empty((rows, D), dtype=torch.float32, device=x.device)
    ckpt = None
    if save:
        block = _lib.load().yuf_gated_scan_block(dtype)
        ckpt = torch.empty((B, (T + block - 1) // block, D), dtype=torch.float32, device=x.device)
    work = _workspace(x, dtype, 0)
    strides = _Strides6(x.stride(0), x.stride(1), forget.stride(0), forget.stride(1),
                        *((0, 0) if gate is None else (gate.stride(0), gate.stride(1))))
    call_on(x.device, "yuf_gated_scan_forward", x.data_ptr(), forget.data_ptr(), _lib.ptr(gate), strides,
            _lib.ptr(lower), _lib.ptr(state), _lib.ptr(cu), 0 if cu is None else rows, y.data_ptr(), last.data_ptr(),
            _lib.ptr(ckpt), _lib.ptr(work), dtype, B, T, D)
    return y, last, ckpt


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, forget, gate, lower, state, cu, rows):
        y, last, ckpt = _forward(x, forget, gate, lower, state, cu, rows, True)
        ctx.save_for_backward(x, forget, gate, lower, state, cu, ckpt)
        ctx.rows = rows
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, forget, gate, lower, state, cu, ckpt = ctx.saved_tensors
        B, T, D = x.shape
        dtype = DTYPES[x.dtype]
        dy = torch.zeros((B, T, D), dtype=x.dtype, device=x.device) if dy is None else unit_rows(dy)
        dlast = None if dlast is None else dlast.contiguous()
        dx, df, dg = (None if t is None else torch.empty((B, T, D), dtype=x.dtype, device=x.device)
                      for t in (x, forget, gate))
        dlower = dstate = None
        if lower is not None and ctx.needs_input_grad[3]:
            dlower = torch.empty_like(lower)
        work = _workspace(x, dtype, 1)
        if state is not None and ctx.needs_input_grad[4]:
            dstate = torch.empty((ctx.rows, D), device=x.device)
        strides = _Strides8(x.stride(0), x.stride(1), forget.stride(0), forget.stride(1),
                            *((0, 0) if gate is None else (gate.stride(0), gate.stride(1))),
                            dy.stride(0), dy.stride(1))
        call_on(x.device, "yuf_gated_scan_backward", x.data_ptr(), forget.data_ptr(), _lib.ptr(gate), dy.data_ptr(),
                strides, _lib.ptr(lower), _lib.ptr(state), _lib.ptr(cu), 0 if cu is None else ctx.rows,
                ckpt.data_ptr(), _lib.ptr(dlast), dx.data_ptr(), df.data_ptr(), _lib.ptr(dg), _lib.ptr(dlower),
                _lib.ptr(dstate), _lib.ptr(work), dtype, B, T, D)
        return dx, df, dg, dlower, dstate, None, None


def gated_scan(x, forget, gate=None, lower=None, state=None, cu_seqlens=None):
    """Run the gated recurrence over ``x [B, T, D]``; returns ``(y, final_state)``.

    ``gate [B, T, D]``, ``lower [D]`` (retention floor in [0, 1)) and ``state
    [B, D]`` (initial state) are optional.  With ``cu_seqlens`` (int32, on the
    device, non-decreasing, from 0) ``x`` is ``[1, total, D]`` and row range
    ``cu[s] : cu[s + 1]`` is sequence ``s`` with its own state: ``state`` and the
    final state are ``[n_sequences, D]``, an empty sequence keeps its state, and
    rows behind the last sequence are not read; their ``y`` and gradients are 0.
    The contents of ``cu_seqlens`` are not checked (that would wait for the GPU)."""
    rows = _check(x, forget, gate, lower, state, cu_seqlens)
    x, forget = unit_rows(x), unit_rows(forget)
    gate = None if gate is None else unit_rows(gate)
    lower = None if lower is None else lower.contiguous()
    state = None if state is None else state.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, forget, gate, lower, state)):
        return _GatedScan.apply(x, forget, gate, lower, state, cu_seqlens, rows)
    return _forward(x, forget, gate, lower, state, cu_seqlens, rows, False)[:2]


def gated_scan_step(x, forget, state, gate=None, lower=None):
    """One token of ``B`` sequences: ``x``, ``forget``, ``gate`` ``[B, D]``; ``state
    [B, D]`` (float32, e.g. a row range of a pool of states) is updated in place.
    Returns ``y [B, D]``.  Not differentiable."""
    _check_tensors(x, forget, gate, lower, 2)
    B, D = x.shape
    if state.dtype != torch.float32:
        raise TypeError("gated scan: state must be float32")
    if state.shape != x.shape or state.device != x.device:
        raise ValueError("gated scan: state must be a [B, D] tensor on x's device")
    stride = state.stride(0)
    if (D > 1 and state.stride(1) != 1) or (B > 1 and stride < D):
        raise ValueError("gated scan: state rows must be contiguous and must not overlap")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, forget, gate, lower, state)):
        raise NotImplementedError("gated_scan_step has no gradients: use gated_scan, or torch.no_grad()")
    x, forget = unit_rows(x), unit_rows(forget)
    gate = None if gate is None else unit_rows(gate)
    lower = None if lower is None else lower.contiguous()
    y = torch.empty((B, D), dtype=x.dtype, device=x.device)
    strides = _Strides3(x.stride(0), forget.stride(0), 0 if gate is None else gate.stride(0))
    call_on(x.device, "yuf_gated_scan_step", x.data_ptr(), forget.data_ptr(), _lib.ptr(gate), strides, _lib.ptr(lower),
            state.data_ptr(), stride, y.data_ptr(), DTYPES[x.dtype], B, D)
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)
    return y
