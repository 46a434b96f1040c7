"""Launch helper of the operators whose tensors may be fp32, bf16 or fp16."""

from __future__ import annotations

import torch

from . import _lib

# torch dtype -> YUF_DTYPE_*
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def call_on(device, name, *args):
    """``_lib.call`` with the device's current stream as the last argument, on that device."""
    index = device.index
    if index == torch.cuda.current_device():
        _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args, torch._C._cuda_getCurrentRawStream(index))


def unit_rows(t):
    """``t`` with a unit stride along its last axis (a copy where it has none)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()
