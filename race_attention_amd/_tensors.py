"""What the calls of the operators around the attention share: argument checks,
rows, pointers and streams."""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib
from .functional import _require_gpu as require_gpu  # noqa: F401  (one check and message)

DTYPES = {torch.bfloat16: _lib.RACE_DTYPE_BF16, torch.float32: _lib.RACE_DTYPE_F32}
_SAME = contextlib.nullcontext()


def native(x, name, *args):
    """The C++ call of that name (csrc/layers_torch.cpp) with these arguments, or None where it does
    not take them: the Python path makes the call then, or raises."""
    if not (torch.is_tensor(x) and x.is_cuda):
        return None
    mod = _lib.calls()
    return None if mod is None else getattr(mod, name)(*args)


def ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def stream(x):
    """The current stream of x's device."""
    return ctypes.c_void_p(torch.cuda.current_stream(x.device).cuda_stream)


def on_device(x):
    """Launches go to x's device, whichever is current."""
    return _SAME if x.device.index == torch.cuda.current_device() else torch.cuda.device(x.device)


def rows2d(x):
    """x [..., D] as rows [R, D] of contiguous columns: a view where its strides allow one.
    (A size of 1 has any stride: given as 0.)"""
    x = x.detach()
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if (x.stride(1) != 1 and x.size(1) > 1) or (x.size(0) > 1 and x.stride(0) < 0):
        x = x.contiguous()
    return x
