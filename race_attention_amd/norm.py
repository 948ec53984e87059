"""Root-mean-square norm with the residual's addition, on the HIP kernels.

``rms_norm(x, weight, residual=None, eps=1e-6)`` normalises x [..., D], or the sum
h = x + residual, by its root mean square and scales it by weight [D]; with a residual
it returns (y, h), h being the next block's residual.  Differentiable in x, weight and
residual.  ``rms_norm_fp8`` gives y in 8-bit blocks for an 8-bit linear layer
(race_attention_amd.fp8), without a gradient.

x is bf16 or fp32; the residual has x's type, or is fp32 beside a bf16 x (the residual
stream of an autocast model); y has x's type and h the residual's.  y normalises the
unrounded sum.
"""
from __future__ import annotations

import ctypes

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from ._tensors import DTYPES, native, on_device, ptr, require_gpu, rows2d, stream
from .fp8 import BlockFp8, _empty_blocks


def _check(x, weight, residual):
    require_gpu(x, weight, *(() if residual is None else (residual,)))
    if x.dim() < 1 or weight.shape != x.shape[-1:]:
        raise ValueError(f"weight must be [D] for x [..., D]; got {tuple(weight.shape)} and {tuple(x.shape)}")
    if x.dtype not in DTYPES or not weight.is_floating_point():
        raise TypeError(f"unsupported dtypes {x.dtype}, {weight.dtype} (x: bf16 or fp32; weight: floating point)")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual {tuple(residual.shape)} and x {tuple(x.shape)} differ in shape")
        if residual.dtype != x.dtype and not (x.dtype is torch.bfloat16 and residual.dtype is torch.float32):
            raise TypeError(f"a {residual.dtype} residual beside a {x.dtype} x: the same type, or fp32 beside bf16")
        if residual.device != x.device:
            raise RuntimeError("x and residual are on different devices")
    if weight.device != x.device:
        raise RuntimeError("x and weight are on different devices")


def _desc(x2, r2, eps):
    d = _lib.NormDesc()
    d.rows, d.D = x2.shape
    d.x_stride = x2.stride(0)
    d.dtype = DTYPES[x2.dtype]
    d.r_dtype = DTYPES[x2.dtype if r2 is None else r2.dtype]
    if r2 is not None:
        d.r_stride = r2.stride(0)
    d.y_stride = d.h_stride = d.D  # outputs are contiguous
    d.eps = float(eps)
    return d


def _weight32(w):
    return w.detach().to(torch.float32).contiguous()


def rms_norm_raw(x, weight, residual, eps, want_rstd):
    """(y, h or None, rstd [rows] or None) without autograd."""
    _check(x, weight, residual)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = None if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    rows = x.numel() // max(1, x.shape[-1])
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if want_rstd else None
    if x.numel() == 0:
        return y, h, rstd
    x2, r2, w = rows2d(x), None if residual is None else rows2d(residual), _weight32(weight)
    d = _desc(x2, r2, eps)
    with on_device(x):
        rc = _lib.load().race_rms_norm(ctypes.byref(d), ptr(x2), ptr(r2), ptr(w), ptr(y), ptr(h), ptr(rstd), stream(x))
    _lib.check(rc, "race_rms_norm")
    return y, h, rstd


def rms_norm_bwd_raw(x, residual, weight, rstd, dy, dh, eps, x_dtype):
    """(dx, dresidual, dw fp32) of the sum x + residual, or of residual alone where x is
    None: dx and dresidual are one tensor where their types are the same."""
    D, shape, r_dtype, dev = weight.numel(), residual.shape, residual.dtype, residual.device
    dx = torch.empty(shape, dtype=x_dtype, device=dev)
    dr = dx if r_dtype == x_dtype else torch.empty(shape, dtype=r_dtype, device=dev)
    if residual.numel() == 0:
        return dx, dr, torch.zeros(D, dtype=torch.float32, device=dev)
    dw = torch.empty(D, dtype=torch.float32, device=dev)
    x2, r2, dy2, w = None if x is None else rows2d(x), rows2d(residual), rows2d(dy.to(x_dtype)), _weight32(weight)
    dh2 = None if dh is None else rows2d(dh.to(r_dtype))
    d = _lib.NormDesc()
    d.rows, d.D = r2.shape
    d.x_stride = 0 if x2 is None else x2.stride(0)
    d.r_stride, d.dy_stride = r2.stride(0), dy2.stride(0)
    d.dh_stride = 0 if dh2 is None else dh2.stride(0)
    d.dx_stride = d.dr_stride = D
    d.dtype, d.r_dtype, d.eps = DTYPES[x_dtype], DTYPES[r_dtype], float(eps)
    lib = _lib.load()
    ws = torch.empty(lib.race_rms_norm_bwd_workspace_bytes(ctypes.byref(d)), dtype=torch.uint8, device=dev)
    with on_device(residual):
        rc = lib.race_rms_norm_bwd(ctypes.byref(d), ptr(x2), ptr(r2), ptr(w), ptr(rstd), ptr(dy2), ptr(dh2), ptr(dx),
                                   None if dr is dx else ptr(dr), ptr(dw), ptr(ws), ws.numel(), stream(residual))
    _lib.check(rc, "race_rms_norm_bwd")
    return dx, dr, dw


class RMSNormFunction(torch.autograd.Function):
    """forward(x, weight, residual or None, eps) -> y, or (y, h) with a residual."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, rstd = rms_norm_raw(x, weight, residual, eps, True)
        # the sum as y used it: an fp32 h holds it, a bf16 one is rounded
        kept = (None, x) if h is None else (None, h) if h.dtype is torch.float32 else (x, residual)
        ctx.save_for_backward(*kept, weight, rstd)
        ctx.cfg = (eps, x.dtype)
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        x, residual, weight, rstd = ctx.saved_tensors
        eps, x_dtype = ctx.cfg
        if dy is None and dh is None:
            return None, None, None, None
        if dy is None:
            dy = torch.zeros(residual.shape, dtype=x_dtype, device=residual.device)
        dx, dr, dw = rms_norm_bwd_raw(x, residual, weight, rstd, dy, dh, eps, x_dtype)
        need = ctx.needs_input_grad
        return (dx if need[0] else None, dw.to(weight.dtype) if need[1] else None, dr if need[2] else None, None)


def rms_norm(x, weight, *, residual=None, eps=1e-6):
    """y, or (y, h) with a residual (see module doc)."""
    out = native(x, "rms_norm", x, weight, residual, float(eps))
    if out is not None:
        return out
    needs = torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                         (residual is not None and residual.requires_grad))
    if needs:
        return RMSNormFunction.apply(x, weight, residual, eps)
    y, h, _ = rms_norm_raw(x.detach(), weight, None if residual is None else residual.detach(), eps, False)
    return y if h is None else (y, h)


def rms_norm_fp8(x, weight, *, residual=None, eps=1e-6):
    """rms_norm with y as a BlockFp8 (one scale for 128 columns of a row).  It has no
    gradient and refuses inputs that ask for one."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or
                                    (residual is not None and residual.requires_grad)):
        raise RuntimeError("rms_norm_fp8 has no backward: call it under torch.no_grad(), or use rms_norm")
    out = native(x, "rms_norm_codes", x, weight, residual, float(eps))
    if out is not None:
        y = BlockFp8(*out[:2])
        return y if residual is None else (y, out[2])
    _check(x, weight, residual)
    y = _empty_blocks(x.shape, x.device)
    h = None if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=x.device)
    if x.numel():
        x2, r2, w = rows2d(x), None if residual is None else rows2d(residual), _weight32(weight)
        d = _desc(x2, r2, eps)
        with on_device(x):
            rc = _lib.load().race_rms_norm_codes(ctypes.byref(d), ptr(x2), ptr(r2), ptr(w), ctypes.byref(y.desc()),
                                                 ptr(h), stream(x))
        _lib.check(rc, "race_rms_norm_codes")
    return y if h is None else (y, h)


class RMSNorm(nn.Module):
    """Root-mean-square norm over the last dimension, with an optional residual:
    forward(x) -> y, forward(x, residual) -> (y, x + residual)."""

    def __init__(self, d, eps=1e-6, device=None):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(d, device=device))

    def forward(self, x, residual=None):
        return rms_norm(x, self.weight, residual=residual, eps=self.eps)

    def extra_repr(self):
        return f"{self.weight.numel()}, eps={self.eps}"
