"""Matrices in 8-bit blocks and linear layers on them.

A ``BlockFp8`` holds e4m3 codes and a power-of-two scale (e8m0) for each 128 columns of a
row, or of 128 rows (weights).  ``quantize`` makes one; ``matmul(a, b)`` is a b^T + bias on the
matrix cores.  Scales are powers of two: a code is then its value rounded once, and the matrix
cores apply the scales.  Products with an fp32 output (the weights' gradients) are summed in
fp32, those with a bf16 output as the 8-bit matrix instructions sum, at twice the rate and
about 2e-5 of the sum's norm off.

``linear(x, weight, bias)`` is a linear layer in 8 bits.  With a tensor as the weight it
is differentiable: the forward quantises x (a scale for 128 columns of a row) and the weight (for
128 x 128), the backward dy likewise, and dx = dy W and dW = dy^T x are 8-bit products
too, of operands quantised along the contraction.  With a BlockFp8 as the weight it serves:
up to 16 rows of x, such as single tokens, are quantised inside the product where the weight
is small enough that this pays.  ``Linear`` is the module,
``Linear.freeze()`` turns its weight into a BlockFp8 once.
"""
from __future__ import annotations

import ctypes

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from ._tensors import DTYPES, native, on_device, ptr, require_gpu, rows2d, stream

BLOCK = 128
_CODES = (torch.float8_e4m3fn, torch.uint8)
_SCALES = (torch.float8_e8m0fnu, torch.uint8)
# rows of dy and x whose product dW is: its operands' pitch is under 2^22 bytes
_MAX_TOKENS = (1 << 22) - 16


class BlockFp8:
    """codes [..., cols] (float8_e4m3fn) and scale [..., ceil(cols / 128)] (float8_e8m0fnu):
    a scale for each 128 columns of block_rows rows (128: codes [rows, cols] and scale
    [ceil(rows / 128), ceil(cols / 128)])."""

    __slots__ = ("codes", "scale", "block_rows")

    def __init__(self, codes, scale, block_rows=1):
        self.codes, self.scale, self.block_rows = codes, scale, block_rows

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    def check(self, name):
        """Raise where codes and scales do not belong together."""
        c, s = self.codes, self.scale
        require_gpu(c, s)
        if c.dtype not in _CODES or s.dtype not in _SCALES:
            raise TypeError(f"{name}: codes {c.dtype} and scales {s.dtype} are not e4m3 and e8m0")
        if self.block_rows not in (1, BLOCK) or c.dim() < 1 or (self.block_rows == BLOCK and c.dim() != 2):
            raise ValueError(f"{name}: a scale is shared by 1 row, or by 128 rows of a matrix")
        want = (-(-c.shape[0] // BLOCK),) if self.block_rows == BLOCK else tuple(c.shape[:-1])
        want += (-(-c.shape[-1] // BLOCK),)
        if tuple(s.shape) != want:
            raise ValueError(f"{name}: codes {tuple(c.shape)} need scales {want}, got {tuple(s.shape)}")
        if s.device != c.device:
            raise RuntimeError(f"{name}: codes and scales are on different devices")

    def desc(self):
        """(of codes and scales as rows) the descriptor that the C calls take."""
        d = _lib.Blocks()
        c, s = rows2d(self.codes), rows2d(self.scale)
        d.codes, d.scale = c.data_ptr(), s.data_ptr()
        d.rows, d.cols = c.shape
        d.ld = c.stride(0) if d.rows > 1 else max(c.stride(0), d.cols)
        d.scale_ld = s.stride(0) if s.shape[0] > 1 else max(s.stride(0), s.shape[1])
        d.block_rows = self.block_rows
        d._keep = (c, s)
        return d

    def dequantize(self, dtype=torch.float32):
        """The values (a plain torch expression, for inspection)."""
        self.check("blocks")
        s = self.scale.view(torch.uint8).to(torch.int32)
        s = torch.where(s == 255, torch.full_like(s, 0x7fc00000),
                        torch.where(s == 0, torch.full_like(s, 1 << 22), s << 23)).view(torch.float32)
        if self.block_rows == BLOCK:
            s = s.repeat_interleave(BLOCK, 0)[:self.codes.shape[0]]
        s = s.repeat_interleave(BLOCK, -1)[..., :self.codes.shape[-1]]
        return (self.codes.view(torch.float8_e4m3fn).float() * s).to(dtype)


def _empty_blocks(shape, device, block_rows=1):
    """Blocks for the kernels to write: rows of whole 16-byte pieces, of which codes is a view."""
    cols = shape[-1]
    ld = -(-cols // 16) * 16
    codes = torch.empty(*shape[:-1], ld, dtype=torch.float8_e4m3fn, device=device)
    rows = (-(-shape[0] // BLOCK),) if block_rows == BLOCK else tuple(shape[:-1])
    scale = torch.empty(*rows, -(-cols // BLOCK), dtype=torch.float8_e8m0fnu, device=device)
    return BlockFp8(codes if ld == cols else codes[..., :cols], scale, block_rows)


def _quantize(x, block_rows, want, want_t, want_sums):
    """(blocks of x [R, C], blocks of its transpose, column sums fp32 [C]), None where not wanted."""
    R, C = x.shape
    y = _empty_blocks((R, C), x.device, block_rows) if want else None
    yt = _empty_blocks((C, R), x.device, block_rows) if want_t else None
    sums = torch.empty(C, dtype=torch.float32, device=x.device) if want_sums else None
    lib = _lib.load()
    ws = None
    if want_sums:
        ws = torch.empty(lib.race_quantize_workspace_bytes(R, C), dtype=torch.uint8, device=x.device)
    with on_device(x):
        rc = lib.race_quantize(ptr(x), DTYPES[x.dtype], R, C, x.stride(0), ctypes.byref(y.desc()) if want else None,
                               ctypes.byref(yt.desc()) if want_t else None, ptr(sums), ptr(ws),
                               0 if ws is None else ws.numel(), stream(x))
    _lib.check(rc, "race_quantize")
    return y, yt, sums


def quantize(x, block_rows=1):
    """x [..., K] (bf16 or fp32) as a BlockFp8: a scale for 128 columns of a row, or with
    block_rows=128 (x [N, K], a weight) of 128 rows.  Not differentiable."""
    require_gpu(x)
    if x.dtype not in DTYPES:
        raise TypeError(f"unsupported dtype {x.dtype} (bf16 or fp32)")
    if block_rows not in (1, BLOCK) or x.dim() < 1 or (block_rows == BLOCK and x.dim() != 2):
        raise ValueError(f"block_rows=1, or 128 for a matrix [N, K]; got {block_rows} for {tuple(x.shape)}")
    if x.numel() == 0:
        return _empty_blocks(x.shape, x.device, block_rows)
    y = _quantize(rows2d(x), block_rows, True, False, False)[0]
    if x.dim() != 2:
        ld = y.codes.stride(0)
        codes = y.codes.as_strided((*x.shape[:-1], ld), torch.empty(*x.shape[:-1], ld, device="meta").stride())
        y = BlockFp8(codes[..., :x.shape[-1]], y.scale.view(*x.shape[:-1], -1), 1)
    return y


def _bias32(bias, n, dev):
    if bias is None:
        return None
    require_gpu(bias)
    if bias.shape != (n,) or not bias.is_floating_point():
        raise ValueError(f"bias must be floating point [{n}]; got {bias.dtype} {tuple(bias.shape)}")
    if bias.device != dev:
        raise RuntimeError("bias is on another device")
    return bias.detach().to(torch.float32).contiguous()


def _matmul(da, db, shape, bias, out_dtype, dev):
    """Product of two descriptors: out [rows of a, rows of b] as ``shape``."""
    lib = _lib.load()
    out = torch.empty(shape, dtype=out_dtype, device=dev)
    nbytes = lib.race_block_matmul_workspace_bytes(ctypes.byref(da), ctypes.byref(db), DTYPES[out_dtype])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with on_device(out):
        rc = lib.race_block_matmul(ctypes.byref(da), ctypes.byref(db), ptr(bias), ptr(out), DTYPES[out_dtype], db.rows,
                                   ptr(ws), nbytes, stream(out))
    _lib.check(rc, "race_block_matmul")
    return out


def matmul(a, b, *, bias=None, out_dtype=torch.bfloat16):
    """a b^T + bias: a BlockFp8 [..., K], b BlockFp8 [N, K], bias [N] or None -> [..., N]."""
    if out_dtype in DTYPES:
        out = native(a.codes, "matmul", a.codes, a.scale, a.block_rows, b.codes, b.scale, b.block_rows, bias,
                     out_dtype is torch.float32)
        if out is not None:
            return out
    a.check("a")
    b.check("b")
    if b.codes.dim() != 2 or a.shape[-1] != b.shape[1]:
        raise ValueError(f"a [..., K] and b [N, K] expected; got {tuple(a.shape)} and {tuple(b.shape)}")
    if out_dtype not in DTYPES:
        raise TypeError(f"unsupported out_dtype {out_dtype} (bf16 or fp32)")
    if a.device != b.device:
        raise RuntimeError("a and b are on different devices")
    shape, bias = (*a.shape[:-1], b.shape[0]), _bias32(bias, b.shape[0], a.device)
    if 0 in shape or a.shape[-1] == 0:
        out = torch.zeros(shape, dtype=out_dtype, device=a.device)
        return out if bias is None else out + bias.to(out_dtype)
    return _matmul(a.desc(), b.desc(), shape, bias, out_dtype, a.device)


def _few_rows():
    return _lib.load().race_block_linear_rows()


def _linear_few(x2, dw, bias, out_dtype):
    """Up to _few_rows() rows, quantised inside the product."""
    lib = _lib.load()
    R, N = x2.shape[0], dw.rows
    out = torch.empty(R, N, dtype=out_dtype, device=x2.device)
    nbytes = lib.race_block_linear_workspace_bytes(R, ctypes.byref(dw), DTYPES[out_dtype])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x2.device) if nbytes else None
    with on_device(x2):
        rc = lib.race_block_linear(ptr(x2), DTYPES[x2.dtype], R, x2.stride(0) if R > 1 else x2.shape[1], ctypes.byref(dw),
                                   ptr(bias), ptr(out), DTYPES[out_dtype], N, ptr(ws), nbytes, stream(x2))
    _lib.check(rc, "race_block_linear")
    return out


class LinearFunction(torch.autograd.Function):
    """forward(x [..., K], weight [N, K], bias [N] or None, out_dtype) -> [..., N]."""

    @staticmethod
    def forward(ctx, x, weight, bias, out_dtype):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        N, K = weight.shape
        x2, w2, b = rows2d(x), rows2d(weight), _bias32(bias, N, x.device)
        R = x2.shape[0]
        wq, wt, _ = _quantize(w2, BLOCK, True, need_x, False)
        if R <= _few_rows():
            xt = _quantize(x2, 1, False, True, False)[1] if need_w else None
            y = _linear_few(x2, wq.desc(), b, out_dtype)
        else:
            xq, xt, _ = _quantize(x2, 1, True, need_w, False)
            y = _matmul(xq.desc(), wq.desc(), (R, N), b, out_dtype, x.device)
        kept = [t for blocks in (xt, wt) for t in ((None, None) if blocks is None else (blocks.codes, blocks.scale))]
        ctx.save_for_backward(*kept)
        ctx.cfg = (x.shape, x.dtype, weight.dtype, None if bias is None else bias.dtype)
        return y.view(*x.shape[:-1], N)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        xc, xs, wc, ws = ctx.saved_tensors
        x_shape, x_dtype, w_dtype, b_dtype = ctx.cfg
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        dy2 = rows2d(dy)
        q, qt, sums = _quantize(dy2, 1, need_x or not need_w, need_w, need_b)
        dx = dw = None
        if need_x:
            wt = BlockFp8(wc, ws, BLOCK)
            dx = _matmul(q.desc(), wt.desc(), x_shape, None, x_dtype, dy.device)
        if need_w:
            xt = BlockFp8(xc, xs, 1)
            dw = _matmul(qt.desc(), xt.desc(), (dy2.shape[1], x_shape[-1]), None, w_dtype, dy.device)
        return dx, dw, sums.to(b_dtype) if need_b else None, None


def _out_dtype(x):
    """x's type, or autocast's."""
    if torch.is_autocast_enabled("cuda"):
        t = torch.get_autocast_dtype("cuda")
        if t not in DTYPES:
            raise TypeError(f"unsupported autocast dtype {t} (bf16 or fp32)")
        return t
    return x.dtype


def linear(x, weight, bias=None):
    """x [..., K] -> [..., N] in 8 bits (see module doc): weight [N, K] as a tensor
    (differentiable) or a BlockFp8 (serving).  The result has x's type, or autocast's."""
    frozen = isinstance(weight, BlockFp8)
    if torch.is_tensor(x) and x.dtype in DTYPES:
        fp32 = _out_dtype(x) is torch.float32
        out = (native(x, "linear", x, weight.codes, weight.scale, weight.block_rows, bias, fp32) if frozen
               else native(x, "linear", x, weight, None, 0, bias, fp32))
        if out is not None:
            return out
    w = weight.codes if frozen else weight
    require_gpu(x, w)
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise ValueError(f"x [..., K] and weight [N, K] expected; got {tuple(x.shape)} and {tuple(w.shape)}")
    if x.dtype not in DTYPES or not (frozen or weight.dtype in DTYPES):
        raise TypeError(f"unsupported dtypes {x.dtype}, {w.dtype} (bf16 or fp32)")
    if w.device != x.device:
        raise RuntimeError("x and weight are on different devices")
    out_dtype, N = _out_dtype(x), w.shape[0]
    grad = torch.is_grad_enabled()
    if frozen:
        weight.check("weight")
        if grad and (x.requires_grad or (bias is not None and bias.requires_grad)):
            raise RuntimeError("a weight in 8 bits has no backward: call under torch.no_grad(), or pass the weight as a tensor")
    elif grad and (x.requires_grad or w.requires_grad or (bias is not None and bias.requires_grad)):
        b = _bias32(bias, N, x.device)  # checks
        if x.numel() == 0 or w.numel() == 0:
            return _empty_linear(x, weight, bias, out_dtype)
        if x.numel() // x.shape[-1] > _MAX_TOKENS:
            raise ValueError(f"more than {_MAX_TOKENS} rows of x in a differentiable call: split them")
        return LinearFunction.apply(x, weight, bias, out_dtype)
    b = _bias32(bias, N, x.device)
    if x.numel() == 0 or w.numel() == 0:
        return _empty_linear(x, w, bias, out_dtype)
    if not frozen:
        weight = _quantize(rows2d(weight), BLOCK, True, False, False)[0]
    x2, dw = rows2d(x), weight.desc()
    R = x2.shape[0]
    if R <= _few_rows():
        y = _linear_few(x2, dw, b, out_dtype)
    else:
        y = _matmul(_quantize(x2, 1, True, False, False)[0].desc(), dw, (R, N), b, out_dtype, x.device)
    return y.view(*x.shape[:-1], N)


def _empty_linear(x, w, bias, out_dtype):
    """No rows, outputs or contraction: zeros, with torch's own gradients of nothing."""
    y = x.to(out_dtype) @ w.to(out_dtype).t() if w.dtype in DTYPES else torch.zeros(
        *x.shape[:-1], w.shape[0], dtype=out_dtype, device=x.device)
    return y if bias is None else y + bias.to(out_dtype)


class Linear(nn.Linear):
    """nn.Linear whose products run in 8 bits (parameters and state_dict are nn.Linear's).
    After freeze() the weight is the BlockFp8 made of it then, for serving."""

    frozen = None

    def freeze(self):
        """Quantise the weight as it is now; forward then uses the result, which has no gradient.
        Loading a state_dict, or another type or GPU, quantises anew; unfreeze() goes back, and so does
        moving the module off the GPU."""
        self.frozen = quantize(self.weight.detach(), BLOCK)
        return self

    def unfreeze(self):
        self.frozen = None
        return self

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        return self._refreeze()

    def _load_from_state_dict(self, *args, **kwargs):
        super()._load_from_state_dict(*args, **kwargs)
        self._refreeze()

    def _refreeze(self):
        if self.frozen is not None:
            self.frozen = None
            if self.weight.is_cuda:
                self.freeze()
        return self

    def forward(self, x):
        if self.frozen is not None:
            return linear(x, self.frozen, None if self.bias is None else self.bias.detach())
        return linear(x, self.weight, self.bias)
