"""The operators around the attention in 64 bits on the CPU: numpy-like torch
expressions of their definitions, for the tests of the kernels."""
import torch

U = 2.0 ** -24   # half a step of fp32, relative
UB = 2.0 ** -8   # of bf16 (torch.finfo(torch.bfloat16).eps / 2)
BLK = 128


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def scale_exponent(amax):
    """The least s with amax / 2^s <= 448, 0 for zeros, by comparing with powers of two (exact in fp64)."""
    s = torch.floor(torch.log2(amax.clamp_min(2.0 ** -140) / 448)) - 1
    for _ in range(4):
        s = torch.where(amax > 448 * torch.exp2(s), s + 1, s)
    return torch.where(amax > 0, s.clamp_min(-127), torch.zeros_like(s))


def blocks_of(x, block_rows=1):
    R, C = x.shape
    full = torch.zeros(-(-R // block_rows) * block_rows, -(-C // BLK) * BLK, dtype=torch.float64)
    full[:R, :C] = x.double()
    return full.view(-1, block_rows, full.shape[1] // BLK, BLK)


def quantize(x, block_rows=1):
    """x [R, C] on the CPU -> (codes fp64 values [R, C], NaN where not finite; exponents [R / rows, C / 128])."""
    R, C = x.shape
    b = blocks_of(x, block_rows)
    amax = torch.where(b.isfinite(), b.abs(), torch.zeros_like(b)).amax((1, 3))
    s = scale_exponent(amax)
    y = b / torch.exp2(s)[:, None, :, None]
    y = torch.where(y.isfinite(), y, torch.full_like(y, float("nan")))
    # |y| <= 448: fp32 holds y exactly (a power of two apart from x), and torch rounds to nearest even
    q = y.float().to(torch.float8_e4m3fn).double()
    return q.reshape(b.shape[0] * block_rows, -1)[:R, :C], s


def values(codes, scale, block_rows=1):
    """fp64 values of stored codes and scale bytes (CPU tensors)."""
    R, C = codes.shape
    s = torch.exp2(scale.view(torch.uint8).double() - 127)
    s = s.repeat_interleave(block_rows, 0)[:R].repeat_interleave(BLK, 1)[:, :C]
    return codes.view(torch.float8_e4m3fn).double() * s


def rounded(x, block_rows=1):
    q, s = quantize(x, block_rows)
    s = torch.exp2(s).repeat_interleave(block_rows, 0)[:x.shape[0]].repeat_interleave(BLK, 1)[:, :x.shape[1]]
    return q * s


def rms_norm(x, w, residual, eps):
    """(y, h, rstd) in fp64."""
    h = x.double() if residual is None else x.double() + residual.double()
    rstd = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h * rstd * w.double(), h, rstd


def rms_norm_bwd(h, rstd, w, dy, dh):
    g = dy.double() * w.double()
    d = rstd * (g - h * rstd ** 2 * (g * h).mean(-1, keepdim=True))
    return d if dh is None else d + dh.double(), (dy.double() * h * rstd).reshape(-1, h.shape[-1]).sum(0)


def mix32(x):
    x = ((x ^ (x >> 16)) * 0x7feb352d) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def random_bits(place, n, seed):
    """The 32-bit random numbers of elements place .. place + n - 1."""
    c = mix32(torch.tensor(seed & 0xffffffff))
    return mix32((torch.arange(place, place + n) + c) & 0xffffffff)


def adamw(p, g, m, v, *, t, lr, betas, eps, wd):
    """(p, m, v) in fp64."""
    (b1, b2), p, g, m, v = betas, p.double(), g.double(), m.double(), v.double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    return p - lr * wd * p - lr / (1 - b1 ** t) * m / (v.sqrt() / (1 - b2 ** t) ** 0.5 + eps), m, v
