"""Root-mean-square norm kernels against fp64 (tests/blocks_ref.py).

Tolerances, per element, u = 2^-24: the sum of squares adds at most `chain` values in one
lane and 8 across lanes, so its relative error is (chain + 9) u, and rstd's half of that and 3 u
for the mean, root and reciprocal; y adds the sum h (u of |h|), two products, and its type's half step.  dx is
rstd (g - h k): k's error is that of a sum of D products over the same chain, relative to the sum of
their magnitudes."""
import math

import pytest
import torch

import blocks_ref as ref
from blocks_ref import U, half_step
from race_attention_amd import _lib, norm
from race_attention_amd.fp8 import BlockFp8

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["c++", "python"])
def path(request, monkeypatch):
    """Every test through the C++ calls and through the Python ones."""
    if request.param == "python":
        monkeypatch.setattr(_lib, "calls", lambda: None)
    else:
        assert _lib.calls() is not None


BF, F32 = torch.bfloat16, torch.float32
EPS = 1e-6


def chain(D):
    return math.ceil(D / 64) + 8 if D <= 1024 else math.ceil(D / 256) + 16


def make(rows, D, dt, rdt, seed=0, grad=False):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, D, generator=g).to(dt)
    r = None if rdt is None else (3 * torch.randn(rows, D, generator=g)).to(rdt)
    w = 1 + 0.2 * torch.randn(D, generator=g)
    dy = torch.randn(rows, D, generator=g).to(dt)
    dh = None if rdt is None else torch.randn(rows, D, generator=g).to(rdt)
    return x, r, w, dy, dh


def check_forward(x, r, w, y, h, eps=EPS):
    y64, h64, _ = ref.rms_norm(x, w, r, eps)
    n = chain(x.shape[-1])
    tol = ((n / 2 + 10) * U + half_step(y.dtype)) * y64.abs() + 2.0 ** -126
    assert ((y.cpu().double() - y64).abs() <= tol).all()
    if r is not None:
        assert torch.equal(h.cpu(), h64.float().to(h.dtype)) or \
            ((h.cpu().double() - h64).abs() <= (half_step(h.dtype) + U) * h64.abs()).all()


def check_backward(x, r, w, dy, dh, dx, dr, dw, eps=EPS):
    _, h64, rstd = ref.rms_norm(x, w, r, eps)
    d64, dw64 = ref.rms_norm_bwd(h64, rstd, w, dy, dh)
    D, n = x.shape[-1], chain(x.shape[-1])
    g = (dy.double() * w.double()).abs()
    size = rstd * (g + h64.abs() * rstd ** 2 * (g * h64.abs()).mean(-1, keepdim=True))
    if dh is not None:
        size = size + dh.double().abs()
    for d in (dx, dr):
        if d is not None:
            tol = (2.5 * n + 40) * U * size + half_step(d.dtype) * d64.abs() + 2.0 ** -126
            assert ((d.cpu().double() - d64).abs() <= tol).all()
    rows = x.numel() // D
    # terms of at most 1024 workgroups: their rows, 4 waves, 64 parts a thread and 16 threads
    terms = math.ceil(rows / 1024) + 4 + 64 + 5
    mag = (dy.double() * h64 * rstd).abs().reshape(-1, D).sum(0)
    assert ((dw.cpu().double() - dw64).abs() <= (terms + n / 2 + 10) * U * mag + 2.0 ** -126).all()


@pytest.mark.parametrize("dt,rdt", [(BF, None), (BF, BF), (BF, F32), (F32, None), (F32, F32)])
@pytest.mark.parametrize("rows,D", [(1, 1), (1, 768), (3, 3), (5, 64), (7, 127), (64, 129), (33, 255), (17, 512),
                                    (1100, 768), (9, 1001), (5, 1024), (4, 1025), (6, 2047), (3, 4096), (2, 5001),
                                    (3, 8192), (2, 16384), (2, 16385), (1, 40000), (4100, 64)])
def test_forward_and_backward(dev, dt, rdt, rows, D):
    x, r, w, dy, dh = make(rows, D, dt, rdt, seed=rows * 7 + D)
    leaves = [t.to(dev).requires_grad_(True) for t in (x, w, r) if t is not None]
    res = norm.rms_norm(leaves[0], leaves[1], residual=leaves[2] if r is not None else None, eps=EPS)
    if r is None:
        check_forward(x, r, w, res.detach(), None)
        dx, dw = torch.autograd.grad(res, leaves, dy.to(dev))
        check_backward(x, r, w, dy, None, dx, None, dw)
        y = norm.rms_norm(leaves[0].detach(), w.to(dev), eps=EPS)
        assert torch.equal(y, res)
    else:
        y, h = res
        assert h.dtype == rdt and y.dtype == dt
        check_forward(x, r, w, y.detach(), h.detach())
        dx, dw, dr = torch.autograd.grad((y, h), leaves, (dy.to(dev), dh.to(dev)))
        assert dx.dtype == dt and dr.dtype == rdt
        check_backward(x, r, w, dy, dh, dx, dr, dw)
        # the gradient of either output alone
        y, h = norm.rms_norm(leaves[0], leaves[1], residual=leaves[2], eps=EPS)
        dx, dw, dr = torch.autograd.grad(y, leaves, dy.to(dev))
        check_backward(x, r, w, dy, None, dx, dr, dw)
        y, h = norm.rms_norm(leaves[0], leaves[1], residual=leaves[2], eps=EPS)
        dx, dw, dr = torch.autograd.grad(h, leaves, dh.to(dev))
        assert torch.equal(dr, dh.to(dev)) and torch.equal(dx, dh.to(dev).to(dt)) and not dw.any()


def test_gradient_against_differences(dev):
    """Central differences of <y, dy> + <h, dh> in fp64 along random directions (the formula itself)."""
    x, r, w, dy, dh = make(6, 300, F32, F32, seed=5)
    leaves = [t.to(dev).requires_grad_(True) for t in (x, w, r)]
    y, h = norm.rms_norm(leaves[0], leaves[1], residual=leaves[2], eps=EPS)
    grads = torch.autograd.grad((y, h), leaves, (dy.to(dev), dh.to(dev)))

    def f(t):
        y, h, _ = ref.rms_norm(t[0], t[1], t[2], EPS)
        return (y * dy.double()).sum() + (h * dh.double()).sum()

    g = torch.Generator().manual_seed(1)
    base = [x.double(), w.double(), r.double()]
    for i in range(3):
        d = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        e = 1e-5
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + e * d, base[i] - e * d
        num = (f(up) - f(down)) / (2 * e)
        got = (grads[i].cpu().double() * d).sum()
        # differences: e^2 third derivatives ~ 1e-9 relative; fp32 gradients: 1e-5 of the sum's size is 100 u
        assert abs(num - got) <= 1e-5 * (grads[i].cpu().double() * d).abs().sum()


@pytest.mark.parametrize("dt,rdt", [(BF, None), (BF, BF), (BF, F32), (F32, F32)])
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 64), (5, 100), (9, 128), (4, 768), (3, 1001), (2, 1300), (3, 4096),
                                    (2, 8200), (1, 20000), (300, 384), (5, 4097), (2, 7000)])
def test_output_in_8_bits(dev, dt, rdt, rows, D):
    x, r, w, _, _ = make(rows, D, dt, rdt, seed=D)
    y = norm.rms_norm_fp8(x.to(dev), w.to(dev), residual=None if r is None else r.to(dev), eps=EPS)
    y, h = (y, None) if r is None else y
    assert isinstance(y, BlockFp8) and y.shape == x.shape and y.scale.shape == (rows, -(-D // 128))
    y64, h64, _ = ref.rms_norm(x, w, r, EPS)
    if r is not None:
        assert ((h.cpu().double() - h64).abs() <= (half_step(h.dtype) + U) * h64.abs()).all()
    scale = torch.exp2(y.scale.view(torch.uint8).cpu().double() - 127)
    rel = (chain(D) / 2 + 10) * U
    amax = ref.blocks_of(y64).abs().amax((1, 3))
    # the scale is the least power of two for amax, whose own error may carry it over a border
    assert (amax <= 448 * scale * (1 + rel)).all() and (amax >= 224 * scale * (1 - rel)).all()
    got = ref.values(y.codes.cpu(), y.scale.cpu())
    s = scale.repeat_interleave(128, 1)[:, :D]
    assert ((got - y64).abs() <= y64.abs() * (2.0 ** -4 + 2 * rel) + s * 2.0 ** -10 * (1 + rel)).all()


def test_rows_of_zeros_and_not_finite(dev):
    """A row of zeros gives zeros (eps alone in the root), infinities and NaN stay in their rows."""
    x = torch.randn(5, 256)
    x[1] = 0
    x[2, 7] = float("nan")
    x[3, 9] = float("inf")
    w = torch.ones(256)
    y = norm.rms_norm(x.to(dev), w.to(dev)).cpu()
    assert not y[1].any() and torch.isnan(y[2]).all() and torch.isnan(y[3, 9]) and not y[3, :9].any()
    check_forward(x[[0, 4]], None, w, y[[0, 4]], None)
    q = norm.rms_norm_fp8(x.to(dev), w.to(dev))
    v = ref.values(q.codes.cpu(), q.scale.cpu())
    assert not v[1].any() and torch.isnan(v[2]).all() and torch.isnan(v[3, 9]) and torch.isfinite(v[[0, 1, 4]]).all()


def test_strides(dev):
    """Rows with a pitch, a token's slice, an expanded residual, permuted leading dimensions, non-contiguous columns."""
    g = torch.Generator().manual_seed(3)
    base = torch.randn(6, 5, 400, generator=g).to(BF).to(dev)
    w = torch.rand(300, generator=g).to(dev)
    for x in (base[:, 0, :300], base[..., 50:350], base.transpose(0, 1)[..., :300], base.transpose(1, 2)[:, :300].transpose(1, 2),
              base[:1, :1, :300], base[:, :, :300].permute(1, 0, 2)):
        y = norm.rms_norm(x, w)
        assert y.shape == x.shape
        check_forward(x.cpu(), None, w.cpu(), y, None)
        r = torch.randn(300, generator=g).to(BF).to(dev).expand(x.shape)
        y, h = norm.rms_norm(x, w, residual=r)
        check_forward(x.cpu(), r.cpu(), w.cpu(), y, h)
    x = base[..., :300].requires_grad_(True)
    y = norm.rms_norm(x, w)
    dx, = torch.autograd.grad(y.sum(), x)  # an expanded gradient: stride 0
    check_backward(x.detach().cpu(), None, w.cpu(), torch.ones(x.shape, dtype=BF), None, dx, None,
                   torch.autograd.grad(norm.rms_norm(x, w.requires_grad_(True)).sum(), w)[0])


@pytest.mark.parametrize("D", [64, 768, 1300, 6000])
@pytest.mark.parametrize("eight", [False, True])
def test_infinite_weights_and_roots(dev, D, eight):
    """An infinite weight, and a row whose squares are under the smallest number (eps 0): the products' infinities,
    NaN where they are 0 times infinity, and the columns and rows beside them as they were."""
    g = torch.Generator().manual_seed(D)
    x, w = torch.randn(4, D, generator=g), torch.ones(D)
    x[1] *= 1e-30
    x[2, 5] = 0
    w[5] = float("inf")
    w[9] = -float("inf")

    def norm_of(x, w):
        if not eight:
            return norm.rms_norm(x.to(dev), w.to(dev), eps=0.0).cpu()
        q = norm.rms_norm_fp8(x.to(dev), w.to(dev), eps=0.0)
        return q.dequantize().float().cpu()

    y, rest = norm_of(x, w), norm_of(x[[0, 2, 3]], torch.ones(D))
    keep = [c for c in range(D) if c not in (5, 9)]
    if eight:  # infinities have no code, and the largest finite value decides the scale
        assert torch.isnan(y[1]).all() and torch.isnan(y[:, [5, 9]]).all()
        assert torch.isfinite(y[[0, 2, 3]][:, keep]).all()
    else:
        assert torch.equal(y[1, keep], torch.copysign(torch.full((D - 2,), float("inf")), x[1, keep]))
        assert torch.isnan(y[2, 5]) and y[0, 5] == torch.sign(x[0, 5]) * float("inf")
        assert y[3, 9] == -torch.sign(x[3, 9]) * float("inf")
        assert torch.equal(y[[0, 2, 3]][:, keep], rest[:, keep])


def test_empty(dev):
    w = torch.ones(64, device=dev, requires_grad=True)
    x = torch.zeros(0, 3, 64, device=dev, requires_grad=True)
    y = norm.rms_norm(x, w)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == dx.shape == x.shape and not dw.any()
    y, h = norm.rms_norm_fp8(x.detach(), w.detach(), residual=x.detach())
    assert y.shape == h.shape == x.shape


def test_refusals(dev):
    x, w = torch.zeros(4, 64, device=dev), torch.ones(64, device=dev)
    with pytest.raises(ValueError):
        norm.rms_norm(x, w[:63])
    with pytest.raises(ValueError):
        norm.rms_norm(x, w, residual=x[:3])
    with pytest.raises(TypeError):
        norm.rms_norm(x.half(), w)
    with pytest.raises(TypeError):
        norm.rms_norm(x, w, residual=x.to(BF))
    with pytest.raises(RuntimeError, match="no backward"):
        norm.rms_norm_fp8(x.requires_grad_(True), w)
    with pytest.raises(RuntimeError):
        norm.rms_norm(x, w.cpu())


def test_offsets_past_32_bits(dev):
    """The last rows of 2.4e9 elements."""
    rows, D = 300000, 8192
    x = torch.zeros(rows, D, dtype=BF, device=dev)
    g = torch.Generator().manual_seed(0)
    tail = torch.randn(3, D, generator=g).to(BF)
    x[-3:] = tail.to(dev)
    w = torch.ones(D)
    y = norm.rms_norm(x, w.to(dev))
    check_forward(tail, None, w, y[-3:], None)
    assert not y[-4].any()
    q = norm.rms_norm_fp8(x, w.to(dev))
    # bf16 y and e4m3 codes of the same number: half a step of either
    v = ref.values(q.codes[-3:].cpu(), q.scale[-3:].cpu())
    y64 = ref.rms_norm(tail, w, None, EPS)[0]
    s = torch.exp2(q.scale[-3:].view(torch.uint8).cpu().double() - 127).repeat_interleave(128, 1)
    assert ((v - y64).abs() <= y64.abs() * (2.0 ** -4 + 100 * U) + s * 2.0 ** -10).all()


def test_streams_and_captured_graphs(dev):
    """On a side stream, and forward with backward captured: replays on new inputs equal eager results bit for bit."""
    x, r, w, dy, dh = (t.to(dev) for t in make(500, 768, BF, BF, seed=9))

    def step():
        y, h = norm.rms_norm(x, w, residual=r, eps=EPS)
        return (y, h) + torch.autograd.grad((y, h), (x, w, r), (dy, dh))

    for t in (x, w, r):
        t.requires_grad_(True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(side, step()))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
            dy.copy_(torch.randn_like(dy))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), k


def test_second_derivatives_are_refused(dev):
    x, w = torch.randn(3, 64, device=dev, requires_grad=True), torch.ones(64, device=dev)
    dx, = torch.autograd.grad(norm.rms_norm(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice|does not require grad"):
        dx.sum().backward()
