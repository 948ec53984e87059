"""The quantiser, the product of 8-bit blocks and the 8-bit linear layer against fp64
(tests/blocks_ref.py).

Codes and scales have to be equal.  Products of small whole numbers are exact whatever the order:
products and sums under 2^16 of a step of 1 lose nothing in the 8-bit matrix instructions, which keep
what is over 2^-18 of the largest product.  Random ones: a block of 128 products is at most
128 * 2^-17 of its largest off, 2^-10 of the sum of magnitudes over all blocks; fp32 outputs are summed
in fp32, K u of it; each output adds its type's half step."""
import pytest
import torch

import blocks_ref as ref
from blocks_ref import U, half_step
from race_attention_amd import _lib, fp8

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["c++", "python"])
def path(request, monkeypatch):
    """Every test through the C++ calls and through the Python ones."""
    if request.param == "python":
        monkeypatch.setattr(_lib, "calls", lambda: None)
    else:
        assert _lib.calls() is not None


BF, F32 = torch.bfloat16, torch.float32


def same(blocks, x, rows=1):
    """blocks hold exactly x's codes and scales."""
    q, s = ref.quantize(x.reshape(-1, x.shape[-1]), rows)
    c = blocks.codes.reshape(-1, x.shape[-1]).cpu().float().double()
    b = blocks.scale.view(torch.uint8).reshape(s.shape).cpu().double() - 127
    assert torch.equal(b, s)
    assert torch.equal(torch.isnan(c), torch.isnan(q)) and torch.equal(c.nan_to_num(), q.nan_to_num())


def hard(R, C, dt, seed=0):
    """Values over many binades with zeros, blocks of zeros, borders of the scale, infinities and NaN."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(R, C, generator=g) * torch.exp2(torch.randint(-20, 20, (R, 1), generator=g).float())
    x = x * torch.exp2(torch.randint(-12, 3, (R, C), generator=g).float())
    x[torch.rand(R, C, generator=g) < 0.05] = 0
    if R > 2:
        x[R // 2] = 0
    if R > 3 and C > 3:
        x[0, 0], x[1, 1], x[3, C - 1] = float("nan"), float("inf"), -float("inf")
    if R > 6:
        x[4] = x[4].clamp(-1, 1)
        x[4, C // 2] = 1.75 * 2 ** 5      # 448 * 2^-3: the scale's border itself
        x[5] = x[5].clamp(-1, 1)
        x[5, C // 2] = 1.7578125 * 2 ** 5  # the bf16 behind it
        x[6] = 2.0 ** -130                # under the smallest scale's codes
    return x.to(dt)


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("R,C", [(1, 1), (1, 128), (1, 768), (2, 130), (7, 16), (9, 1000), (128, 128), (129, 257),
                                 (300, 1001), (8, 4096), (1000, 384), (257, 31)])
def test_quantizer(dev, dt, R, C):
    x = hard(R, C, dt, seed=R + C)
    xd = x.to(dev)
    same(fp8.quantize(xd), x)
    same(fp8.quantize(xd, 128), x, 128)
    # transposes and column sums from the same reading
    for rows in (1, 128):
        y, yt, _ = fp8._quantize(xd, rows, True, True, False)
        same(y, x, rows)
        same(yt, x.t().contiguous(), rows)
    y, yt, sums = fp8._quantize(torch.nan_to_num(xd, 0, 0, 0), 1, False, True, True)
    f = torch.nan_to_num(x, 0, 0, 0).double()
    assert y is None
    # at most 8 + 16 + rows / 2048 + 5 terms in a chain
    assert ((sums.cpu().double() - f.sum(0)).abs() <= (30 + R / 2048) * U * f.abs().sum(0)).all()
    # codes of a row behind its last column are zeros up to 16
    pad = fp8.quantize(xd).codes
    if C % 16 and R > 1:
        full = pad.as_strided((R, pad.stride(0)), (pad.stride(0), 1))
        assert not full[:, C:].view(torch.uint8).any()


def test_quantizer_layouts(dev):
    g = torch.Generator().manual_seed(1)
    base = torch.randn(6, 10, 400, generator=g).to(BF).to(dev)
    for x in (base, base[..., 3:303], base.transpose(0, 1), base[:, ::2], base.transpose(1, 2), base[0, 0], base[:, 0],
              base[0, :1].expand(7, 400)):
        q = fp8.quantize(x)
        assert q.shape == x.shape and q.scale.shape == (*x.shape[:-1], -(-x.shape[-1] // 128))
        same(q, x.contiguous().cpu())
    v = fp8.quantize(base[..., :300])
    assert torch.equal(v.dequantize().cpu().double().reshape(60, 300),
                       ref.rounded(base[..., :300].reshape(60, 300).cpu()))
    assert fp8.quantize(base[:0]).shape == (0, 10, 400)


def whole(R, C, block_rows, seed, dev):
    """Blocks of small whole numbers with scales 1/2, 1, 2: (BlockFp8, fp64 values)."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-4, 5, (R, C), generator=g).float().to(torch.float8_e4m3fn)
    rb = -(-R // block_rows)
    scale = torch.randint(126, 129, (rb, -(-C // 128)), generator=g).to(torch.uint8).view(torch.float8_e8m0fnu)
    return fp8.BlockFp8(codes.to(dev), scale.to(dev), block_rows), ref.values(codes, scale, block_rows)


@pytest.mark.parametrize("rows_a,rows_b", [(1, 128), (1, 1), (128, 128), (128, 1)])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 16, 128), (1, 2304, 768), (3, 17, 130), (16, 96, 1000), (17, 100, 512),
                                   (33, 257, 4096), (64, 64, 77), (65, 63, 128), (100, 300, 640), (128, 128, 1),
                                   (130, 1000, 1001), (257, 259, 272), (300, 777, 1000), (1024, 1280, 256), (64, 8192, 528),
                                   (4097, 129, 144), (1, 16, 16384), (129, 130, 8192)])
def test_products_of_whole_numbers_are_exact(dev, M, N, K, rows_a, rows_b):
    a, a64 = whole(M, K, rows_a, 3 * M + K, dev)
    b, b64 = whole(N, K, rows_b, 5 * N + K, dev)
    y64 = a64 @ b64.t()
    for dt in (F32, BF):
        y = fp8.matmul(a, b, out_dtype=dt)
        assert torch.equal(y.cpu(), y64.to(dt)), (dt, (y.cpu().double() - y64).abs().max())
    bias = torch.randint(-50, 50, (N,)).float()
    y = fp8.matmul(a, b, bias=bias.to(dev), out_dtype=F32)
    assert torch.equal(y.cpu().double(), y64 + bias.double())


@pytest.mark.parametrize("M,N,K", [(2, 300, 1000), (40, 512, 4096), (200, 130, 3001), (700, 512, 2048)])
@pytest.mark.parametrize("dt", [BF, F32])
def test_products_of_random_numbers(dev, M, N, K, dt):
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-9, 9, (M, 1), generator=g).float())
    w = torch.randn(N, K, generator=g)
    a, b = fp8.quantize(x.to(dev)), fp8.quantize(w.to(dev), 128)
    a64, b64 = ref.values(a.codes.cpu(), a.scale.cpu()), ref.values(b.codes.cpu(), b.scale.cpu(), 128)
    y64, mag = a64 @ b64.t(), a64.abs() @ b64.abs().t()
    y = fp8.matmul(a, b, out_dtype=dt).cpu().double()
    tol = half_step(dt) * y64.abs() + (2.0 ** -10 if dt is BF else K * U) * mag
    assert ((y - y64).abs() <= tol).all()


def test_pitches_and_alignment(dev):
    """Operands inside larger arrays, at any byte: views of codes and scales, read in place or copied."""
    g = torch.Generator().manual_seed(2)
    codes = torch.randint(-4, 5, (400, 700), generator=g).float().to(torch.float8_e4m3fn).to(dev)
    scale = torch.randint(126, 129, (400, 9), generator=g).to(torch.uint8).view(torch.float8_e8m0fnu).to(dev)
    for c0, K, s0 in ((0, 512, 0), (16, 512, 1), (1, 500, 2), (3, 640, 4), (700 - 130, 130, 7)):
        nk = -(-K // 128)
        for M in (5, 70, 300):
            a = fp8.BlockFp8(codes[:M, c0:c0 + K], scale[:M, s0:s0 + nk])
            b = fp8.BlockFp8(codes[50:350, c0:c0 + K], scale[50:53, s0:s0 + nk], 128)
            y64 = ref.values(a.codes.cpu(), a.scale.cpu()) @ ref.values(b.codes.cpu(), b.scale.cpu(), 128).t()
            assert torch.equal(fp8.matmul(a, b, out_dtype=F32).cpu().double(), y64)
            assert torch.equal(fp8.matmul(a, b).cpu(), y64.to(BF))


def test_what_is_not_finite_stays_in_its_row(dev):
    x = torch.randn(200, 256)
    x[7, 200], x[9, 3] = float("nan"), float("inf")
    w = torch.randn(130, 256)
    for M in (10, 200):
        y = fp8.linear(x[:M].to(dev), w.to(dev)).cpu()
        assert torch.isnan(y[[7, 9]]).all() and torch.isfinite(y[[i for i in range(M) if i not in (7, 9)]]).all()
    z = torch.zeros(3, 256)
    assert not fp8.linear(z.to(dev), w.to(dev)).any()


def linear_ref(x, w, b, dy):
    x2 = x.reshape(-1, x.shape[-1])
    wq, q = ref.rounded(w, 128), ref.rounded(x2)
    y, mag = q @ wq.t(), q.abs() @ wq.abs().t()
    if b is not None:
        y = y + b.double()
    if dy is None:
        return y, mag
    d2 = dy.reshape(-1, dy.shape[-1])
    d, dt, xt = ref.rounded(d2), ref.rounded(d2.t().contiguous()), ref.rounded(x2.t().contiguous())
    return (y, mag), (d @ wq, d.abs() @ wq.abs()), (dt @ xt.t(), dt.abs() @ xt.abs().t()), (d2.double().sum(0), d2.double().abs().sum(0))


def near(got, want, mag, n):
    tol = half_step(got.dtype) * want.abs() + (2.0 ** -10 if got.dtype is BF else n * U) * mag
    assert ((got.cpu().double().reshape(want.shape) - want).abs() <= tol).all()


@pytest.mark.parametrize("xdt,wdt,bias", [(BF, F32, True), (BF, BF, False), (F32, F32, True)])
@pytest.mark.parametrize("shape,N", [((1, 128), 64), ((3, 5, 100), 33), ((64, 256), 300), ((2, 33, 384), 1536), ((130, 1000), 257),
                                     ((700, 129), 128), ((1, 1), 1), ((4, 500, 64), 96)])
def test_linear_layer_and_its_gradients(dev, xdt, wdt, bias, shape, N):
    g = torch.Generator().manual_seed(N)
    x = torch.randn(shape, generator=g).to(xdt)
    w = (0.05 * torch.randn(N, shape[-1], generator=g)).to(wdt)
    b = torch.randn(N, generator=g) if bias else None
    dy = torch.randn(*shape[:-1], N, generator=g).to(xdt)
    leaves = [t.to(dev).requires_grad_(True) for t in (x, w, b) if t is not None]
    y = fp8.linear(*leaves)
    assert y.dtype == xdt and y.shape == dy.shape
    dx, dw, *db = torch.autograd.grad(y, leaves, dy.to(dev))
    assert dx.dtype == xdt and dw.dtype == wdt and dx.shape == x.shape and dw.shape == w.shape
    (y64, ymag), (dx64, xmag), (dw64, wmag), (db64, bmag) = linear_ref(x, w, b, dy)
    rows = x.numel() // shape[-1]
    near(y.detach(), y64, ymag + (0 if b is None else b.double().abs()), shape[-1] + 2)
    near(dx, dx64, xmag, N)
    near(dw, dw64, wmag, rows)
    if bias:
        assert ((db[0].cpu().double() - db64).abs() <= (30 + rows / 2048) * U * bmag).all()
    # without gradients, and with the weight in 8 bits: the same product
    with torch.no_grad():
        assert torch.equal(fp8.linear(leaves[0], leaves[1], leaves[2] if bias else None), y)
        assert torch.equal(fp8.linear(leaves[0], fp8.quantize(leaves[1], 128), leaves[2] if bias else None), y)
    # gradients of some inputs alone
    for i in range(len(leaves)):
        part = [t.detach().requires_grad_(i == j) for j, t in enumerate(leaves)]
        got, = torch.autograd.grad(fp8.linear(*part), part[i], dy.to(dev))
        assert torch.equal(got, (dx, dw, *db)[i])


@pytest.mark.parametrize("dt", [BF, F32])
@pytest.mark.parametrize("R,N,K", [(1, 768, 768), (16, 96, 1000), (1, 16, 4096), (1, 16, 4097), (5, 300, 5000),
                                   (16, 4096, 4096), (16, 4112, 4096), (3, 33000, 520), (17, 100, 4100)])
def test_rows_quantised_inside_or_before_the_product(dev, dt, R, N, K):
    """A serving call's rows have the quantiser's codes, wherever they are formed: the product of its codes, bit for
    bit; the last row of a larger batch of the same kernel too, and rows with a pitch."""
    g = torch.Generator().manual_seed(N + K)
    x = (torch.randn(R, K, generator=g) * torch.exp2(torch.randint(-9, 9, (R, K), generator=g).float())).to(dt).to(dev)
    w = fp8.quantize(torch.randn(N, K, generator=g).to(dev), 128)
    bias = torch.randn(N, generator=g).to(dev)
    with torch.no_grad():
        y = fp8.linear(x, w, bias)
        assert torch.equal(y, fp8.matmul(fp8.quantize(x), w, bias=bias, out_dtype=dt))
        wide = torch.full((R, K + 24), float("nan"), dtype=dt, device=dev)
        wide[:, :K] = x
        assert torch.equal(fp8.linear(wide[:, :K], w, bias), y)


def test_linear_gradient_follows_differences(dev):
    """The 8-bit gradients are those of the layer up to the rounding of their operands to e4m3: a product
    of two operands that are each at most 2^-4 off per value is 2^-3 (1 + 2^-5) of the sum of magnitudes off."""
    g = torch.Generator().manual_seed(4)
    x, w, dy = (torch.randn(s, generator=g) for s in ((100, 256), (192, 256), (100, 192)))
    leaves = [t.to(dev).requires_grad_(True) for t in (x, w)]
    dx, dw = torch.autograd.grad(fp8.linear(*leaves), leaves, dy.to(dev))
    for got, a, b in ((dx, dy, w), (dw, dy.t(), x)):
        want, mag = a.double() @ b.double(), a.double().abs() @ b.double().abs()
        assert ((got.cpu().double() - want).abs() <= 0.13 * mag + 1e-6).all()
        # and in the mean far nearer: errors of random signs
        assert ((got.cpu().double() - want).norm() / want.norm()) < 0.06


def test_frozen_module(dev):
    torch.manual_seed(0)
    m = fp8.Linear(384, 100).to(dev)
    x = torch.randn(5, 384, device=dev)
    want = m(x).detach()
    m.freeze()
    with pytest.raises(RuntimeError, match="no backward"):
        m(x.clone().requires_grad_(True))
    assert torch.equal(m(x), want) and list(m.state_dict()) == ["weight", "bias"]
    other = fp8.Linear(384, 100).to(dev)
    m.load_state_dict(other.state_dict())  # quantised anew
    assert torch.equal(m(x), other(x).detach())
    with torch.no_grad():
        m.weight.zero_()
    assert torch.equal(m.unfreeze()(x).detach(), m.bias.detach().expand(5, 100))
    m.to(torch.bfloat16)
    with torch.autocast("cuda", dtype=BF):
        assert other(x).dtype is BF
    with torch.autocast("cuda", dtype=torch.float16), pytest.raises(TypeError):
        other(x)


def test_empty(dev):
    w, b = torch.randn(8, 64, device=dev, requires_grad=True), torch.randn(8, device=dev, requires_grad=True)
    x = torch.zeros(0, 3, 64, device=dev, requires_grad=True)
    y = fp8.linear(x, w, b)
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == (0, 3, 8) and not gw.any() and not gb.any()
    e = fp8.quantize(torch.zeros(4, 0, device=dev))
    assert not fp8.matmul(e, fp8.quantize(torch.zeros(5, 0, device=dev), 128)).any()


def test_refusals(dev):
    x, w = torch.zeros(4, 128, device=dev), torch.zeros(8, 128, device=dev)
    a, b = fp8.quantize(x), fp8.quantize(w, 128)
    for bad in (lambda: fp8.quantize(x.half()), lambda: fp8.linear(x.half(), w), lambda: fp8.linear(x, w.double()),
                lambda: fp8.matmul(a, b, out_dtype=torch.float16),
                lambda: fp8.matmul(fp8.BlockFp8(x, a.scale), b)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: fp8.quantize(x, 64), lambda: fp8.quantize(x[None], 128), lambda: fp8.linear(x[:, :100], w),
                lambda: fp8.linear(x, w, torch.zeros(7, device=dev)), lambda: fp8.matmul(a, fp8.BlockFp8(a.codes, b.scale)),
                lambda: fp8.matmul(a, fp8.BlockFp8(b.codes, b.scale, 2)), lambda: fp8.matmul(a, fp8.quantize(w[:, :64], 128))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        fp8.linear(x, w.cpu())


def test_outputs_past_32_bits(dev):
    """2.8e9 outputs, and codes past 2^31 bytes: the last rows and columns."""
    M, N, K = 70000, 40000, 32
    a, a64 = whole(M, K, 1, 1, dev)
    b, b64 = whole(N, K, 128, 2, dev)
    y = fp8.matmul(a, b)
    for i in (0, 69999, 54321):
        assert torch.equal(y[i].cpu(), (a64[i] @ b64.t()).to(BF))
    del y
    M, K = 270000, 8192
    x = torch.zeros(M, K, dtype=BF, device=dev)
    x[-2:] = torch.randint(-4, 5, (2, K)).to(BF).to(dev)
    q = fp8.quantize(x)
    same(fp8.BlockFp8(q.codes[-3:], q.scale[-3:]), x[-3:].cpu())
    b, b64 = whole(100, K, 128, 3, dev)
    y = fp8.matmul(q, b, out_dtype=F32)
    assert torch.equal(y[-2:].cpu().double(), x[-2:].cpu().double() @ b64.t()) and not y[-3].any()


def test_streams_and_captured_graphs(dev):
    """A training step and a token's step on a side stream and captured: replays equal eager results bit for bit."""
    torch.manual_seed(1)
    x = torch.randn(300, 384, device=dev, dtype=BF, requires_grad=True)
    w = (0.05 * torch.randn(1001, 384, device=dev)).requires_grad_(True)
    b = torch.randn(1001, device=dev, requires_grad=True)
    dy = torch.randn(300, 1001, device=dev, dtype=BF)
    tok, wq = torch.randn(2, 384, device=dev, dtype=BF), fp8.quantize(w.detach(), 128)

    def step():
        y = fp8.linear(x, w, b)
        with torch.no_grad():
            z = fp8.linear(tok, wq, b)
        return (y, z) + torch.autograd.grad(y, (x, w, b), dy)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(side, step()))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            for t in (x, dy, tok):
                t.copy_(torch.randn_like(t))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(p, q) for p, q in zip(got, step())), k
