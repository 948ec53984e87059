"""AdamW steps against fp64 (tests/blocks_ref.py).

Tolerances, u = 2^-24: m and v are a sum of two terms whose factors are rounded to fp32 (4 u of each
term's size); the step is a quotient of these, a root and constants (10 u of m's terms over the
denominator), p takes 3 u of itself and its type's half step.  An 8-bit state is a neighbour in e4m3 of the exact value: less
than a spacing off, and the neighbour that the random number chooses unless it falls on the border."""
import copy

import pytest
import torch

import blocks_ref as ref
from blocks_ref import U, half_step
from race_attention_amd import _lib, optim
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
HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
SHAPES = [(1,), (3, 5), (127,), (128,), (129,), (1000, 3), (0,), (64, 768), (4097,), (2, 3, 4, 5), (10001,)]


def make(shapes, pdt, gdt, dev, bits, seed=0):
    g = torch.Generator().manual_seed(seed)
    ps = [torch.randn(s, generator=g).to(pdt) for s in shapes]
    gs = [(torch.randn(s, generator=g) * 10 ** (3 * torch.rand(s, generator=g) - 3)).to(gdt) for s in shapes]
    ms = [0.1 * torch.randn(s, generator=g) for s in shapes]
    rs = [0.1 * (0.1 + torch.randn(s, generator=g).abs()) for s in shapes]
    if bits == 32:
        st = [ms, [r * r for r in rs]]
    else:
        st = []
        for group in (ms, rs):
            out = []
            for t in group:
                n = t.numel()
                q, s = ref.quantize(t.reshape(1, -1)) if n else (t.reshape(1, 0), torch.zeros(1, 0))
                out.append(BlockFp8(q.float().to(torch.float8_e4m3fn).view(t.shape),
                                    (s.view(-1) + 127).to(torch.uint8).view(torch.float8_e8m0fnu)))
            st.append(out)
    return ps, gs, *st


def to_dev(xs, dev):
    return [BlockFp8(x.codes.to(dev), x.scale.to(dev)) if isinstance(x, BlockFp8) else x.to(dev) for x in xs]


def state_values(s):
    n = s.codes.numel()
    return ref.values(s.codes.cpu().reshape(1, n), s.scale.cpu()[None]).view(s.codes.shape) if n else s.codes.cpu().double()


def check_p(p, p0, g, m0, v0, t, h):
    p64, m64, v64 = ref.adamw(p0, g, m0, v0, t=t, lr=h["lr"], betas=h["betas"], eps=h["eps"], wd=h["weight_decay"])
    b1, b2 = h["betas"]
    msize = b1 * m0.double().abs() + (1 - b1) * g.double().abs()
    step = h["lr"] / (1 - b1 ** t) / (v64.sqrt() / (1 - b2 ** t) ** 0.5 + h["eps"])
    tol = 16 * U * step * msize + 4 * U * p0.double().abs() + half_step(p.dtype) * p64.abs() + 2.0 ** -126
    assert ((p.cpu().double() - p64).abs() <= tol).all()
    return m64, v64, msize


@pytest.mark.parametrize("pdt,gdt", [(F32, F32), (F32, BF), (BF, BF), (BF, F32)])
@pytest.mark.parametrize("t", [1, 1000])
def test_states_in_32_bits(dev, pdt, gdt, t):
    ps, gs, ms, vs = make(SHAPES, pdt, gdt, dev, 32)
    P, G, M, V = (to_dev(x, dev) for x in (ps, gs, ms, vs))
    optim.adamw_step(P, G, M, V, step=t, **HYPER)
    for p, p0, g, m, m0, v, v0 in zip(P, ps, gs, M, ms, V, vs):
        m64, v64, msize = check_p(p, p0, g, m0, v0, t, HYPER)
        assert ((m.cpu().double() - m64).abs() <= 4 * U * msize).all()
        assert ((v.cpu().double() - v64).abs() <= 5 * U * v64).all()


@pytest.mark.parametrize("pdt,gdt", [(F32, F32), (BF, BF), (F32, BF), (BF, F32)])
def test_states_in_8_bits(dev, pdt, gdt):
    t, seed = 7, 123
    ps, gs, ms, rs = make(SHAPES, pdt, gdt, dev, 8)
    P, G, M, R = (to_dev(x, dev) for x in (ps, gs, ms, rs))
    optim.adamw_step(P, G, M, R, step=t, seed=seed, **HYPER)
    place = 0
    for p, p0, g, m, m0, r, r0 in zip(P, ps, gs, M, ms, R, rs):
        n = p0.numel()
        if not n:
            continue
        mv, rv = state_values(m0), state_values(r0)
        m64, v64, _ = check_p(p, p0, g, mv, rv * rv, t, HYPER)
        bits = ref.random_bits(place, n, seed)
        for got, want, u in ((m, m64, bits & 0xffff), (r, v64.sqrt(), bits >> 16)):
            want = want.reshape(1, n)
            amax = ref.blocks_of(want).abs().amax((1, 3))
            scale = torch.exp2(got.scale.cpu().view(torch.uint8).double() - 127)[None]
            assert (amax <= 448 * scale * (1 + 8 * U)).all() and (amax >= 224 * scale * (1 - 8 * U)).all()
            s = scale.repeat_interleave(128, 1)[:, :n]
            y = want / s
            spacing = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
            q = got.codes.cpu().float().double().reshape(1, n)
            assert ((q - y).abs() <= spacing * (1 + 1e-4)).all()
            up = y.abs() / spacing + u.double() / 65536
            chosen = torch.sign(y) * torch.floor(up) * spacing
            border = (up - torch.round(up)).abs() < 1e-4  # 16 u of y / spacing <= 16, and more
            assert torch.equal(q[~border], chosen[~border]) and border.float().mean() < 1e-2
        place += -(-n // 128) * 128


def test_8_bit_rounding_is_unbiased_and_states_move(dev):
    """v under a constant gradient converges to g^2 although b2 = 0.999 moves it by less than half a code a step."""
    n = 1 << 16
    g = torch.full((n,), 0.5, device=dev)
    p, m, r = torch.zeros(n, device=dev), *(optim.empty_state8(g) for _ in range(2))
    steps = 500
    for t in range(1, steps + 1):
        optim.adamw_step([p], [g], [m], [r], step=t, seed=t, lr=0.0, weight_decay=0.0)
    want = (0.25 * (1 - 0.999 ** steps)) ** 0.5
    got = (r.codes.float().view(-1, 128) * torch.exp2(r.scale.view(torch.uint8).float() - 127)[:, None]).flatten()
    # the root's rounding is unbiased, its square's mean is then larger by the variance, at most (2^-4)^2 / 4 a step,
    # a thousandth of which enters; the mean over 65536 elements deviates by far less than a percent
    assert abs(got.double().mean().item() / want - 1) < 0.02
    assert got.std() / got.mean() < 0.2


def test_reproducible_and_seeded(dev):
    ps, gs, ms, rs = make([(5000,), (300, 7)], F32, F32, dev, 8)
    out = []
    for seed in (5, 5, 6):
        P, G, M, R = (to_dev(x, dev) for x in (ps, gs, ms, rs))
        optim.adamw_step(P, G, M, R, step=3, seed=seed, **HYPER)
        out.append((P, M, R))
    eq = [all(torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) for a, b in zip(x, y)) for x, y in
          ((out[0][1], out[1][1]), (out[0][1], out[2][1]))]
    assert eq == [True, False]
    assert all(torch.equal(a, b) for a, b in zip(out[0][0], out[2][0]))  # p does not depend on the rounding


@pytest.mark.parametrize("bits", [32, 8])
def test_not_finite_gradients_stay_in_their_elements(dev, bits):
    ps, gs, ms, vs = make([(300,)], F32, F32, dev, bits)
    gs[0][5], gs[0][200] = float("nan"), float("inf")
    P, G, M, V = (to_dev(x, dev) for x in (ps, gs, ms, vs))
    optim.adamw_step(P, G, M, V, step=2, **HYPER)
    bad = torch.zeros(300, dtype=torch.bool)
    bad[[5, 200]] = True
    assert torch.equal(~torch.isfinite(P[0].cpu()), bad)
    if bits == 8:
        assert torch.equal(torch.isnan(M[0].codes.float()).cpu(), bad)
    keep = ~bad
    mv, vv = (ms[0], vs[0]) if bits == 32 else (state_values(ms[0]), state_values(vs[0]) ** 2)
    check_p(P[0][keep.to(dev)], ps[0][keep], gs[0][keep], mv[keep], vv[keep], 2, HYPER)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_unaligned_views(dev, bits):
    """More tensors than a launch takes, at offsets that no vector fits; what lies between them stays as it was."""
    g = torch.Generator().manual_seed(0)
    sizes = [int(torch.randint(1, 700, (1,), generator=g)) for _ in range(131)]
    ps, gs, ms, vs = make([(n,) for n in sizes], F32, F32, dev, bits, seed=4)

    def packed(xs, gap, fill):
        buf = torch.full((sum(x.numel() + gap for x in xs) + gap,), fill, dtype=xs[0].dtype, device=dev) if \
            xs[0].dtype is F32 else torch.zeros(sum(x.numel() + gap for x in xs) + gap, dtype=xs[0].dtype, device=dev)
        at, views = gap, []
        for x in xs:
            views.append(buf[at:at + x.numel()])
            views[-1].copy_(x)
            at += x.numel() + gap
        return buf, views

    buf, P = packed(ps, 3, 7.25)
    _, G = packed(gs, 1, 0.0)
    if bits == 32:
        mbuf, M = packed(ms, 1, 3.5)
        _, V = packed(vs, 5, 0.0)
    else:
        mbuf, mc = packed([m.codes for m in ms], 3, 0)
        M = [BlockFp8(c, m.scale.to(dev)) for c, m in zip(mc, ms)]
        V = to_dev(vs, dev)
    optim.adamw_step(P, G, M, V, step=4, seed=9, **HYPER)
    A, B, C, D = (to_dev(x, dev) for x in (ps, gs, ms, vs))
    optim.adamw_step(A, B, C, D, step=4, seed=9, **HYPER)
    assert all(torch.equal(a, b) for a, b in zip(P, A))
    raw = (lambda s: s) if bits == 32 else (lambda s: s.codes.view(torch.uint8))
    assert all(torch.equal(raw(a), raw(b)) for a, b in zip(M + V, C + D))
    gaps = torch.ones(buf.numel(), dtype=torch.bool, device=dev)
    at = 3
    for n in sizes:
        gaps[at:at + n] = False
        at += n + 3
    assert (buf[gaps] == 7.25).all()


def test_refusals(dev):
    p = torch.zeros(8, 8, device=dev)
    s = optim.empty_state8(p)
    for a in ([p], [p.t()], [p], [p]), ([p], [p[:4]], [p], [p]), ([p], [p], [p], [p[:, :4]]), ([p, p.to(BF)], [p, p], [p, p], [p, p]), \
            ([p], [p], [s], [BlockFp8(s.codes, s.scale[:0])]), ([p, p], [p, p], [p, p.clone()], [p, p.clone()]), \
            ([p], [p.clone()], [p.clone()], [p]):
        with pytest.raises(ValueError):
            optim.adamw_step(*a, step=1, lr=0.1)
    for a in ([p.half()], [p.half()], [p], [p]), ([p], [p], [p.to(BF)], [p]), ([p], [p], [s], [p]), ([p], [p], [p], [s]):
        with pytest.raises(TypeError):
            optim.adamw_step(*a, step=1, lr=0.1)
    with pytest.raises(RuntimeError):
        optim.adamw_step([p], [p.cpu()], [p], [p], step=1, lr=0.1)
    with pytest.raises(ValueError):
        optim.adamw_step([p], [p], [p.clone()], [p.clone()], step=torch.zeros(2, device=dev), lr=0.1)


def test_saved_tensors_notice_the_step(dev):
    """A graph that saved a parameter refuses its backward after the step, as after any in-place operation."""
    p = torch.ones(4, device=dev, requires_grad=True)
    x = torch.ones(4, device=dev, requires_grad=True)
    y = (p * x).sum()
    q = p.detach()
    optim.adamw_step([q], [torch.ones_like(q)], [torch.zeros_like(q)], [torch.zeros_like(q)], step=1, lr=0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def _params(dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=g).to(dev)) for s in ((64, 33), (129,), (7, 5, 3))]


def test_optimizer_equals_torch(dev):
    """30 steps of the module against torch's AdamW in fp64: p after t steps is at most the steps' own errors off."""
    ours, theirs = _params(dev), [torch.nn.Parameter(p.detach().cpu().double()) for p in _params(dev)]
    h = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)
    a, b = optim.AdamW(ours, **h), torch.optim.AdamW(theirs, **h)
    g = torch.Generator().manual_seed(1)
    for k in range(30):
        for p, q in zip(ours, theirs):
            q.grad = torch.randn(p.shape, generator=g).double()
            p.grad = q.grad.float().to(dev)
        q = theirs[2].grad
        if k % 3 == 1:  # a parameter without a gradient is left alone
            ours[2].grad = theirs[2].grad = None
        a.step()
        b.step()
    assert a.state[ours[2]]["step"] == 20
    for p, q in zip(ours, theirs):
        # a step is at most lr (1 + small) in size and 30 u of that off, p 4 u of itself a step
        assert ((p.detach().cpu().double() - q.detach()).abs() <= 30 * (60 * U * h["lr"] + 4 * U * q.detach().abs())).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_optimizer_state_dict(dev, bits, capturable):
    """Saved and loaded in the middle: the run goes on bit for bit, states keep their types (bf16 parameters)."""
    def run(resume):
        ps = _params(dev)
        ps[1] = torch.nn.Parameter(ps[1].detach().to(BF))
        opt = optim.AdamW(ps, lr=1e-2, bits=bits, seed=3, capturable=capturable)
        g = torch.Generator().manual_seed(2)
        for k in range(6):
            if resume and k == 3:
                saved = copy.deepcopy(opt.state_dict())
                opt = optim.AdamW(ps, lr=1e-2, bits=bits, seed=3, capturable=capturable)
                opt.load_state_dict(saved)
            for p in ps:
                p.grad = torch.randn(p.shape, generator=g).to(p.dtype).to(dev)
            opt.step()
        return ps, opt
    (a, oa), (b, ob) = run(False), run(True)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    for x, y in zip(a, b):
        for name, s in oa.state[x].items():
            if torch.is_tensor(s):
                t = ob.state[y][name]
                assert s.dtype == t.dtype and torch.equal(s.view(torch.uint8) if s.dim() else s, t.view(torch.uint8) if t.dim() else t)
    with pytest.raises(ValueError):
        optim.AdamW(_params(dev), bits=40 - bits).load_state_dict(oa.state_dict())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(dev, bits):
    """Replays of a captured step equal eager steps: the step's number, and with it the bias corrections and
    the random numbers, lives on the GPU."""
    def build():
        ps = _params(dev)
        for p in ps:
            p.grad = torch.zeros_like(p)
        return ps, optim.AdamW(ps, lr=1e-2, bits=bits, capturable=True)
    (pa, a), (pb, b) = build(), build()
    g = torch.Generator().manual_seed(3)

    def fill():
        for x, y in zip(pa, pb):
            t = torch.randn(x.shape, generator=g).to(dev)
            x.grad.copy_(t)
            y.grad.copy_(t)
    fill()
    a.step()
    b.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step()
    for k in range(4):
        fill()
        a.step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(pa, pb)), k
    assert float(b.state[pb[0]]["step"]) == 5.0


def test_elements_past_32_bits(dev):
    n = (1 << 31) + 300
    p, g = torch.zeros(n, dtype=BF, device=dev), torch.zeros(n, dtype=BF, device=dev)
    s = [optim.empty_state8(p) for _ in range(2)]
    g[-5:] = 1
    optim.adamw_step([p], [g], [s[0]], [s[1]], step=1, lr=0.5, weight_decay=0.0)
    assert (p[-5:] == -0.5).all() and not p[:-5].any()  # the first step is lr, rounded exactly to bf16
