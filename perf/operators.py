"""The operators around RACE attention that this framework is measured on: what stands
before, in and after the linear layers of its blocks.

  norm      root-mean-square norm with the residual's addition, forward        norm.rms_norm
  norm_grad the same with its backward pass                                    norm.rms_norm
  norm_fp8  the same with an output in 8 bits, one scale for 128 columns       norm.rms_norm_fp8
  matmul    8-bit product of operands that hold a scale for each block of 128  fp8.matmul
  linear    a served linear layer: weights in 8 bits, activations quantised in the call
                                                                               fp8.linear
  train     a linear layer in 8 bits with its three gradients                  fp8.linear
  adamw     one AdamW step over many tensors, states in 32 or in 8 bits        optim.adamw_step

``run`` computes a case with elementary torch operations in 32 bits, or with the
framework's operators where ``own`` is true; ``exact`` is written apart from both, in
64 bits.  8-bit codes are e4m3, scales powers of two 2^s with s = ceil(log2(amax / 448))
of a block's finite values, so that x / 2^s is exact.
"""
import math

import torch

own = False

EPS = 1e-6
BETAS, LR, DECAY, ADAM_EPS, STEP = (0.9, 0.999), 6e-4, 0.1, 1e-8, 100
BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def _norm(name, op, dtype, rows, D, residual):
    case = {"op": op, "dtype": dtype, "rows": rows, "D": D, "residual": residual}
    return {"name": name, **case} if name else case


def _product(name, op, M, N, K, bias=False):
    case = {"op": op, "M": M, "N": N, "K": K, "bias": bias}
    return {"name": name, **case} if name else case


def _adamw(name, bits, grads, layers, d, vocab):
    case = {"op": "adamw", "bits": bits, "grads": grads, "layers": layers, "d": d, "vocab": vocab}
    return {"name": name, **case} if name else case


def listed():
    return [
        # one step of decoding for 8 sequences of the 768-wide decoder: latency
        _norm("norm_decode", "norm", "bf16", 8, 768, True),
        # the decoder's training batch, 8 x 8192 tokens: forward and backward
        _norm("norm_train", "norm_grad", "bf16", 65536, 768, True),
        # a long prompt of a 4096-wide model, output for an 8-bit linear layer
        _norm("norm_fp8_prompt", "norm_fp8", "bf16", 8192, 4096, True),
        # single precision, a row length that no vector or block divides
        _norm("norm_fp32_ragged", "norm_grad", "fp32", 4001, 1001, False),
        # one token through the decoder's joint query, key and value projection: latency
        _product("linear_token", "linear", 1, 2304, 768),
        # a batch of 16 single tokens through a 4096-wide projection: the weights' bytes
        _product("linear_batch16", "linear", 16, 4096, 4096, True),
        # a long prompt through a wide layer, both operands in 8 bits: the matrix cores
        _product("matmul_prompt", "matmul", 8192, 8192, 8192),
        # odd numbers of rows, columns and a contraction that no block divides
        _product("matmul_ragged", "matmul", 4001, 777, 1000),
        # the ViT encoder's first MLP layer in training: 64 x 785 tokens, 384 -> 1536
        _product("linear_train", "train", 50240, 1536, 384, True),
        # the ViT encoder's parameters, 6 layers, all in single precision
        _adamw("adamw_vit", 32, "fp32", 6, 384, 10),
        # the GPT decoder's parameters, 12 layers and two vocabulary matrices
        _adamw("adamw_gpt", 32, "fp32", 12, 768, 50257),
        # the same with states in 8 bits
        _adamw("adamw_gpt_8bit", 8, "fp32", 12, 768, 50257),
    ]


def _log(rng, lo, hi, multiple=1):
    """A whole number spread over [lo, hi] in its logarithm, a multiple in three of four draws."""
    x = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    m = multiple if rng.random() < 0.75 else 1
    return max(lo, min(hi, m * max(1, round(x / m))))


def draw(rng):
    op = rng.choice(["norm", "norm_grad", "norm_fp8", "matmul", "matmul", "linear", "linear", "train", "adamw", "adamw"])
    if op == "adamw":
        vocab = rng.choice([10, 1000, 50257])
        return _adamw(None, rng.choice([32, 8]), rng.choice(["fp32", "fp32", "bf16"]), rng.randint(1, 12),
                      _log(rng, 64, 768, 64), vocab)
    if op.startswith("norm"):
        D = _log(rng, 64, 8192, 64)
        rows = _log(rng, 1, min(65536, 50000000 // D), 8)
        dtype = "bf16" if op == "norm_fp8" or rng.random() < 0.7 else "fp32"
        return _norm(None, op, dtype, rows, D, rng.random() < 0.7)
    N, K = _log(rng, 64, 8192, 64), _log(rng, 64, 8192, 64)
    M = _log(rng, 1, 64) if op == "linear" and rng.random() < 0.7 else _log(rng, 64, 50000, 32)
    M = max(1, min(M, int(5e11 / (N * K)), int(2e8 / (N + K))))
    return _product(None, op, M, N, K, op != "matmul" and rng.random() < 0.5)


def _shapes(case):
    """The parameters of a model of ``layers`` blocks: the sizes of lm.LMModel and vit.VisionTransformer."""
    d, shapes = case["d"], [(case["vocab"], case["d"]), (785, case["d"])]
    for _ in range(case["layers"]):
        shapes += [(d, d)] * 4 + [(d,)] * 5 + [(4 * d, d), (4 * d,), (d, 4 * d), (d,)]
    return shapes + [(d,), (d,), (case["vocab"], d)]


# ------------------------------------------------------------------ inputs
def _inputs(case, seed):
    """What a case is computed from, from the seed alone: tensors on the GPU."""
    g = torch.Generator("cuda").manual_seed(1000003 * int(seed) + 29)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"].startswith("norm"):
        dt = DTYPES[case["dtype"]]
        R, D = case["rows"], case["D"]
        x = {"x": normal(R, D).to(dt), "w": (1 + 0.1 * normal(D)).to(torch.float32)}
        if case["residual"]:
            # a residual stream is larger than one block's output and has a few strong columns
            x["residual"] = (3 * normal(R, D) * (1 + 10 * (torch.rand(D, generator=g, device="cuda") < 0.01))).to(dt)
        if case["op"] == "norm_grad":
            x["dy"] = normal(R, D).to(dt)
            if case["residual"]:
                x["dh"] = normal(R, D).to(dt)
        return x
    if case["op"] == "adamw":
        sizes = [math.prod(s) for s in _shapes(case)]
        # the tensors stand one behind the other, each in whole blocks of 128
        n = sum(-(-s // BLOCK) * BLOCK for s in sizes)
        keep = torch.zeros(n, device="cuda")
        at = 0
        for s in sizes:
            keep[at:at + s] = 1
            at += -(-s // BLOCK) * BLOCK
        spread = torch.exp(normal(n // BLOCK, 1)).expand(-1, BLOCK).reshape(n)
        x = {"p": 0.02 * normal(n) * keep, "g": (1e-3 * spread * normal(n) * keep).to(DTYPES[case["grads"]])}
        m = 3e-4 * spread * normal(n) * keep
        root = 1e-3 * spread * (0.5 + normal(n).abs()) * keep
        if case["bits"] == 32:
            return {**x, "m": m, "v": root * root}
        x["m"], x["m_scale"] = _quantize(m.view(1, n))
        x["r"], x["r_scale"] = _quantize(root.view(1, n))
        return {k: t.view(-1) for k, t in x.items()}
    M, N, K = case["M"], case["N"], case["K"]
    # activations with a few strong channels, weights of a trained layer's size
    x = {"x": (normal(M, K) * (1 + 8 * (torch.rand(K, generator=g, device="cuda") < 0.02))).to(torch.bfloat16),
         "w": 0.02 * normal(N, K)}
    if case["bias"]:
        x["bias"] = 0.1 * normal(N)
    if case["op"] == "train":
        x["dy"] = (1e-3 * normal(M, N)).to(torch.bfloat16)
    else:
        x["w"], x["w_scale"] = _quantize(x["w"], 128)
        if case["op"] == "matmul":
            x["x"], x["x_scale"] = _quantize(x["x"].float())
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    if case["op"] in ("norm_grad", "train"):
        for name in ("x", "w", "residual", "bias"):
            if name in x:
                x[name].requires_grad_(True)
    if case["op"] == "adamw":
        # the model's tensors, as views of the buffers that hold them
        views, at, blocks = [], 0, 0
        for shape in _shapes(case):
            n = math.prod(shape)
            views.append([x[k][at:at + n].view(shape) for k in ("p", "g", "m", "v" if "v" in x else "r")])
            nb = -(-n // BLOCK)
            if case["bits"] == 8:
                views[-1] += [x[k][blocks:blocks + nb] for k in ("m_scale", "r_scale")]
            at, blocks = at + nb * BLOCK, blocks + nb
        x["tensors"] = [list(t) for t in zip(*views)]
    return {"case": case, **x}


# ------------------------------------------------------------------ the plain forms, in 32 bits
def _exponent(amax):
    """s of a block: the least with amax / 2^s <= 448; 0 for a block of zeros."""
    m, e = torch.frexp(amax)
    s = (e - 9 + (m > 0.875).to(e.dtype)).clamp(-127, 127)
    return torch.where(amax == 0, torch.zeros_like(s), s)


def _scaled(x, s):
    """x * 2^s for whole numbers s from -127 to 127, exactly (torch.ldexp's power is not exact)."""
    bits = torch.where(s > -127, (s.to(torch.int32) + 127) << 23, torch.full_like(s, 1 << 22, dtype=torch.int32))
    return x * bits.view(torch.float32)


def _blocks(x, rows):
    """x [R,C] fp32 -> its blocks [R/rows, rows, C/128, 128], padded with zeros."""
    R, C = x.shape
    x = torch.nn.functional.pad(x, (0, -C % BLOCK, 0, -R % rows))
    return x.view(-1, rows, x.shape[1] // BLOCK, BLOCK)


def _quantize(x, rows=1):
    """x [R,C] fp32 -> codes [R,C] e4m3, scales [R/rows, C/128] e8m0."""
    R, C = x.shape
    b = _blocks(x, rows)
    s = _exponent(torch.where(b.isfinite(), b.abs(), torch.zeros_like(b)).amax((1, 3)))
    codes = _scaled(b, -s[:, None, :, None]).to(torch.float8_e4m3fn)
    codes = codes.reshape(b.shape[0] * rows, -1)[:R, :C].contiguous()
    return codes, (s + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _values(codes, scale, rows=1):
    """What codes stand for, fp32 [R,C]."""
    R, C = codes.shape
    s = scale.view(torch.uint8).to(torch.int32) - 127
    s = s.repeat_interleave(rows, 0)[:R].repeat_interleave(BLOCK, 1)[:, :C]
    return _scaled(codes.float(), s)


def _rounded(x, rows=1):
    return _values(*_quantize(x, rows), rows)


def _plain_norm(state, grads):
    x, w = state["x"].detach().float(), state["w"].detach()
    h = x + state["residual"].detach().float() if "residual" in state else x
    rstd = torch.rsqrt((h * h).mean(-1, keepdim=True) + EPS)
    y = h * rstd * w
    out = {"y": y, "h": h} if "residual" in state else {"y": y}
    if grads:
        dy = state["dy"].float()
        gw = dy * w
        dx = rstd * (gw - h * rstd * rstd * (gw * h).mean(-1, keepdim=True))
        dx = dx + state["dh"].float() if "dh" in state else dx
        out.update(dx=dx, dw=(dy * h * rstd).sum(0))
        if "residual" in state:
            out["dresidual"] = dx
    return out


def _plain_adamw(state):
    eight = state["case"]["bits"] == 8
    b1, b2 = BETAS
    p, g = state["p"], state["g"].float()
    m = _values(state["m"][None], state["m_scale"][None])[0] if eight else state["m"]
    v = _values(state["r"][None], state["r_scale"][None])[0].square() if eight else state["v"]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    root = v.sqrt()
    p.mul_(1 - LR * DECAY).sub_(LR / (1 - b1 ** STEP) * m / (root / math.sqrt(1 - b2 ** STEP) + ADAM_EPS))
    if not eight:
        state["m"].copy_(m)
        state["v"].copy_(v)
        return {k: state[k] for k in ("p", "m", "v")}
    u = _bits(p.numel(), STEP)
    for name, t, r in (("m", m, u & 0xffff), ("r", root, u >> 16)):
        codes, scale = _stochastic(t, r.float() / 65536)
        state[name].copy_(codes)
        state[name + "_scale"].copy_(scale)
    return {k: state[k] for k in ("p", "m", "m_scale", "r", "r_scale")}


def _mix(x):
    """32 random-looking bits of each 32-bit whole number (two rounds of xor-shift and multiplication)."""
    x = ((x ^ (x >> 16)) * 0x7feb352d) & 0xffffffff
    x = ((x ^ (x >> 15)) * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def _bits(n, seed):
    """The random numbers of a step: one 32-bit number for each element's place in the buffers."""
    at = torch.arange(n, device="cuda")
    return _mix((at + _mix(torch.tensor(seed, device="cuda"))) & 0xffffffff)


def _stochastic(x, u):
    """x [n] fp32 to e4m3 with scales of 128 elements, rounded up with the probability of the remainder."""
    b = x.view(-1, BLOCK)
    s = _exponent(b.abs().amax(1))
    y = _scaled(b, -s[:, None]).view(-1)
    step = torch.frexp(y)[1].clamp_min(-5) - 4  # the spacing of e4m3 at y is 2^step
    q = _scaled(torch.floor(_scaled(y.abs(), -step) + u), step)
    return torch.copysign(q, y).to(torch.float8_e4m3fn), (s + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _plain(state):
    case = state["case"]
    op = case["op"]
    if op in ("norm", "norm_grad"):
        out = _plain_norm(state, op == "norm_grad")
        return {k: v if k == "dw" else v.to(state["x"].dtype) for k, v in out.items()}
    if op == "norm_fp8":
        out = _plain_norm(state, False)
        codes, scale = _quantize(out.pop("y"))
        return {"codes": codes, "scale": scale, **{k: v.to(state["x"].dtype) for k, v in out.items()}}
    if op == "adamw":
        return _plain_adamw(state)
    x, w = state["x"].detach(), state["w"].detach()
    if op == "train":
        x, dy = x.float(), state["dy"].float()
        wq = _rounded(w, 128)
        y = _rounded(x) @ wq.t()
        y = y + state["bias"].detach() if case["bias"] else y
        out = {"y": y.bfloat16(), "dx": (_rounded(dy) @ wq).bfloat16(),
               "dw": _rounded(dy.t()) @ _rounded(x.t()).t()}
        if case["bias"]:
            out["dbias"] = dy.sum(0)
        return out
    a = _values(x, state["x_scale"]) if op == "matmul" else _rounded(x.float())
    y = a @ _values(w, state["w_scale"], 128).t()
    y = y + state["bias"] if case["bias"] else y
    return {"y": y.bfloat16()}


# ------------------------------------------------------------------ one pass
def run(state):
    if not own:
        with torch.no_grad():
            return _plain(state)
    from race_attention_amd import fp8, norm, optim
    op = state["case"]["op"]
    if op.startswith("norm"):
        x, w, residual = state["x"], state["w"], state.get("residual")
        if op == "norm_fp8":
            y = norm.rms_norm_fp8(x, w, residual=residual, eps=EPS)
            y, h = y if residual is not None else (y, None)
            return {"codes": y.codes, "scale": y.scale, **({} if h is None else {"h": h})}
        y = norm.rms_norm(x, w, residual=residual, eps=EPS)
        y, h = y if residual is not None else (y, None)
        if op == "norm":
            return {"y": y} if h is None else {"y": y, "h": h}
        if h is None:
            dx, dw = torch.autograd.grad(y, (x, w), state["dy"])
            return {"y": y.detach(), "dx": dx, "dw": dw}
        dx, dw, dr = torch.autograd.grad((y, h), (x, w, residual), (state["dy"], state["dh"]))
        return {"y": y.detach(), "h": h.detach(), "dx": dx, "dw": dw, "dresidual": dr}
    if op == "adamw":
        p, g, m, v, *scales = state["tensors"]
        if scales:
            m, v = ([fp8.BlockFp8(*t) for t in zip(c, s)] for c, s in zip((m, v), scales))
        optim.adamw_step(p, g, m, v, step=STEP, lr=LR, betas=BETAS, eps=ADAM_EPS, weight_decay=DECAY, seed=STEP)
        return {k: state[k] for k in (("p", "m", "m_scale", "r", "r_scale") if scales else ("p", "m", "v"))}
    if op == "train":
        leaves = [state[k] for k in ("x", "w", "bias") if k in state]
        y = fp8.linear(state["x"], state["w"], state.get("bias"))
        grads = torch.autograd.grad(y, leaves, state["dy"])
        return {"y": y.detach(), **dict(zip(("dx", "dw", "dbias"), grads))}
    w = fp8.BlockFp8(state["w"], state["w_scale"], 128)
    if op == "linear":
        return {"y": fp8.linear(state["x"], w, state.get("bias"))}
    return {"y": fp8.matmul(fp8.BlockFp8(state["x"], state["x_scale"]), w)}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """Each input read once and each output written once; the products as 2 operations a multiply-add."""
    op = case["op"]
    if op == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        g = 2 if case["grads"] == "bf16" else 4
        state = 16 if case["bits"] == 32 else 4 + 4 / BLOCK
        return {"bytes": n * (8 + g + state), "flops": 14 * n}
    if op.startswith("norm"):
        n, e = case["rows"] * case["D"], 2 if case["dtype"] == "bf16" else 4
        extra = 2 if case["residual"] else 0  # residual in, sum out
        if op == "norm_fp8":
            return {"bytes": n * (e * (1 + extra) + 1 + 1 / BLOCK) + 4 * case["D"], "flops": 6 * n}
        if op == "norm":
            return {"bytes": n * e * (2 + extra) + 4 * case["D"], "flops": 5 * n}
        # backward: dy in, dx out, and for a residual the sum's gradient in and its own out
        return {"bytes": n * e * (4 + 2 * extra) + 8 * case["D"], "flops": 16 * n}
    M, N, K = case["M"], case["N"], case["K"]
    bias = 4 * N if case["bias"] else 0
    if op == "train":
        return {"bytes": 2 * (2 * M * K + 2 * M * N) + 8 * N * K + 2 * bias, "flops": 6 * M * N * K}
    a = M * K * (1 + 1 / BLOCK) if op == "matmul" else 2 * M * K
    return {"bytes": a + N * K + 2 * M * N + bias, "flops": 2 * M * N * K}


# ------------------------------------------------------------------ the same in 64 bits
def _exact_scale(b):
    """The powers of two of blocks [R, rows, C, 128]: the least one not under amax / 448."""
    amax = torch.nan_to_num(b, nan=0.0, posinf=0.0, neginf=0.0).abs().amax((1, 3), keepdim=True)
    s = torch.round(torch.log2(amax / 448))
    # the logarithm's own error decides nothing: amax is held against the powers of two around it
    s = torch.where(amax > 448 * torch.exp2(s), s + 1, torch.where(amax <= 448 * torch.exp2(s - 1), s - 1, s))
    return torch.where(amax > 0, torch.exp2(s.clamp(-127, 127)), torch.ones_like(s))


def _spacing(y):
    """The distance of e4m3 numbers around |y|: 3 bits behind the leading one, 2^-9 below 2^-6."""
    lead = torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6)))
    # log2 of a number just below a power of two may round up to it
    lead = torch.where(torch.exp2(lead) > y.abs().clamp_min(2.0 ** -6), lead - 1, lead)
    return torch.exp2(lead - 3)


def _exact_codes(x, rows=1):
    """x [R,C] fp64 -> (codes as numbers [R,C], scales [R/rows, C/128]); ties of the codes go to even."""
    R, C = x.shape
    full = torch.zeros(-(-R // rows) * rows, -(-C // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    full[:R, :C] = x
    b = full.view(-1, rows, full.shape[1] // BLOCK, BLOCK)
    scale = _exact_scale(b)
    y = b / scale
    step = _spacing(y)
    q = torch.round(y / step) * step
    return q.reshape(full.shape)[:R, :C], scale[:, 0, :, 0], (q * scale).reshape(full.shape)[:R, :C]


def _stored(codes, scale, rows=1):
    """fp64 values of stored codes [R,C]: each block of the padded matrix times its scale."""
    R, C = codes.shape
    full = torch.zeros(scale.shape[0] * rows, scale.shape[1] * BLOCK, dtype=torch.float64, device=codes.device)
    full[:R, :C] = codes.double()
    b = full.view(scale.shape[0], rows, scale.shape[1], BLOCK)
    return (b * scale.float().double()[:, None, :, None]).reshape(full.shape)[:R, :C]


def _exact_norm(x, grads):
    w = x["w"].double()
    h = x["x"].double()
    if "residual" in x:
        h = h + x["residual"].double()
    D = h.shape[1]
    norm = torch.sqrt(h.square().sum(1) / D + EPS)[:, None]
    unit = h / norm
    out = {"y": unit * w}
    if "residual" in x:
        out["h"] = h
    if grads:
        dy = x["dy"].double()
        gw = dy * w
        dx = (gw - unit * (gw * unit).sum(1, keepdim=True) / D) / norm
        if "dh" in x:
            dx = dx + x["dh"].double()
        out["dx"], out["dw"] = dx, (dy * unit).sum(0)
        if "residual" in x:
            out["dresidual"] = dx
    return out


def _exact_adamw(case, x):
    b1, b2 = BETAS
    p, g = x["p"].double(), x["g"].double()
    if case["bits"] == 8:
        m, v = (_stored(x[k][None], x[k + "_scale"][None])[0] for k in ("m", "r"))
        v = v * v
    else:
        m, v = x["m"].double(), x["v"].double()
    m = m + (1 - b1) * (g - m)
    v = v + (1 - b2) * (g * g - v)
    mean, square = m / (1 - b1 ** STEP), v / (1 - b2 ** STEP)
    p = p - LR * (DECAY * p + mean / (square.sqrt() + ADAM_EPS))
    if case["bits"] == 32:
        return {"p": p, "m": m, "v": v}
    out = {"p": p}
    bits = _bits(p.numel(), STEP)
    for name, t, u in (("m", m, bits % 65536), ("r", v.sqrt(), bits // 65536)):
        b = t.view(-1, 1, 1, BLOCK)
        scale = _exact_scale(b)
        y = (b / scale).reshape(-1)
        step = _spacing(y)
        out[name] = torch.sign(y) * torch.floor(y.abs() / step + u.double() / 65536) * step
        out[name + "_scale"] = scale.reshape(-1)
    return out


@torch.no_grad()
def exact(case, seed):
    x, op = _inputs(case, seed), case["op"]
    if op in ("norm", "norm_grad"):
        return _exact_norm(x, op == "norm_grad")
    if op == "norm_fp8":
        out = _exact_norm(x, False)
        codes, scale, _ = _exact_codes(out.pop("y"))
        return {"codes": codes, "scale": scale, **out}
    if op == "adamw":
        return _exact_adamw(case, x)
    if op == "train":
        a, w, dy = x["x"].double(), _exact_codes(x["w"].double(), 128)[2], x["dy"].double()
        out = {"y": _exact_codes(a)[2] @ w.t() + (x["bias"].double() if case["bias"] else 0),
               "dx": _exact_codes(dy)[2] @ w,
               "dw": _exact_codes(dy.t().contiguous())[2] @ _exact_codes(a.t().contiguous())[2].t()}
        if case["bias"]:
            out["dbias"] = dy.sum(0)
        return out
    a = _stored(x["x"], x["x_scale"]) if op == "matmul" else _exact_codes(x["x"].double())[2]
    y = a @ _stored(x["w"], x["w_scale"], 128).t()
    return {"y": y + x["bias"].double() if case["bias"] else y}
