"""AdamW over many tensors at once on the HIP kernels, states in 32 or in 8 bits.

``adamw_step`` updates lists of tensors in place, 48 tensors a launch; ``AdamW`` is the
torch optimizer over it.  With 8 bits the states m and sqrt(v) are e4m3 codes with a
power-of-two scale for each 128 neighbouring elements (2.02 bytes a parameter in place of
8), rounded stochastically from a hash of the seed and the element's place, so a step is
reproducible.  (Rounded to the nearest, a state that changes by less than half the distance
of neighbouring codes a step would never move.)
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from ._tensors import DTYPES, native, on_device, require_gpu, stream
from .fp8 import _CODES, _SCALES, BLOCK, BlockFp8


def empty_state8(p):
    """The 8-bit state of zeros for a tensor: codes of its shape, a scale for each 128 elements."""
    return BlockFp8(torch.zeros(p.shape, dtype=torch.float8_e4m3fn, device=p.device),
                    torch.full((-(-p.numel() // BLOCK),), 127, dtype=torch.uint8, device=p.device).view(torch.float8_e8m0fnu))


def _bad(i, what):
    return ValueError(f"tensor {i}: {what}")


def _check_tensor(i, p, g, m, v, eight, like):
    require_gpu(p, g)
    if p.dtype not in DTYPES or g.dtype not in DTYPES:
        raise TypeError(f"tensor {i}: unsupported dtypes {p.dtype}, {g.dtype} (bf16 or fp32)")
    if (p.dtype, g.dtype, p.device) != like:
        raise _bad(i, "the tensors of a call have one type and device, and so have the gradients")
    if g.shape != p.shape:
        raise _bad(i, f"gradient {tuple(g.shape)} of a parameter {tuple(p.shape)}")
    parts = [p, g]
    for s in (m, v):
        if eight:
            if not isinstance(s, BlockFp8) or s.codes.dtype not in _CODES or s.scale.dtype not in _SCALES:
                raise TypeError(f"tensor {i}: states are BlockFp8 of e4m3 codes and e8m0 scales")
            if s.codes.shape != p.shape or s.scale.shape != (-(-p.numel() // BLOCK),):
                raise _bad(i, "codes have the parameter's shape and a scale for each 128 elements")
            parts += [s.codes, s.scale]
        else:
            if not torch.is_tensor(s) or s.dtype != torch.float32:
                raise TypeError(f"tensor {i}: states are fp32 tensors")
            if s.shape != p.shape:
                raise _bad(i, f"state {tuple(s.shape)} of a parameter {tuple(p.shape)}")
            parts.append(s)
    for t in parts:
        if t.device != p.device:
            raise _bad(i, "parameter, gradient and states are on one device")
        if not t.is_contiguous():
            raise _bad(i, "parameter, gradient and states are contiguous")


def _adamw_native(params, grads, ms, vs, eight, step, lr, betas, eps, weight_decay, seed):
    """The C++ call, where it takes these arguments."""
    scales = [[], []]
    if eight:
        if not all(isinstance(s, BlockFp8) for s in ms + vs):
            return False
        scales = [[s.scale for s in group] for group in (ms, vs)]
        ms, vs = [s.codes for s in ms], [s.codes for s in vs]
    return bool(native(params[0], "adamw", params, grads, ms, vs, *scales, eight, step, float(lr), float(betas[0]),
                       float(betas[1]), float(eps), float(weight_decay), int(seed) & 0xffffffff))


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
               seed=0):
    """One AdamW step, in place, over lists of tensors of one type (parameters and gradients
    bf16 or fp32) on one device.

    States: fp32 tensors, or BlockFp8 of m and of sqrt(v) (``empty_state8``).  step: the step's
    number from 1, or a CUDA fp32 tensor of one element that holds it when the kernels run (for
    captured graphs; it is then added to seed).  seed: of the 8-bit states' rounding; take another one
    each step.

    A parameter or state that stands in the lists twice is refused; ones that overlap otherwise must
    not be given."""
    params, grads, ms, vs = list(params), list(grads), list(exp_avgs), list(exp_avg_sqs)
    if not len(params) == len(grads) == len(ms) == len(vs):
        raise ValueError("lists of different lengths")
    if not params:
        return
    eight = isinstance(ms[0], BlockFp8)
    if _adamw_native(params, grads, ms, vs, eight, step, lr, betas, eps, weight_decay, seed):
        return
    d = _lib.AdamwDesc()
    d.lr, (d.beta_m, d.beta_v), d.eps, d.weight_decay = float(lr), map(float, betas), float(eps), float(weight_decay)
    p0, g0 = params[0], grads[0]
    if torch.is_tensor(step):
        if not step.is_cuda:
            step = float(step)
        elif step.dtype != torch.float32 or step.numel() != 1 or step.device != p0.device:
            raise ValueError("a step tensor is fp32, of one element, on the parameters' device")
    if torch.is_tensor(step):
        d.step_ptr = step.data_ptr()
    else:
        d.step = float(step)
    d.seed, d.bits = int(seed) & 0xffffffff, 8 if eight else 32
    like = (p0.dtype, g0.dtype, p0.device)
    table = (_lib.AdamwTensor * len(params))()
    for i, (p, g, m, v) in enumerate(zip(params, grads, ms, vs)):
        _check_tensor(i, p, g, m, v, eight, like)
        t = table[i]
        t.p, t.g, t.n = p.data_ptr(), g.data_ptr(), p.numel()
        if eight:
            t.m, t.m_scale, t.v, t.v_scale = (x.data_ptr() for s in (m, v) for x in (s.codes, s.scale))
        else:
            t.m, t.v = m.data_ptr(), v.data_ptr()
    at = [x for t in table if t.n for x in (t.p, t.m, t.v)]
    if len(set(at)) < len(at):
        raise ValueError("a tensor stands in the lists twice")
    d.p_dtype, d.g_dtype = DTYPES[p0.dtype], DTYPES[g0.dtype]
    with on_device(p0):
        rc = _lib.load().race_adamw(ctypes.byref(d), table, len(params), stream(p0))
    _lib.check(rc, "race_adamw")
    # the kernels wrote behind autograd's back: a graph that saved these tensors has to notice
    written = params + ([x for s in ms + vs for x in (s.codes, s.scale)] if eight else ms + vs)
    torch.autograd.graph.increment_version([t for t in written if not t.is_inference()])


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's step (decoupled weight decay, no amsgrad) in one launch for up to 48
    tensors, with states in 32 or 8 bits.

    Parameters and gradients are bf16 or fp32 on the GPU.  state: "step" and, with 32 bits,
    "exp_avg" and "exp_avg_sq" in fp32; with 8 bits the codes and scales "exp_avg",
    "exp_avg_scale", "exp_avg_root", "exp_avg_root_scale" of m and sqrt(v).
    capturable=True keeps one step number for each parameter group on the GPU, so that a captured
    step() counts on when it is replayed (lr and the other numbers stay as captured)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, bits=32, seed=0,
                 capturable=False):
        if bits not in (8, 32):
            raise ValueError(f"states have 8 or 32 bits (got {bits})")
        if not (0 <= betas[0] < 1 and 0 <= betas[1] < 1) or not (lr >= 0 and eps >= 0 and weight_decay >= 0):
            raise ValueError(f"betas in [0, 1), lr, eps and weight_decay >= 0; got {betas}, {lr}, {eps}, {weight_decay}")
        self.bits, self.seed = bits, int(seed)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, capturable=capturable))

    def _init_state(self, p, group, state):
        if self.bits == 8:
            for name in ("exp_avg", "exp_avg_root"):
                s = empty_state8(p)
                state[name], state[name + "_scale"] = s.codes, s.scale
        else:
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        if group["capturable"]:
            others = [self.state[q]["step"] for q in group["params"] if "step" in self.state[q] and q.device == p.device]
            state["step"] = others[0] if others else torch.zeros((), dtype=torch.float32, device=p.device)
        else:
            state["step"] = 0

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for gi, group in enumerate(self.param_groups):
            calls = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW does not support sparse gradients")
                state = self.state[p]
                if not state:
                    self._init_state(p, group, state)
                if not group["capturable"]:
                    state["step"] += 1
                key = (p.dtype, p.grad.dtype, p.device, None if group["capturable"] else state["step"])
                calls.setdefault(key, []).append((p, state))
            if group["capturable"]:
                for t in {id(s["step"]): s["step"] for c in calls.values() for _, s in c}.values():
                    t += 1
            for ci, ((_, _, _, step), items) in enumerate(calls.items()):
                if self.bits == 8:
                    ms = [BlockFp8(s["exp_avg"], s["exp_avg_scale"]) for _, s in items]
                    vs = [BlockFp8(s["exp_avg_root"], s["exp_avg_root_scale"]) for _, s in items]
                else:
                    ms, vs = [s["exp_avg"] for _, s in items], [s["exp_avg_sq"] for _, s in items]
                t = items[0][1]["step"] if step is None else step
                # another sequence of random numbers for every step, group and call
                seed = self.seed + 0x9e3779b9 * (64 * gi + ci) + (0 if step is None else step)
                adamw_step([p for p, _ in items], [p.grad.contiguous() for p, _ in items], ms, vs, step=t,
                           lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                           seed=seed)
        return loss

    def load_state_dict(self, state_dict):
        """As torch's, but a state keeps the type that it was saved in (torch casts it to the parameter's)."""
        super().load_state_dict(state_dict)
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        want = {"exp_avg", "exp_avg_scale", "exp_avg_root", "exp_avg_root_scale"} if self.bits == 8 else {"exp_avg", "exp_avg_sq"}
        for i, p in zip(saved, params):
            if i not in state_dict["state"]:
                continue
            old = state_dict["state"][i]
            if set(old) != want | {"step"}:
                raise ValueError(f"a state of {sorted(old)} is not one of {self.bits} bits")
            for name in want:
                self.state[p][name] = old[name].to(p.device, copy=True)
        for group in self.param_groups:  # one step number a group and device, as _init_state gives
            shared = {}
            for p in group["params"]:
                if "step" not in self.state[p]:
                    continue
                step = float(self.state[p]["step"])
                if group["capturable"]:
                    if p.device not in shared:
                        shared[p.device] = torch.tensor(step, dtype=torch.float32, device=p.device)
                    self.state[p]["step"] = shared[p.device]
                else:
                    self.state[p]["step"] = int(step)
