"""RACE blocks and models with root-mean-square norms, 8-bit linear layers and AdamW: the operators
as they run together."""
import copy

import pytest
import torch
import torch.nn.functional as F

from race_attention_amd import _lib, fp8, lm, norm, optim, race, vit

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["c++", "python"])
def path(request, monkeypatch):
    """Every test through the C++ calls and through the Python ones."""
    if request.param == "python":
        monkeypatch.setattr(_lib, "calls", lambda: None)
    else:
        assert _lib.calls() is not None


LM = dict(vocab_size=97, context_length=80, emb_dim=128, n_heads=2, n_layers=2, drop_rate=0.0, qkv_bias=True, K=2, L=2, M=1)
VIT = dict(img_size=12, patch_size=4, num_channels=1, embed_dim=128, num_heads=2, transformer_units=2, drop_rate=0.0,
           qkv_bias=False, K=2, L=2, M=1, num_classes=5)


def run(model, x, y):
    logits = model(x)
    loss = F.cross_entropy(logits.reshape(-1, logits.shape[-1]).float(), y.reshape(-1))
    return logits.detach(), dict(zip(dict(model.named_parameters()), torch.autograd.grad(loss, list(model.parameters()))))


class PlainNorm(torch.nn.Module):
    def __init__(self, m):
        super().__init__()
        self.weight, self.eps = m.weight, m.eps

    def forward(self, x, residual=None):
        h = x if residual is None else x + residual
        y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + self.eps) * self.weight
        return y if residual is None else (y, h)


def with_plain_norms(model):
    model = copy.deepcopy(model)
    for m in list(model.modules()):
        for name, c in list(m.named_children()):
            if isinstance(c, norm.RMSNorm):
                setattr(m, name, PlainNorm(c))
    return model


@pytest.mark.parametrize("kind", ["lm", "vit"])
def test_models_with_rms_norms(dev, kind):
    """fp32: the model with its fused norms against the same one with torch expressions in their place."""
    torch.manual_seed(0)
    if kind == "lm":
        model = lm.LMModel({**LM, "norm": "rms"}, device=dev).to(dev)
        x = torch.randint(0, 97, (2, 70), device=dev)
        y = torch.randint(0, 97, (2, 70), device=dev)
    else:
        model = vit.VisionTransformer({**VIT, "norm": "rms"}, device=dev).to(dev)
        x, y = torch.randn(3, 1, 12, 12, device=dev), torch.randint(0, 5, (3,), device=dev)
    a, ga = run(model, x, y)
    b, gb = run(with_plain_norms(model), x, y)
    # both are fp32 chains of some thousand roundings (2 blocks, rows of 128): 1e-4 is 1700 u
    assert (a - b).norm() <= 1e-4 * b.norm()
    for n in ga:
        assert (ga[n] - gb[n]).norm() <= 1e-3 * gb[n].norm() + 1e-7, n


def test_block_takes_a_tensor_or_a_branch_and_residual(dev):
    torch.manual_seed(1)
    b = race.RACEBlock({**LM, "norm": "rms"}, device=dev).to(dev)
    x = torch.randn(2, 40, 128, device=dev)
    with torch.no_grad():
        whole = b(x)
        branch, h = b((x, None))
        assert torch.equal(whole, branch + h)
        split = b((0.25 * x, 0.75 * x))
        assert (race.sum_of(split) - whole).norm() <= 1e-5 * whole.norm()


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_autocast_training_step_in_8_bits(dev, kind):
    """bf16 autocast over fp32 parameters, 8-bit linear layers, 8-bit AdamW: finite, near the model with torch's
    linear layers (e4m3 operands: 2^-4 a value, random signs), and every parameter moves."""
    torch.manual_seed(2)
    cfg = {**LM, "norm": kind}
    plain = lm.LMModel(cfg, device=dev).to(dev)
    eight = lm.LMModel({**cfg, "linear": "fp8"}, device=dev).to(dev)
    eight.load_state_dict(plain.state_dict())
    x, y = (torch.randint(0, 97, (2, 64), device=dev) for _ in range(2))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        a, ga = run(plain, x, y)
        b, gb = run(eight, x, y)
    assert a.dtype == b.dtype and torch.isfinite(b).all()
    assert (a - b).float().norm() <= 0.2 * a.float().norm()
    for n in ga:
        assert gb[n].dtype == ga[n].dtype and torch.isfinite(gb[n]).all(), n
    before = {n: p.detach().clone() for n, p in eight.named_parameters()}
    opt = optim.AdamW(eight.parameters(), lr=1e-3, bits=8)
    for n, p in eight.named_parameters():
        p.grad = gb[n]
    opt.step()
    for n, p in eight.named_parameters():
        assert torch.isfinite(p).all()
        assert not gb[n].any() or not torch.equal(p, before[n]), n


def test_served_path_norm_to_product(dev):
    """What a served block runs for a prompt and for a token: residual norm in 8 bits, then the product; equal to the
    same steps apart (the codes are the quantiser's of the unrounded y, so within one e4m3 rounding)."""
    torch.manual_seed(3)
    w, g = 0.05 * torch.randn(300, 256, device=dev), torch.rand(256, device=dev) + 0.5
    wq = fp8.quantize(w, 128)
    for rows in (1, 5, 200):
        x, r = (torch.randn(rows, 256, device=dev, dtype=torch.bfloat16) for _ in range(2))
        y8, h8 = norm.rms_norm_fp8(x, g, residual=r)
        y32, h = norm.rms_norm(x.float(), g, residual=r.float())
        want = fp8.matmul(fp8.quantize(y32), wq)
        got = fp8.matmul(y8, wq)
        assert torch.equal(h8, h.to(torch.bfloat16))
        # a code may round the other way where two fp32 chains differ: few, and by one e4m3 step of one value
        assert ((got - want).float().norm() <= 2e-3 * want.float().norm())


def test_frozen_model_serves(dev):
    """freeze() on every 8-bit layer: logits equal the unfrozen model's, under inference_mode and captured."""
    torch.manual_seed(4)
    model = lm.LMModel({**LM, "norm": "rms", "linear": "fp8"}, device=dev).to(dev).to(torch.bfloat16).eval()
    x = torch.randint(0, 97, (1, 70), device=dev)
    with torch.inference_mode():
        want = model(x)
        for m in model.modules():
            if isinstance(m, fp8.Linear):
                m.freeze()
        assert torch.equal(model(x), want)
