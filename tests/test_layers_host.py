"""The operators around the attention on the CPU: descriptors, sizes and refusals
(checked on the host before any launch; no compute call is made here)."""
import ctypes

import pytest
import torch

from race_attention_amd import _lib, fp8, norm, optim, race, vit, lm

P = ctypes.c_void_p(4096)  # stands for a device pointer: the calls below end before any is used


def _norm_desc(**kw):
    d = _lib.NormDesc()
    d.rows, d.D = 8, 768
    for n in ("x_stride", "r_stride", "y_stride", "h_stride", "dy_stride", "dh_stride", "dx_stride", "dr_stride"):
        setattr(d, n, 768)
    d.dtype = d.r_dtype = _lib.RACE_DTYPE_BF16
    d.eps = 1e-6
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _blocks(rows=256, cols=512, **kw):
    b = _lib.Blocks()
    b.codes, b.scale, b.rows, b.cols = 4096, 4096, rows, cols
    b.ld, b.scale_ld, b.block_rows = -(-cols // 16) * 16, -(-cols // 128), 1
    for k, v in kw.items():
        setattr(b, k, v)
    return b


def test_struct_layouts_match_the_header():
    assert ctypes.sizeof(_lib.NormDesc) == 10 * 8 + 2 * 4 + 4 + 4
    assert ctypes.sizeof(_lib.Blocks) == 6 * 8 + 8
    assert ctypes.sizeof(_lib.AdamwTensor) == 7 * 8
    assert ctypes.sizeof(_lib.AdamwDesc) == 6 * 8 + 8 + 4 * 4 and _lib.AdamwDesc.seed.offset == 56


@pytest.mark.parametrize("kw,code,msg", [
    (dict(rows=0), -1, "rows and D"), (dict(D=0), -1, "rows and D"), (dict(dtype=2), -1, "dtype"),
    (dict(dtype=_lib.RACE_DTYPE_F32), -2, "bf16 residual"), (dict(eps=float("nan")), -1, "eps"),
    (dict(eps=-1.0), -1, "eps"), (dict(x_stride=-768), -1, "x row stride"), (dict(y_stride=700), -1, "y row stride"),
    (dict(h_stride=767), -1, "h row stride"), (dict(D=(1 << 30) + 1), -2, "columns"),
])
def test_norm_refusals(kw, code, msg):
    lib = _lib.load()
    d = _norm_desc(**kw)
    assert lib.race_rms_norm(ctypes.byref(d), P, P, P, P, P, P, None) == code and msg in _lib.last_error()


def test_norm_pointer_refusals():
    lib = _lib.load()
    d = _norm_desc()
    r = ctypes.byref(d)
    assert lib.race_rms_norm(None, P, P, P, P, P, P, None) == -1
    assert lib.race_rms_norm(r, None, P, P, P, P, P, None) == -1 and "x is NULL" in _lib.last_error()
    assert lib.race_rms_norm(r, P, P, P, P, None, P, None) == -1 and "together" in _lib.last_error()
    assert lib.race_rms_norm(r, P, None, P, P, P, P, None) == -1 and "together" in _lib.last_error()
    assert lib.race_rms_norm(r, ctypes.c_void_p(4097), P, P, P, P, P, None) == -1 and "aligned" in _lib.last_error()
    assert lib.race_rms_norm_bwd_workspace_bytes(r) == 2 * 768 * 4  # 8 rows: two workgroups of four
    assert lib.race_rms_norm_bwd(r, P, P, P, P, P, P, P, P, P, P, 2 * 768 * 4 - 1, None) == -3
    assert lib.race_rms_norm_bwd(r, P, P, P, P, P, P, P, P, P, None, 1 << 20, None) == -3
    b = _blocks(8, 768)
    assert lib.race_rms_norm_codes(r, P, P, P, ctypes.byref(_blocks(8, 767)), P, None) == -1
    assert lib.race_rms_norm_codes(r, P, P, P, ctypes.byref(_blocks(8, 768, block_rows=128)), P, None) == -1
    assert lib.race_rms_norm_codes(r, P, P, P, ctypes.byref(_blocks(8, 768, ld=770)), P, None) == -1
    assert lib.race_rms_norm_codes(r, P, None, P, ctypes.byref(b), P, None) == -1


@pytest.mark.parametrize("kw,msg", [
    (dict(rows=0), "rows and cols"), (dict(cols=0), "rows and cols"), (dict(ld=511), "row pitch"),
    (dict(scale_ld=3), "row pitch"), (dict(block_rows=64), "1 or 128"), (dict(codes=0), "NULL"), (dict(scale=0), "NULL"),
])
def test_block_refusals(kw, msg):
    lib = _lib.load()
    good, bad = _blocks(), _blocks(**kw)
    assert lib.race_block_matmul_workspace_bytes(ctypes.byref(good), ctypes.byref(bad), 1) == 0
    assert msg in _lib.last_error()
    rc = lib.race_block_matmul(ctypes.byref(bad), ctypes.byref(good), None, P, 1, 256, P, 1 << 30, None)
    assert rc == -1 and msg in _lib.last_error()
    rc = lib.race_quantize(P, 1, bad.rows, bad.cols, 512, ctypes.byref(bad), None, None, None, 0, None)
    assert rc == -1


def test_product_refusals():
    lib = _lib.load()
    a, b = _blocks(300, 512), _blocks(256, 384)
    r = ctypes.byref
    assert lib.race_block_matmul(r(a), r(b), None, P, 1, 256, None, 0, None) == -1 and "columns" in _lib.last_error()
    b = _blocks(256, 512)
    assert lib.race_block_matmul(r(a), r(b), None, P, 7, 256, P, 1 << 30, None) == -1 and "out_dtype" in _lib.last_error()
    assert lib.race_block_matmul(r(a), r(b), None, P, 1, 255, P, 1 << 30, None) == -1 and "out row" in _lib.last_error()
    assert lib.race_block_matmul(r(a), r(b), None, None, 1, 256, P, 1 << 30, None) == -1
    # an unaligned operand is copied: a workspace
    a = _blocks(300, 1001, ld=1001)
    b = _blocks(256, 1001, ld=1001)
    need = lib.race_block_matmul_workspace_bytes(r(a), r(b), 1)
    assert need >= (300 + 256) * 1008
    assert lib.race_block_matmul(r(a), r(b), None, P, 1, 256, P, need - 1, None) == -3
    assert lib.race_block_linear(P, 1, lib.race_block_linear_rows() + 1, 512, r(_blocks()), None, P, 1, 256, P, 1 << 30,
                                 None) == -2
    assert lib.race_block_linear(P, 3, 1, 512, r(_blocks()), None, P, 1, 256, P, 1 << 30, None) == -1
    assert lib.race_block_linear_workspace_bytes(0, r(_blocks()), 1) == 0
    wide = _blocks(256, 8192)  # rows of x are quantised into the workspace first
    need = lib.race_block_linear_workspace_bytes(16, r(wide), 1)
    assert need >= 16 * (8192 + 64)
    assert lib.race_block_linear(P, 1, 16, 8192, r(wide), None, P, 1, 256, None, 0, None) == -3
    assert lib.race_block_linear(P, 1, 16, 8192, r(wide), None, P, 1, 256, P, need - 1, None) == -3
    long = _blocks(300, 1 << 23)
    assert lib.race_block_matmul(r(long), r(long), None, P, 1, 300, P, 1 << 40, None) == -2 and "2^22" in _lib.last_error()


def test_quantizer_refusals():
    lib = _lib.load()
    r = ctypes.byref
    y, yt = _blocks(256, 512), _blocks(512, 256)
    assert lib.race_quantize(P, 1, 256, 512, 512, None, None, None, None, 0, None) == -1
    assert lib.race_quantize(P, 1, 256, 512, 512, r(yt), None, None, None, 0, None) == -1
    assert lib.race_quantize(P, 1, 256, 512, 512, r(y), r(y), None, None, 0, None) == -1
    assert lib.race_quantize(P, 1, 256, 512, 512, r(y), r(_blocks(512, 256, block_rows=128)), None, None, 0, None) == -1
    assert lib.race_quantize(P, 1, 256, 512, 512, r(_blocks(256, 512, ld=520)), None, None, None, 0, None) == -1
    assert lib.race_quantize(P, 1, 256, 512, 512, r(y), r(yt), P, None, 0, None) == -3
    assert lib.race_quantize_workspace_bytes(256, 512) == 2 * 512 * 4


def _adam(**kw):
    d = _lib.AdamwDesc()
    d.lr, d.beta_m, d.beta_v, d.eps, d.weight_decay, d.step = 1e-3, 0.9, 0.999, 1e-8, 0.1, 1
    d.bits, d.p_dtype, d.g_dtype = 32, 0, 0
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw", [dict(bits=16), dict(p_dtype=5), dict(beta_m=1.0), dict(beta_v=-0.1), dict(lr=float("nan")),
                                dict(eps=-1.0), dict(step=0), dict(weight_decay=float("inf")), dict(step_ptr=4098)])
def test_adamw_refusals(kw):
    lib = _lib.load()
    t = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(4096, 4096, 4096, 4096, 4096, 4096, 8))
    assert lib.race_adamw(ctypes.byref(_adam(**kw)), t, 1, None) == -1


def test_adamw_tensor_refusals():
    lib = _lib.load()
    for bad in (dict(p=None), dict(g=4098), dict(m=None), dict(v=4097), dict(n=-1)):
        t = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(4096, 4096, 4096, 4096, None, None, 8))
        for k, v in bad.items():
            setattr(t[0], k, v)
        assert lib.race_adamw(ctypes.byref(_adam()), t, 1, None) == -1, bad
    t = (_lib.AdamwTensor * 1)(_lib.AdamwTensor(4096, 4096, 4096, 4096, None, None, 8))
    assert lib.race_adamw(ctypes.byref(_adam(bits=8)), t, 1, None) == -1 and "scale" in _lib.last_error()
    assert lib.race_adamw(ctypes.byref(_adam()), None, 0, None) == 0  # no tensors: nothing to do
    assert lib.race_adamw(ctypes.byref(_adam()), None, 1, None) == -1


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 128), torch.ones(128)
    for call in (lambda: norm.rms_norm(x, w), lambda: norm.rms_norm_fp8(x, w), lambda: fp8.quantize(x),
                 lambda: fp8.linear(x, torch.zeros(8, 128)), lambda: norm.RMSNorm(128)(x), lambda: fp8.Linear(128, 8)(x),
                 lambda: optim.adamw_step([x], [x], [x], [x], step=1, lr=1e-3)):
        with pytest.raises(RuntimeError, match="ROCm GPUs only"):
            call()


def test_optimizer_arguments():
    p = torch.nn.Parameter(torch.zeros(3))
    for kw in (dict(bits=16), dict(betas=(1.0, 0.9)), dict(lr=-1.0), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            optim.AdamW([p], **kw)
    with pytest.raises(ValueError, match="lengths"):
        optim.adamw_step([p], [], [], [], step=1, lr=1.0)


def test_block_options():
    cfg = dict(emb_dim=128, n_heads=2, K=2, L=2, M=1, drop_rate=0.0, qkv_bias=False, vocab_size=11, context_length=8,
               n_layers=1)
    plain = race.RACEBlock(cfg)
    assert type(plain.norm1) is torch.nn.LayerNorm and type(plain.att.q) is torch.nn.Linear
    b = race.RACEBlock({**cfg, "norm": "rms", "linear": "fp8"})
    assert type(b.norm1) is norm.RMSNorm and type(b.att.o) is fp8.Linear and type(b.ff[0]) is fp8.Linear
    # the linear layers' parameters are nn.Linear's: checkpoints fit either
    fp = race.RACEBlock({**cfg, "linear": "fp8"})
    assert fp.load_state_dict(plain.state_dict()) is not None and list(fp.state_dict()) == list(plain.state_dict())
    v = vit.VisionTransformer(dict(img_size=8, patch_size=4, num_channels=1, embed_dim=128, num_heads=2,
                                   transformer_units=1, drop_rate=0.0, qkv_bias=False, K=2, L=2, M=1, num_classes=3,
                                   norm="rms", linear="fp8"))
    assert type(v.mlp_head[0]) is norm.RMSNorm and type(v.transformer_layers[0].att.out) is fp8.Linear
    assert type(lm.LMModel({**cfg, "norm": "rms"}).final_norm) is norm.RMSNorm
    for bad in (dict(norm="batch"), dict(linear="int8")):
        with pytest.raises(ValueError):
            race.RACEBlock({**cfg, **bad})


def test_dequantize_matches_the_definition():
    """BlockFp8.dequantize (torch expressions; shown here on the CPU through its parts)."""
    from blocks_ref import quantize, rounded
    g = torch.Generator().manual_seed(0)
    x = torch.randn(130, 300, generator=g) * torch.exp2(torch.randint(-30, 30, (130, 300), generator=g).float())
    for rows in (1, 128):
        q, s = quantize(x, rows)
        v = rounded(x, rows)
        # a code is at most half a step off: 2^-4 of the value, or 2^-10 of the scale below 2^-6
        e = torch.exp2(s).repeat_interleave(rows, 0)[:130].repeat_interleave(128, 1)[:, :300]
        assert ((v - x.double()).abs() <= x.double().abs() * 2 ** -4 + e * 2 ** -10).all()
        assert (q.abs() <= 448).all()
