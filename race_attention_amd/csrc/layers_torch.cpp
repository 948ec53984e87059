// layers_torch.cpp -- the calls of race_attention_amd.norm, fp8 and optim as C++ over
// the C ABI, with C++ autograd functions, as race_torch.cpp has those of the attention.
//
// A norm of a few rows or a token's linear layer is 5 us of kernel; the Python path to it
// takes 15, with autograd 130, and an AdamW step over 90 tensors 200.  These functions
// take ordinary calls (plain tensors on the current device, types and shapes that agree);
// for everything else they return None and the Python path makes the call or raises.
#include "race_torch.h"

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <vector>

namespace {

#define LAYER_FNS(X)                                                                                               \
    X(race_rms_norm) X(race_rms_norm_codes) X(race_rms_norm_bwd_workspace_bytes) X(race_rms_norm_bwd)              \
    X(race_quantize_workspace_bytes) X(race_quantize) X(race_block_matmul_workspace_bytes) X(race_block_matmul)   \
    X(race_block_linear_rows) X(race_block_linear_workspace_bytes) X(race_block_linear) X(race_adamw)              \
    X(race_last_error)
struct Layers {
#define X(f) decltype(&::f) f = nullptr;
    LAYER_FNS(X)
#undef X
} lib;

// A status that is an error: in a forward call the Python path makes the call again and raises it
// (NotTaken), the engine's thread raises it itself.
struct Status : NotTaken {
    const char *what;
    int rc;
    std::string text;
};
void check(const char *what, int rc) {
    if (rc != RACE_OK) throw Status{{}, what, rc, lib.race_last_error()};
}
template <typename F> variable_list backward_of(F &&f) {
    try {
        at::NoGradGuard ng;
        return f();
    } catch (const Status &s) {
        raise_race_error(s.what, s.rc, s.text.c_str());
    }
}

constexpr int64_t BLOCK = 128;
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool typed(const Tensor &x) { return x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat; }
int32_t dtype_of(at::ScalarType t) { return t == at::kBFloat16 ? RACE_DTYPE_BF16 : RACE_DTYPE_F32; }
int32_t dtype_of(const Tensor &x) { return dtype_of(x.scalar_type()); }

// x [..., D] as rows of contiguous columns (a view where the strides allow one)
Tensor rows2d(const Tensor &x) {
    Tensor y = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    return y.size(1) > 1 && y.stride(1) != 1 ? y.contiguous() : y;
}
int64_t row_stride(const Tensor &x) { return x.size(0) > 1 ? x.stride(0) : std::max(x.stride(0), x.size(1)); }
Tensor f32(const Tensor &x) { return x.detach().to(at::kFloat).contiguous(); }

// an argument: a tensor itself, not a subclass, plain and on the current device
bool usable_arg(py::handle h, Tensor &out) {
    if (!is_tensor(h)) return false;
    out = THPVariable_Unpack(h.ptr());
    return plain(out) && out.device().index() == c10::hip::current_device();
}
bool optional_arg(py::handle h, Tensor &out) { return h.is_none() || usable_arg(h, out); }

// Gradients that cannot be differentiated again say so, as torch's once_differentiable does.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", (int64_t)grads.size());
    for (Tensor &g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    return (*error)(std::move(grads));
}

// ------------------------------------------------------------ norm
struct Normed {
    Tensor y, h, rstd;
};
race_norm_desc norm_desc(const Tensor &x2, const Tensor &r2, double eps) {
    race_norm_desc d{};
    d.rows = x2.size(0);
    d.D = x2.size(1);
    d.x_stride = row_stride(x2);
    d.dtype = dtype_of(x2);
    d.r_dtype = r2.defined() ? dtype_of(r2) : d.dtype;
    if (r2.defined()) d.r_stride = row_stride(r2);
    d.y_stride = d.h_stride = d.D;
    d.eps = (float)eps;
    return d;
}
Normed norm_forward(const Tensor &x, const Tensor &w, const Tensor &residual, double eps, bool want_rstd) {
    const Tensor x2 = rows2d(x), r2 = residual.defined() ? rows2d(residual) : residual, w32 = f32(w);
    Normed n;
    n.y = at::empty(x.sizes(), x.options());
    if (residual.defined()) n.h = at::empty(x.sizes(), residual.options());
    if (want_rstd) n.rstd = fp32({x2.size(0)}, x);
    const race_norm_desc d = norm_desc(x2, r2, eps);
    if (lib.race_rms_norm(&d, ptr(x2), r2.defined() ? ptr(r2) : nullptr, fptr(w32), ptr(n.y),
                          n.h.defined() ? ptr(n.h) : nullptr, fptr(n.rstd), stream_of(x)) != RACE_OK)
        throw NotTaken();
    return n;
}

struct Norm : torch::autograd::Function<Norm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &w,
                                 const std::optional<Tensor> &oresidual, double eps) {
        const Tensor residual = oresidual.value_or(Tensor());
        const Normed n = norm_forward(x, w, residual, eps, true);
        ctx->set_materialize_grads(false);
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["type"] = (int64_t)x.scalar_type();
        ctx->saved_data["residual"] = residual.defined();  // (an absent one is no edge)
        // the sum as y used it: an fp32 h holds it, a bf16 one is rounded
        if (!n.h.defined()) ctx->save_for_backward({Tensor(), x, w, n.rstd});
        else if (n.h.scalar_type() == at::kFloat) ctx->save_for_backward({Tensor(), n.h, w, n.rstd});
        else ctx->save_for_backward({x, residual, w, n.rstd});
        return n.h.defined() ? variable_list{n.y, n.h} : variable_list{n.y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        Tensor dy = grads[0], dh = grads.size() > 1 ? grads[1] : Tensor();
        if (!dy.defined() && !dh.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        return once(backward_of([&]() -> variable_list {
            const Tensor x2 = saved[0].defined() ? rows2d(saved[0]) : Tensor(), r = saved[1], r2 = rows2d(r), &w = saved[2];
            const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
            const Tensor dy2 = rows2d(dy.defined() ? dy.to(type) : at::zeros(r.sizes(), r.options().dtype(type)));
            const Tensor dh2 = dh.defined() ? rows2d(dh.to(r.scalar_type())) : Tensor();
            const Tensor w32 = f32(w);
            const Tensor dx = at::empty(r.sizes(), r.options().dtype(type));
            const Tensor dr = r.scalar_type() == type ? dx : at::empty(r.sizes(), r.options());
            Tensor dw = fp32({w.size(0)}, r);
            race_norm_desc d{};
            d.rows = r2.size(0);
            d.D = r2.size(1);
            d.x_stride = x2.defined() ? row_stride(x2) : 0;
            d.r_stride = row_stride(r2);
            d.dy_stride = dy2.size(0) > 1 ? dy2.stride(0) : d.D;
            d.dh_stride = dh2.defined() && dh2.size(0) > 1 ? dh2.stride(0) : d.D;
            d.dx_stride = d.dr_stride = d.D;
            d.dtype = dtype_of(type);
            d.r_dtype = dtype_of(r);
            d.eps = (float)ctx->saved_data["eps"].toDouble();
            const Tensor ws = bytes(lib.race_rms_norm_bwd_workspace_bytes(&d), r);
            check("race_rms_norm_bwd",
                  lib.race_rms_norm_bwd(&d, x2.defined() ? ptr(x2) : nullptr, ptr(r2), fptr(w32), fptr(saved[3]), ptr(dy2),
                                        dh2.defined() ? ptr(dh2) : nullptr, ptr(dx), dr.is_same(dx) ? nullptr : ptr(dr),
                                        fptr(dw), ptr(ws), (size_t)ws.numel(), stream_of(r)));
            return {ctx->needs_input_grad(0) ? dx : Tensor(),
                    ctx->needs_input_grad(1) ? dw.to(w.scalar_type()) : Tensor(),
                    ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(2) ? dr : Tensor(), Tensor()};
        }));
    }
};

// x, weight and residual of a norm, or false
bool norm_args(py::handle hx, py::handle hw, py::handle hr, Tensor &x, Tensor &w, Tensor &r) {
    if (redirected() || !usable_arg(hx, x) || !usable_arg(hw, w) || !optional_arg(hr, r)) return false;
    if (!typed(x) || x.dim() < 1 || x.numel() == 0 || w.dim() != 1 || w.size(0) != x.size(-1) ||
        !at::isFloatingType(w.scalar_type()))
        return false;
    return !r.defined() || (r.sizes() == x.sizes() && typed(r) &&
                            (r.scalar_type() == x.scalar_type() || r.scalar_type() == at::kFloat));
}
bool wants_grad(std::initializer_list<const Tensor *> xs) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor *x : xs)
        if (x->defined() && x->requires_grad()) return true;
    return false;
}
std::optional<Tensor> given(const Tensor &x) { return x.defined() ? std::optional<Tensor>(x) : std::nullopt; }

py::object rms_norm(py::handle hx, py::handle hw, py::handle hr, double eps) {
    Tensor x, w, r;
    if (!norm_args(hx, hw, hr, x, w, r)) return py::none();
    try {
        variable_list out;
        {
            py::gil_scoped_release nogil;
            if (wants_grad({&x, &w, &r})) {
                out = Norm::apply(x, w, given(r), eps);
            } else {
                at::NoGradGuard ng;
                const Normed n = norm_forward(x, w, r, eps, false);
                out = n.h.defined() ? variable_list{n.y, n.h} : variable_list{n.y};
            }
        }
        return out.size() == 1 ? py::cast(out[0]) : py::object(py::make_tuple(out[0], out[1]));
    } catch (const NotTaken &) {
        return py::none();
    }
}

// ------------------------------------------------------------ 8-bit blocks
struct Blocks {
    Tensor codes, scale;  // rows
    int32_t block_rows = 1;
    race_blocks desc() const {
        race_blocks b{};
        b.codes = codes.data_ptr();
        b.scale = scale.data_ptr();
        b.rows = codes.size(0);
        b.cols = codes.size(1);
        b.ld = row_stride(codes);
        b.scale_ld = row_stride(scale);
        b.block_rows = block_rows;
        return b;
    }
};
// blocks for the kernels to write: rows of whole 16-byte pieces
Blocks empty_blocks(int64_t rows, int64_t cols, int64_t block_rows, const Tensor &like) {
    const int64_t ld = ceil_div(cols, 16) * 16;
    Blocks b;
    b.codes = at::empty({rows, ld}, like.options().dtype(at::kFloat8_e4m3fn));
    if (ld != cols) b.codes = b.codes.narrow(1, 0, cols);
    b.scale = at::empty({ceil_div(rows, block_rows), ceil_div(cols, BLOCK)}, like.options().dtype(at::kFloat8_e8m0fnu));
    b.block_rows = (int32_t)block_rows;
    return b;
}
struct Quantized {
    Blocks y, t;
    Tensor sums;
};
Quantized quantize(const Tensor &x2, int64_t block_rows, bool want, bool want_t, bool want_sums) {
    const int64_t R = x2.size(0), C = x2.size(1);
    Quantized q;
    race_blocks y{}, t{};
    if (want) y = (q.y = empty_blocks(R, C, block_rows, x2)).desc();
    if (want_t) t = (q.t = empty_blocks(C, R, block_rows, x2)).desc();
    Tensor ws;
    if (want_sums) {
        q.sums = fp32({C}, x2);
        ws = bytes(lib.race_quantize_workspace_bytes(R, C), x2);
    }
    check("race_quantize", lib.race_quantize(ptr(x2), dtype_of(x2), R, C, row_stride(x2), want ? &y : nullptr,
                                             want_t ? &t : nullptr, fptr(q.sums), ws.defined() ? ptr(ws) : nullptr,
                                             ws.defined() ? (size_t)ws.numel() : 0, stream_of(x2)));
    return q;
}
Tensor product(const Blocks &a, const Blocks &b, at::IntArrayRef shape, const Tensor &bias, at::ScalarType type) {
    const Tensor out = at::empty(shape, a.codes.options().dtype(type));
    const race_blocks da = a.desc(), db = b.desc();
    const size_t n = lib.race_block_matmul_workspace_bytes(&da, &db, dtype_of(type));
    const Tensor ws = n ? bytes(n, out) : Tensor();
    check("race_block_matmul", lib.race_block_matmul(&da, &db, fptr(bias), ptr(out), dtype_of(type), db.rows,
                                                     n ? ptr(ws) : nullptr, n, stream_of(out)));
    return out;
}
Tensor product_few(const Tensor &x2, const Blocks &b, at::IntArrayRef shape, const Tensor &bias, at::ScalarType type) {
    const Tensor out = at::empty(shape, x2.options().dtype(type));
    const race_blocks db = b.desc();
    const size_t n = lib.race_block_linear_workspace_bytes(x2.size(0), &db, dtype_of(type));
    const Tensor ws = n ? bytes(n, out) : Tensor();
    check("race_block_linear",
          lib.race_block_linear(ptr(x2), dtype_of(x2), x2.size(0), row_stride(x2), &db, fptr(bias), ptr(out),
                                dtype_of(type), db.rows, n ? ptr(ws) : nullptr, n, stream_of(out)));
    return out;
}
std::vector<int64_t> out_shape(const Tensor &x, int64_t N) {
    std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
    s.back() = N;
    return s;
}

struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const std::optional<Tensor> &obias,
                          int64_t type) {
        const Tensor bias = obias.value_or(Tensor());
        // (an absent bias is no edge: its gradient is asked for by its own flag)
        const bool need_x = x.requires_grad(), need_w = w.requires_grad();
        const Tensor x2 = rows2d(x), b = bias.defined() ? f32(bias) : Tensor();
        const int64_t N = w.size(0), R = x2.size(0);
        const Quantized qw = quantize(rows2d(w), BLOCK, true, need_x, false);
        Quantized qx;
        Tensor y;
        if (R <= lib.race_block_linear_rows()) {
            if (need_w) qx = quantize(x2, 1, false, true, false);
            y = product_few(x2, qw.y, out_shape(x, N), b, (at::ScalarType)type);
        } else {
            qx = quantize(x2, 1, true, need_w, false);
            y = product(qx.y, qw.y, out_shape(x, N), b, (at::ScalarType)type);
        }
        ctx->save_for_backward({qx.t.codes, qx.t.scale, qw.t.codes, qw.t.scale});
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["x"] = (int64_t)x.scalar_type();
        ctx->saved_data["w"] = (int64_t)w.scalar_type();
        ctx->saved_data["need_x"] = need_x;
        ctx->saved_data["need_w"] = need_w;
        ctx->saved_data["b"] = bias.defined() && bias.requires_grad() ? (int64_t)bias.scalar_type() : (int64_t)-1;
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        return once(backward_of([&]() -> variable_list {
            auto is = [&](const char *k) { return ctx->saved_data[k].toInt(); };
            const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
            const bool need_x = ctx->saved_data["need_x"].toBool(), need_w = ctx->saved_data["need_w"].toBool();
            const int64_t bt = is("b");
            const Tensor dy2 = rows2d(grads[0]);
            const Quantized q = quantize(dy2, 1, need_x || !need_w, need_w, bt >= 0);
            Tensor dx, dw;
            if (need_x) dx = product(q.y, Blocks{saved[2], saved[3], (int32_t)BLOCK}, shape, Tensor(), (at::ScalarType)is("x"));
            if (need_w)
                dw = product(q.t, Blocks{saved[0], saved[1], 1}, {dy2.size(1), shape.back()}, Tensor(),
                             (at::ScalarType)is("w"));
            return {dx, dw, bt >= 0 ? q.sums.to((at::ScalarType)bt) : Tensor(), Tensor()};
        }));
    }
};

// codes and scales of a matrix [N, K] in blocks, or false
bool block_args(py::handle hc, py::handle hs, int64_t block_rows, Blocks &b, bool matrix) {
    if (!usable_arg(hc, b.codes) || !usable_arg(hs, b.scale)) return false;
    const Tensor &c = b.codes, &s = b.scale;
    if ((c.scalar_type() != at::kFloat8_e4m3fn && c.scalar_type() != at::kByte) ||
        (s.scalar_type() != at::kFloat8_e8m0fnu && s.scalar_type() != at::kByte))
        return false;
    if ((block_rows != 1 && block_rows != BLOCK) || c.dim() < 1 || ((matrix || block_rows == BLOCK) && c.dim() != 2) ||
        c.numel() == 0 || s.dim() != c.dim())
        return false;
    for (int64_t i = 0; i + 1 < c.dim(); ++i)
        if (s.size(i) != (block_rows == 1 ? c.size(i) : ceil_div(c.size(i), BLOCK))) return false;
    if (s.size(-1) != ceil_div(c.size(-1), BLOCK)) return false;
    b.block_rows = (int32_t)block_rows;
    return true;
}
bool bias_arg(py::handle h, int64_t N, Tensor &bias) {
    return optional_arg(h, bias) && (!bias.defined() || (bias.dim() == 1 && bias.size(0) == N &&
                                                         at::isFloatingType(bias.scalar_type())));
}
// f()'s tensor without the interpreter's lock, or None where its call was not taken
template <typename F> py::object taken(F &&f) {
    try {
        Tensor out;
        {
            py::gil_scoped_release nogil;
            out = f();
        }
        return py::cast(out);
    } catch (const NotTaken &) {
        return py::none();
    }
}
at::ScalarType type_of(bool fp32_out) { return fp32_out ? at::kFloat : at::kBFloat16; }

py::object matmul(py::handle ac, py::handle as, int64_t ar, py::handle bc, py::handle bs, int64_t br, py::handle hbias,
                  bool fp32_out) {
    Blocks a, b;
    Tensor bias;
    if (redirected() || !block_args(ac, as, ar, a, false) || !block_args(bc, bs, br, b, true) ||
        a.codes.size(-1) != b.codes.size(1) || !bias_arg(hbias, b.codes.size(0), bias))
        return py::none();
    return taken([&]() -> Tensor {
        at::NoGradGuard ng;
        const auto shape = out_shape(a.codes, b.codes.size(0));
        a.codes = rows2d(a.codes);
        a.scale = rows2d(a.scale);
        b.codes = rows2d(b.codes);
        b.scale = rows2d(b.scale);
        return product(a, b, shape, bias.defined() ? f32(bias) : bias, type_of(fp32_out));
    });
}

// weight: a tensor (hs None), or codes and scales of 128 x 128 or 1 x 128 blocks
py::object linear(py::handle hx, py::handle hw, py::handle hs, int64_t block_rows, py::handle hbias, bool fp32_out) {
    Tensor x, w, bias;
    Blocks b;
    const bool frozen = !hs.is_none();
    if (redirected() || !usable_arg(hx, x) || !typed(x) || x.dim() < 1 || x.numel() == 0) return py::none();
    if (frozen) {
        if (!block_args(hw, hs, block_rows, b, true)) return py::none();
        w = b.codes;
    } else if (!usable_arg(hw, w) || !typed(w) || w.dim() != 2 || w.numel() == 0) {
        return py::none();
    }
    if (x.size(-1) != w.size(1) || !bias_arg(hbias, w.size(0), bias)) return py::none();
    const int64_t N = w.size(0), R = x.numel() / x.size(-1);
    const bool grad = frozen ? wants_grad({&x, &bias}) : wants_grad({&x, &w, &bias});
    if (grad && (frozen || R > ((int64_t)1 << 22) - 16)) return py::none();
    const at::ScalarType type = type_of(fp32_out);
    return taken([&]() -> Tensor {
        if (grad) return Linear::apply(x, w, given(bias), (int64_t)type);
        at::NoGradGuard ng;
        const Tensor x2 = rows2d(x), b32 = bias.defined() ? f32(bias) : Tensor();
        if (frozen) {
            b.codes = rows2d(b.codes);
            b.scale = rows2d(b.scale);
        } else {
            b = quantize(rows2d(w), BLOCK, true, false, false).y;
        }
        if (R <= lib.race_block_linear_rows()) return product_few(x2, b, out_shape(x, N), b32, type);
        return product(quantize(x2, 1, true, false, false).y, b, out_shape(x, N), b32, type);
    });
}

// (codes, scale) or (codes, scale, h) of a norm in 8-bit blocks
py::object rms_norm_codes(py::handle hx, py::handle hw, py::handle hr, double eps) {
    Tensor x, w, r;
    if (!norm_args(hx, hw, hr, x, w, r) || wants_grad({&x, &w, &r}) || x.dim() != 2) return py::none();
    Blocks y;
    Tensor h;
    const py::object done = taken([&]() -> Tensor {
        at::NoGradGuard ng;
        const Tensor x2 = rows2d(x), r2 = r.defined() ? rows2d(r) : r, w32 = f32(w);
        y = empty_blocks(x.size(0), x.size(1), 1, x);
        if (r.defined()) h = at::empty(x.sizes(), r.options());
        const race_norm_desc d = norm_desc(x2, r2, eps);
        const race_blocks b = y.desc();
        check("race_rms_norm_codes",
              lib.race_rms_norm_codes(&d, ptr(x2), r2.defined() ? ptr(r2) : nullptr, fptr(w32), &b,
                                      h.defined() ? ptr(h) : nullptr, stream_of(x)));
        return y.codes;
    });
    if (done.is_none()) return done;
    return h.defined() ? py::object(py::make_tuple(y.codes, y.scale, h)) : py::object(py::make_tuple(y.codes, y.scale));
}

// ------------------------------------------------------------ AdamW
// Lists of tensors; with 8 bits the scales' lists too.  False: a call for the Python path.
bool adamw(py::list ps, py::list gs, py::list ms, py::list vs, py::list mscales, py::list vscales, bool eight,
           py::handle hstep, double lr, double b1, double b2, double eps, double wd, uint32_t seed) {
    const size_t n = ps.size();
    if (redirected() || !n || gs.size() != n || ms.size() != n || vs.size() != n ||
        (eight && (mscales.size() != n || vscales.size() != n)))
        return false;
    race_adamw_desc d{};
    Tensor step;
    if (PyFloat_Check(hstep.ptr()) || PyLong_Check(hstep.ptr())) {
        d.step = PyFloat_AsDouble(hstep.ptr());
    } else {
        if (!usable_arg(hstep, step) || step.scalar_type() != at::kFloat || step.numel() != 1) return false;
        d.step_ptr = fptr(step);
    }
    std::vector<race_adamw_tensor> table(n);
    std::vector<Tensor> written;
    written.reserve(n * (eight ? 5 : 3));
    std::vector<const void *> seen;
    seen.reserve(3 * n);
    Tensor p0, g0;
    for (size_t i = 0; i < n; ++i) {
        Tensor p, g, m, v, sm, sv;
        if (!usable_arg(ps[i], p) || !usable_arg(gs[i], g) || !usable_arg(ms[i], m) || !usable_arg(vs[i], v)) return false;
        if (!i) {
            p0 = p;
            g0 = g;
            if (!typed(p) || !typed(g)) return false;
        }
        if (p.scalar_type() != p0.scalar_type() || g.scalar_type() != g0.scalar_type()) return false;
        if (g.sizes() != p.sizes() || m.sizes() != p.sizes() || v.sizes() != p.sizes() || !p.is_contiguous() ||
            !g.is_contiguous() || !m.is_contiguous() || !v.is_contiguous())
            return false;
        auto state = [&](const Tensor &s) {
            return eight ? s.scalar_type() == at::kFloat8_e4m3fn || s.scalar_type() == at::kByte
                         : s.scalar_type() == at::kFloat;
        };
        if (!state(m) || !state(v)) return false;
        race_adamw_tensor &t = table[i];
        t.p = ptr(p);
        t.g = ptr(g);
        t.m = ptr(m);
        t.v = ptr(v);
        t.n = p.numel();
        if (eight) {
            if (!usable_arg(mscales[i], sm) || !usable_arg(vscales[i], sv)) return false;
            for (const Tensor &s : {sm, sv})
                if ((s.scalar_type() != at::kFloat8_e8m0fnu && s.scalar_type() != at::kByte) || s.dim() != 1 ||
                    s.size(0) != ceil_div(p.numel(), BLOCK) || !s.is_contiguous())
                    return false;
            t.m_scale = ptr(sm);
            t.v_scale = ptr(sv);
            written.push_back(sm);
            written.push_back(sv);
        }
        if (t.n) {
            seen.push_back(t.p);
            seen.push_back(t.m);
            seen.push_back(t.v);
        }
        written.push_back(std::move(p));
        written.push_back(std::move(m));
        written.push_back(std::move(v));
    }
    std::sort(seen.begin(), seen.end());
    if (std::adjacent_find(seen.begin(), seen.end()) != seen.end()) return false;  // twice in the lists: refused there
    d.lr = lr;
    d.beta_m = b1;
    d.beta_v = b2;
    d.eps = eps;
    d.weight_decay = wd;
    d.seed = seed;
    d.bits = eight ? 8 : 32;
    d.p_dtype = dtype_of(p0);
    d.g_dtype = dtype_of(g0);
    if (lib.race_adamw(&d, table.data(), (int64_t)n, stream_of(p0)) != RACE_OK) return false;
    for (const Tensor &t : written)
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();  // saved tensors notice
    return true;
}

}  // namespace

void bind_layers(void *library, const std::string &path) {
    Layers l;
#define X(f)                                                       \
    l.f = reinterpret_cast<decltype(&::f)>(dlsym(library, #f));    \
    TORCH_CHECK(l.f, path, " does not export ", #f);
    LAYER_FNS(X)
#undef X
    lib = l;
}

void add_layers(py::module_ &m) {
    m.def("rms_norm", &rms_norm);
    m.def("rms_norm_codes", &rms_norm_codes);
    m.def("matmul", &matmul);
    m.def("linear", &linear);
    m.def("adamw", &adamw);
}
