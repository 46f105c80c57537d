// torch_binding_tokens.cpp -- the extension's operators on token rows, over the
// C ABI: RMS norm with the residual's addition, dropout, and the language model
// head with its cross entropy.
//   rms_norm(x, weight, eps, out_dtype?)                                      -> y
//   add_rms_norm(x, residual, weight, eps, dropout_p, seed, out_dtype?)       -> (y, h)
//   rms_norm_fp8(x, weight, eps, residual?)                                   -> (q, scale[, h])
//   dropout(x, dropout_p, seed)                                               -> y
//   linear_cross_entropy(x, weight, target, ignore_index, reduction)          -> loss
// All but rms_norm_fp8 are differentiable; their autograd nodes are C++ (from Python
// functions the forward and backward of a small call took 103 us of host time, 2 x 255
// rows of 771).  Arguments that do not fit raise ValueError.
// Tensors of any leading dimensions; a last
// dimension that is not of unit stride, or leading ones that are no single stride,
// are copied.  Outputs, state and workspaces come from the torch caching allocator
// on x's device; launches go to the current stream, with no synchronisation.
#include <torch/extension.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <cmath>
#include <cstring>
#include <memory>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/fa2_mi355x.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<Tensor> Maybe;

void *stream_of(const Tensor &t) {
    return reinterpret_cast<void *>(at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream());
}

void check_rc(int rc, const char *op) {
    TORCH_CHECK(rc == FA2_OK, op, ": ", fa2_status_string(rc), ": ", fa2_last_error());
}

int type_of(c10::ScalarType s, const char *op) {
    if (s == torch::kHalf) return FA2_F16;
    if (s == torch::kBFloat16) return FA2_BF16;
    TORCH_CHECK_VALUE(s == torch::kFloat, op, ": fp16, bf16 or fp32 tensors only");
    return FA2_F32;
}

void check_gpu(const Tensor &t, const Tensor &like, const char *op, const char *name) {
    TORCH_CHECK_VALUE(t.is_cuda() && t.device() == like.device(), op, ": ", name, " must be on x's GPU");
}

void check_rows(const Tensor &x, const char *op) {
    TORCH_CHECK_VALUE(x.is_cuda() && x.layout() == c10::kStrided && x.dim() >= 1, op, " takes GPU tensors (..., d)");
}

void check_p(double p, const char *op) {
    TORCH_CHECK_VALUE(p >= 0.0 && (float)p < 1.f, op, ": dropout probability ", p, " outside [0, 1)");
}

// A gradient that was asked for with create_graph: an error where it is differentiated.
variable_list once(variable_list grads, const char *op) {
    if (!at::GradMode::is_enabled()) return grads;
    auto err = std::make_shared<torch::autograd::DelayedError>(std::string(op) + " has no second derivative", (int64_t)grads.size());
    return (*err)(std::move(grads));
}

// t as [rows, last dimension] with unit stride in the last: a view where its
// strides allow one, else a copy.
Tensor as_rows(const Tensor &t) {
    const int64_t cols = t.size(-1);
    if (t.dim() == 2 && (t.stride(1) == 1 || cols == 1) && t.stride(0) >= 0) return t;
    if (t.is_contiguous()) return t.view({-1, cols});
    if (t.numel() == 0) return t.reshape({t.numel() / (cols ? cols : 1), cols});
    const Tensor r = t.reshape({-1, cols});
    return r.stride(1) == 1 || cols == 1 ? r : r.contiguous();
}

Tensor like(const Tensor &t, c10::ScalarType s) { return torch::empty(t.sizes(), t.options().dtype(s)); }

void check_norm(const Tensor &x, const Maybe &res, const Tensor &w, double eps, c10::ScalarType y_dtype, const char *op) {
    check_rows(x, op);
    const int64_t d = x.size(-1);
    TORCH_CHECK_VALUE(d >= 1 && d <= FA2_ROW_MAX, op, ": rows of 1 to ", FA2_ROW_MAX, " elements, got ", d);
    check_gpu(w, x, op, "weight");
    TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == d, op, ": weight must be (", d, ",)");
    type_of(x.scalar_type(), op);
    type_of(w.scalar_type(), op);
    if (res) {
        check_gpu(*res, x, op, "residual");
        TORCH_CHECK_VALUE(res->sizes() == x.sizes(), op, ": residual must have x's shape");
        TORCH_CHECK_VALUE(res->scalar_type() == x.scalar_type() || res->scalar_type() == torch::kFloat, op,
                          ": residual must be of x's type or fp32");
    }
    const bool fits = y_dtype == x.scalar_type() || y_dtype == torch::kFloat8_e4m3fn ||
                      (x.scalar_type() == torch::kFloat && (y_dtype == torch::kHalf || y_dtype == torch::kBFloat16));
    TORCH_CHECK_VALUE(fits, op, ": out_dtype must be x's type (fp16, bf16 or fp32 where x is fp32)");
    TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite((float)eps), op, ": eps ", eps, " is negative or not finite");
}

// y, h and rstd (keep) or scale of one call whose arguments have been checked.
struct NormOut {
    Tensor y, h, stat;
};

NormOut norm_run(const Tensor &x, const Maybe &res, const Tensor &w, double eps, double p, int64_t seed,
                 c10::ScalarType y_dtype, bool keep, const char *op) {
    const bool fp8 = y_dtype == torch::kFloat8_e4m3fn;
    at::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const Tensor xr = as_rows(x), wc = w.contiguous();
    const Tensor rr = res ? as_rows(*res) : Tensor();
    Tensor y = like(x, y_dtype), h = res ? like(x, res->scalar_type()) : Tensor(), stat;
    if (fp8) {
        std::vector<int64_t> shape = x.sizes().vec();
        shape.back() = 1;
        stat = torch::empty(shape, x.options().dtype(torch::kFloat));
    } else if (keep) {
        stat = torch::empty({xr.size(0)}, x.options().dtype(torch::kFloat));
    }
    fa2_rms_norm_params q;
    memset(&q, 0, sizeof(q));
    q.x = xr.data_ptr();
    q.x_stride = xr.stride(0);
    q.x_type = type_of(x.scalar_type(), op);
    q.weight = wc.data_ptr();
    q.weight_type = type_of(w.scalar_type(), op);
    if (res) {
        q.residual = rr.data_ptr();
        q.residual_stride = rr.stride(0);
        q.residual_type = type_of(res->scalar_type(), op);
        q.h = h.data_ptr();
    }
    q.y = y.data_ptr();
    q.y_type = fp8 ? FA2_E4M3 : type_of(y_dtype, op);
    (fp8 ? q.scale : q.rstd) = stat.defined() ? stat.data_ptr<float>() : nullptr;
    q.rows = xr.size(0);
    q.cols = (int32_t)x.size(-1);
    q.eps = (float)eps;
    q.dropout_p = (float)p;
    q.seed = (uint32_t)seed;
    check_rc(fa2_rms_norm_fwd(&q, stream_of(x)), op);
    return {y, h, stat};
}

struct NormGrads {
    Tensor dx, dres, dw;
};

NormGrads norm_grads(const Tensor &dy, const Maybe &dh, const Tensor &h, const Tensor &w, const Tensor &rstd,
                     at::ScalarType xs, double p, int64_t seed, bool want_dx, bool want_dres, bool want_dw) {
    const char *op = "rms_norm backward";
    at::hip::HIPGuardMasqueradingAsCUDA guard(h.device());
    const Tensor dyr = as_rows(dy), hr = as_rows(h), wc = w.contiguous();
    const Tensor dhr = dh ? as_rows(*dh) : Tensor();
    // Without dropout, and with one type, dx and dresidual are the same numbers.
    const bool same = p == 0.0 && xs == h.scalar_type() && want_dx && want_dres;
    Tensor dx = want_dx ? like(h, xs) : Tensor(), dres = same ? dx : want_dres ? like(h, h.scalar_type()) : Tensor();
    Tensor dw = want_dw ? torch::empty_like(wc) : Tensor(), ws;
    fa2_rms_norm_bwd_params q;
    memset(&q, 0, sizeof(q));
    q.rows = hr.size(0);
    q.cols = (int32_t)h.size(-1);
    q.dy = dyr.data_ptr();
    q.dy_stride = dyr.stride(0);
    q.y_type = type_of(dy.scalar_type(), op);
    if (dh) {
        q.dh = dhr.data_ptr();
        q.dh_stride = dhr.stride(0);
    }
    q.h = hr.data_ptr();
    q.h_stride = hr.stride(0);
    q.h_type = type_of(h.scalar_type(), op);
    q.x_type = type_of(xs, op);
    q.weight = wc.data_ptr();
    q.weight_type = type_of(w.scalar_type(), op);
    q.rstd = rstd.data_ptr<float>();
    q.dx = want_dx ? dx.data_ptr() : nullptr;
    q.dresidual = want_dres && !same ? dres.data_ptr() : nullptr;
    q.dropout_p = (float)p;
    q.seed = (uint32_t)seed;
    size_t bytes = 0;
    if (want_dw) {
        q.dweight = dw.data_ptr();
        bytes = fa2_rms_norm_bwd_workspace_bytes(q.rows, q.cols);
        ws = torch::empty({(int64_t)(bytes / 4)}, h.options().dtype(torch::kFloat));
    }
    check_rc(fa2_rms_norm_bwd(&q, bytes ? ws.data_ptr() : nullptr, bytes, stream_of(h)), op);
    return {dx, dres, dw};
}

Tensor drop_run(const Tensor &x, double p, int64_t seed) {
    const char *op = "dropout";
    at::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    Tensor y = like(x, x.scalar_type());
    fa2_dropout_params q;
    memset(&q, 0, sizeof(q));
    q.type = type_of(x.scalar_type(), op);
    if (x.numel() == 0) return y;
    const Tensor xr = as_rows(x);
    TORCH_CHECK_VALUE(x.size(-1) <= INT32_MAX, op, ": rows of less than 2^31 elements");
    q.x = xr.data_ptr();
    q.y = y.data_ptr();
    q.x_stride = xr.stride(0);
    q.rows = xr.size(0);
    q.cols = (int32_t)x.size(-1);
    q.dropout_p = (float)p;
    q.seed = (uint32_t)seed;
    check_rc(fa2_dropout(&q, stream_of(x)), op);
    return y;
}

// The gradient is the same call on dy with the same seed.
struct DropoutFn : torch::autograd::Function<DropoutFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, double p, int64_t seed) {
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        return drop_run(x, p, seed);
    }
    static variable_list backward(AutogradContext *ctx, variable_list dy) {
        return once({drop_run(dy[0], ctx->saved_data["p"].toDouble(), ctx->saved_data["seed"].toInt()), Tensor(), Tensor()}, "dropout");
    }
};

bool wants_grad(const Tensor &t) { return t.requires_grad() && at::GradMode::is_enabled(); }

Tensor dropout(const Tensor &x, double p, int64_t seed) {
    check_rows(x, "dropout");
    type_of(x.scalar_type(), "dropout");
    check_p(p, "dropout");
    if (p == 0.0) return x;
    return wants_grad(x) ? DropoutFn::apply(x, p, seed) : drop_run(x, p, seed);
}

// rms_norm (no residual: one output) and add_rms_norm (y, h).  Keeps h, which the
// residual stream holds anyway, and one fp32 a row; the dropout mask is formed again.
struct NormFn : torch::autograd::Function<NormFn> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Maybe &res, const Tensor &w, double eps, double p,
                                 int64_t seed, at::ScalarType y_dtype) {
        const NormOut o = norm_run(x, res, w, eps, p, seed, y_dtype, true, "rms_norm");
        ctx->save_for_backward({res ? o.h : x, w, o.stat});
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;
        ctx->saved_data["x"] = (int64_t)x.scalar_type();
        ctx->set_materialize_grads(false);
        return res ? variable_list{o.y, o.h} : variable_list{o.y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &h = saved[0], &w = saved[1];
        const double p = ctx->saved_data["p"].toDouble();
        const int64_t seed = ctx->saved_data["seed"].toInt();
        const at::ScalarType xs = (at::ScalarType)ctx->saved_data["x"].toInt();
        const Tensor &dy = g[0], dh = g.size() > 1 ? g[1] : Tensor();
        // Edges count the tensors among the inputs: x, residual (if any), weight.
        const bool res = g.size() > 1, want_x = ctx->needs_input_grad(0), want_r = res && ctx->needs_input_grad(1),
                   want_w = ctx->needs_input_grad(res ? 2 : 1);
        Tensor dx, dr, dw;
        if (dy.defined()) {
            const NormGrads o = norm_grads(dy, dh.defined() ? Maybe(dh) : Maybe(), h, w, saved[2], xs, p, seed, want_x, want_r, want_w);
            dx = o.dx;
            dr = o.dres;
            dw = o.dw;
        } else if (dh.defined()) {   // only the stream's gradient: no norm in it
            if (want_x) dx = (p > 0 ? drop_run(dh, p, seed) : dh).to(xs);
            if (want_r) dr = dh;
            if (want_w) dw = torch::zeros_like(w);
        }
        return once({dx, dr, dw, Tensor(), Tensor(), Tensor(), Tensor()}, "rms_norm");
    }
};

Tensor rms_norm(const Tensor &x, const Tensor &w, double eps, c10::optional<at::ScalarType> out_dtype) {
    const at::ScalarType y = out_dtype.value_or(x.scalar_type());
    check_norm(x, Maybe(), w, eps, y, "rms_norm");
    if (wants_grad(x) || wants_grad(w)) return NormFn::apply(x, Maybe(), w, eps, 0.0, (int64_t)0, y)[0];
    return norm_run(x, Maybe(), w, eps, 0.0, 0, y, false, "rms_norm").y;
}

std::tuple<Tensor, Tensor> add_rms_norm(const Tensor &x, const Maybe &res, const Tensor &w, double eps, double p, int64_t seed,
                                        c10::optional<at::ScalarType> out_dtype) {
    const at::ScalarType y = out_dtype.value_or(x.scalar_type());
    TORCH_CHECK_VALUE(res, "add_rms_norm: residual is missing (rms_norm needs none)");
    check_norm(x, res, w, eps, y, "add_rms_norm");
    check_p(p, "add_rms_norm");
    if (wants_grad(x) || wants_grad(*res) || wants_grad(w)) {
        const variable_list o = NormFn::apply(x, res, w, eps, p, seed, y);
        return {o[0], o[1]};
    }
    const NormOut o = norm_run(x, res, w, eps, p, seed, y, false, "add_rms_norm");
    return {o.y, o.h};
}

py::tuple rms_norm_fp8(const Tensor &x, const Tensor &w, double eps, const Maybe &res) {
    check_norm(x, res, w, eps, torch::kFloat8_e4m3fn, "rms_norm_fp8");
    TORCH_CHECK(!wants_grad(x) && !wants_grad(w) && !(res && wants_grad(*res)), "rms_norm_fp8 is inference-only (no backward)");
    const NormOut o = norm_run(x, res, w, eps, 0.0, 0, torch::kFloat8_e4m3fn, true, "rms_norm_fp8");
    return res ? py::make_tuple(o.y, o.stat, o.h) : py::make_tuple(o.y, o.stat);
}

// The weight as rows that the products read in place: 16-byte rows unless the
// hidden size is padded anyway.
Tensor weight_rows(const Tensor &w) {
    const bool rows = w.stride(1) == 1 && w.stride(0) >= w.size(1) && w.stride(0) < (1 << 22);
    const bool fits = reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0 && w.stride(0) % 8 == 0;
    if (rows && (fits || w.size(1) % 8 != 0)) return w;
    return w.clone(at::MemoryFormat::Contiguous);
}

Tensor bytes_of(size_t n, const Tensor &like) { return torch::empty({(int64_t)n}, like.options().dtype(torch::kByte)); }

void xent_common(fa2_xent_params &q, const Tensor &w, int64_t rows, int64_t ignore_index, int64_t reduction, const char *op) {
    memset(&q, 0, sizeof(q));
    q.type = type_of(w.scalar_type(), op);
    q.rows = rows;
    q.hidden = (int32_t)w.size(1);
    q.vocab = (int32_t)w.size(0);
    q.ignore_index = ignore_index;
    q.reduction = (int32_t)reduction;
}

void check_xent(const Tensor &x, const Tensor &w, const Tensor &target, const char *op) {
    check_rows(x, op);
    TORCH_CHECK_VALUE(x.scalar_type() == torch::kHalf || x.scalar_type() == torch::kBFloat16, op, ": fp16 or bf16 only");
    check_gpu(w, x, op, "weight");
    check_gpu(target, x, op, "target");
    TORCH_CHECK_VALUE(w.dim() == 2 && x.size(-1) == w.size(1) && x.scalar_type() == w.scalar_type(), op,
                      ": weight must be (V, d) with x's last dimension and type");
    TORCH_CHECK_VALUE(w.size(0) >= 1 && w.size(0) <= (1 << 24) && w.size(1) >= 1 && w.size(1) <= FA2_ROW_MAX &&
                          target.numel() <= (1 << 24),
                      op, ": d of 1 to ", FA2_ROW_MAX, ", V of 1 to 2^24, at most 2^24 tokens");
    TORCH_CHECK_VALUE(target.scalar_type() == torch::kLong && target.sizes() == x.sizes().slice(0, x.dim() - 1), op,
                      ": target must be int64 with x's leading dimensions");
}

struct XentOut {
    Tensor loss, state;
};

XentOut xent_run(const Tensor &x, const Tensor &w, const Tensor &target, int64_t ignore_index, int64_t reduction, bool keep) {
    const char *op = "linear_cross_entropy";
    at::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    const int64_t rows = target.numel();
    fa2_xent_params q;
    xent_common(q, w, rows, ignore_index, reduction, op);
    const Tensor xr = as_rows(x), wr = weight_rows(w), tc = target.contiguous();
    Tensor loss = reduction == FA2_REDUCE_NONE ? torch::empty(target.sizes(), x.options().dtype(torch::kFloat))
                                               : torch::empty({}, x.options().dtype(torch::kFloat));
    q.x = xr.data_ptr();
    q.x_stride = xr.stride(0);
    q.weight = wr.data_ptr();
    q.weight_stride = wr.stride(0);
    q.target = tc.data_ptr<int64_t>();
    q.loss = loss.data_ptr<float>();
    const size_t state_bytes = fa2_xent_state_bytes(rows, q.hidden);
    Tensor state;
    if (keep) {
        state = bytes_of(state_bytes, x);
        q.state = state.data_ptr();
        q.state_bytes = state_bytes;
    }
    const size_t bytes = fa2_xent_fwd_workspace_bytes(rows, q.hidden, q.vocab) + (keep ? 0 : state_bytes);
    const Tensor ws = bytes_of(bytes, x);
    check_rc(fa2_xent_fwd(&q, ws.data_ptr(), bytes, stream_of(x)), op);
    return {loss, state};
}

std::tuple<Tensor, Tensor> xent_grads(const Tensor &dloss, const Tensor &w, const Tensor &state, int64_t rows, int64_t ignore_index,
                                      int64_t reduction, bool want_dx, bool want_dw) {
    const char *op = "linear_cross_entropy backward";
    at::hip::HIPGuardMasqueradingAsCUDA guard(w.device());
    fa2_xent_params q;
    xent_common(q, w, rows, ignore_index, reduction, op);
    const Tensor wr = weight_rows(w), g = dloss.contiguous();
    q.weight = wr.data_ptr();
    q.weight_stride = wr.stride(0);
    q.dloss = g.data_ptr<float>();
    q.dloss_stride = reduction == FA2_REDUCE_NONE ? 1 : 0;
    q.state = state.data_ptr();
    q.state_bytes = (size_t)state.numel();
    Tensor dx = want_dx ? torch::empty({rows, w.size(1)}, w.options()) : Tensor();
    Tensor dw = want_dw ? torch::empty({w.size(0), w.size(1)}, w.options()) : Tensor();
    q.dx = want_dx ? dx.data_ptr() : nullptr;
    q.dweight = want_dw ? dw.data_ptr() : nullptr;
    const size_t bytes = fa2_xent_bwd_workspace_bytes(rows, q.hidden, q.vocab);
    const Tensor ws = bytes_of(bytes, w);
    check_rc(fa2_xent_bwd(&q, ws.data_ptr(), bytes, stream_of(w)), op);
    return {dx, dw};
}

// Keeps the weight and the forward's state (log-sum-exp and packed states of the
// tokens that count), no logits.
struct XentFn : torch::autograd::Function<XentFn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const Tensor &target, int64_t ignore_index,
                          int64_t reduction) {
        const XentOut o = xent_run(x, w, target, ignore_index, reduction, true);
        ctx->save_for_backward({w, o.state});
        ctx->saved_data["shape"] = x.sizes().vec();
        ctx->saved_data["ignore"] = ignore_index;
        ctx->saved_data["reduction"] = reduction;
        return o.loss;
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        const variable_list saved = ctx->get_saved_variables();
        const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
        int64_t rows = 1;
        for (size_t i = 0; i + 1 < shape.size(); ++i) rows *= shape[i];
        const auto [dx, dw] = xent_grads(g[0], saved[0], saved[1], rows, ctx->saved_data["ignore"].toInt(),
                                         ctx->saved_data["reduction"].toInt(), ctx->needs_input_grad(0), ctx->needs_input_grad(1));
        return once({dx.defined() ? dx.view(shape) : dx, dw, Tensor(), Tensor(), Tensor()}, "linear_cross_entropy");
    }
};

Tensor linear_cross_entropy(const Tensor &x, const Tensor &w, const Tensor &target, int64_t ignore_index, int64_t reduction) {
    check_xent(x, w, target, "linear_cross_entropy");
    if (wants_grad(x) || wants_grad(w)) return XentFn::apply(x, w, target, ignore_index, reduction);
    return xent_run(x, w, target, ignore_index, reduction, false).loss;
}

}  // namespace

void bind_token_ops(pybind11::module_ &m) {
    m.def("rms_norm", &rms_norm, "RMS norm");
    m.def("add_rms_norm", &add_rms_norm, "residual addition and RMS norm");
    m.def("rms_norm_fp8", &rms_norm_fp8, "residual addition and RMS norm, 8-bit output with scales");
    m.def("dropout", &dropout, "dropout from the counter-based generator");
    m.def("linear_cross_entropy", &linear_cross_entropy, "language model head with cross entropy");
}
