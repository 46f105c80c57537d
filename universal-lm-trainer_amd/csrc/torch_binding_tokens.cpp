// torch_binding_tokens.cpp -- the extension's operators on token rows, over the
// C ABI: RMS norm with the residual's addition, dropout, and the language model
// head with its cross entropy.
//   rms_norm_fwd(x, residual?, weight, eps, dropout_p, seed, y_dtype, keep) -> [y, h?, rstd?]
//   rms_norm_fp8(x, residual?, weight, eps)                                 -> [q, scale, h?]
//   rms_norm_bwd(dy, dh?, h, weight, rstd, x_dtype, dropout_p, seed, want_dx, want_dres, want_dw)
//                                                                           -> [dx?, dres?, dw?]
//   dropout(x, dropout_p, seed)                                             -> y
//   xent_fwd(x, weight, target, ignore_index, reduction)                    -> [loss, state]
//   xent_bwd(dloss, weight, state, rows, ignore_index, reduction, want_dx, want_dw) -> [dx?, dw?]
// (? = may be None / undefined.)  Tensors of any leading dimensions; a last
// dimension that is not of unit stride, or leading ones that are no single stride,
// are copied.  Outputs, state and workspaces come from the torch caching allocator
// on x's device; launches go to the current stream, with no synchronisation.
#include <torch/extension.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <cstring>
#include <vector>

#include "../../include/fa2_mi355x.h"

namespace {

using torch::Tensor;
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
    TORCH_CHECK(s == torch::kFloat, op, ": fp16, bf16 or fp32 tensors only");
    return FA2_F32;
}

void check_gpu(const Tensor &t, const Tensor &like, const char *op, const char *name) {
    TORCH_CHECK(t.is_cuda() && t.device() == like.device(), op, ": ", name, " must be on x's GPU");
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

void check_norm(const Tensor &x, const Maybe &res, const Tensor &w, const char *op) {
    TORCH_CHECK(x.is_cuda() && x.dim() >= 1 && x.size(-1) >= 1, op, ": x must be a GPU tensor of rows");
    check_gpu(w, x, op, "weight");
    TORCH_CHECK(w.dim() == 1 && w.size(0) == x.size(-1), op, ": weight must have x's last dimension");
    if (res) {
        check_gpu(*res, x, op, "residual");
        TORCH_CHECK(res->sizes() == x.sizes(), op, ": residual must have x's shape");
    }
}

// y, h and rstd or scale of one call.
std::vector<Tensor> norm_run(const Tensor &x, const Maybe &res, const Tensor &w, double eps, double p, int64_t seed,
                             c10::ScalarType y_dtype, bool keep, const char *op) {
    check_norm(x, res, w, op);
    TORCH_CHECK(x.size(-1) <= FA2_ROW_MAX, op, ": rows of at most ", FA2_ROW_MAX, " elements");
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

std::vector<Tensor> rms_norm_fwd(Tensor x, Maybe res, Tensor w, double eps, double p, int64_t seed,
                                 at::ScalarType y_dtype, bool keep) {
    return norm_run(x, res, w, eps, p, seed, y_dtype, keep, "rms_norm");
}

std::vector<Tensor> rms_norm_fp8(Tensor x, Maybe res, Tensor w, double eps) {
    std::vector<Tensor> v = norm_run(x, res, w, eps, 0.0, 0, torch::kFloat8_e4m3fn, true, "rms_norm_fp8");
    return {v[0], v[2], v[1]};
}

std::vector<Tensor> rms_norm_bwd(Tensor dy, Maybe dh, Tensor h, Tensor w, Tensor rstd, at::ScalarType xs, double p,
                                 int64_t seed, bool want_dx, bool want_dres, bool want_dw) {
    const char *op = "rms_norm backward";
    check_norm(h, dh, w, op);
    check_gpu(dy, h, op, "dy");
    TORCH_CHECK(dy.sizes() == h.sizes() && rstd.numel() == h.numel() / h.size(-1) && rstd.dtype() == torch::kFloat &&
                    rstd.device() == h.device() && rstd.is_contiguous(),
                op, ": dy and rstd must fit h");
    TORCH_CHECK(!dh || dh->scalar_type() == h.scalar_type(), op, ": dh must be of h's type");
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

Tensor dropout(Tensor x, double p, int64_t seed) {
    const char *op = "dropout";
    TORCH_CHECK(x.is_cuda() && x.dim() >= 1, op, ": x must be a GPU tensor of rows");
    at::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    Tensor y = like(x, x.scalar_type());
    fa2_dropout_params q;
    memset(&q, 0, sizeof(q));
    q.type = type_of(x.scalar_type(), op);
    if (x.numel() == 0) return y;
    const Tensor xr = as_rows(x);
    TORCH_CHECK(x.size(-1) <= INT32_MAX, op, ": rows of less than 2^31 elements");
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

// The weight as rows that the products read in place: 16-byte rows unless the
// hidden size is padded anyway.
Tensor weight_rows(const Tensor &w) {
    const bool rows = w.stride(1) == 1 && w.stride(0) >= w.size(1) && w.stride(0) < (1 << 22);
    const bool fits = reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0 && w.stride(0) % 8 == 0;
    if (rows && (fits || w.size(1) % 64 != 0)) return w;
    return w.clone(at::MemoryFormat::Contiguous);
}

Tensor bytes_of(size_t n, const Tensor &like) { return torch::empty({(int64_t)n}, like.options().dtype(torch::kByte)); }

void xent_common(fa2_xent_params &q, const Tensor &w, int64_t rows, int64_t ignore_index, int64_t reduction, const char *op) {
    TORCH_CHECK(w.dim() == 2 && w.size(0) >= 1 && w.size(1) >= 1, op, ": weight must be [vocab, hidden]");
    TORCH_CHECK(w.dtype() == torch::kHalf || w.dtype() == torch::kBFloat16, op, ": fp16 or bf16 only");
    TORCH_CHECK(rows <= (1 << 24) && w.size(0) <= (1 << 24) && w.size(1) <= FA2_ROW_MAX, op,
                ": at most 2^24 rows, a vocabulary of 2^24 and ", FA2_ROW_MAX, " hidden elements");
    memset(&q, 0, sizeof(q));
    q.type = type_of(w.scalar_type(), op);
    q.rows = rows;
    q.hidden = (int32_t)w.size(1);
    q.vocab = (int32_t)w.size(0);
    q.ignore_index = ignore_index;
    q.reduction = (int32_t)reduction;
}

std::vector<Tensor> xent_fwd(Tensor x, Tensor w, Tensor target, int64_t ignore_index, int64_t reduction) {
    const char *op = "linear_cross_entropy";
    TORCH_CHECK(x.is_cuda() && x.dim() >= 1, op, ": x must be a GPU tensor of rows");
    check_gpu(w, x, op, "weight");
    check_gpu(target, x, op, "target");
    TORCH_CHECK(w.dim() == 2 && x.size(-1) == w.size(1) && x.dtype() == w.dtype(), op,
                ": weight must be [vocab, hidden] with x's last dimension and type");
    TORCH_CHECK(target.dtype() == torch::kLong && target.sizes() == x.sizes().slice(0, x.dim() - 1), op,
                ": target must be int64 with x's leading dimensions");
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
    q.state_bytes = fa2_xent_state_bytes(rows, q.hidden);
    Tensor state = bytes_of(q.state_bytes, x);
    q.state = state.data_ptr();
    const size_t bytes = fa2_xent_fwd_workspace_bytes(rows, q.hidden, q.vocab);
    const Tensor ws = bytes_of(bytes, x);
    check_rc(fa2_xent_fwd(&q, ws.data_ptr(), bytes, stream_of(x)), op);
    return {loss, state};
}

std::vector<Tensor> xent_bwd(Tensor dloss, Tensor w, Tensor state, int64_t rows, int64_t ignore_index, int64_t reduction,
                             bool want_dx, bool want_dw) {
    const char *op = "linear_cross_entropy backward";
    TORCH_CHECK(w.is_cuda() && w.dim() == 2, op, ": weight must be [vocab, hidden] on the GPU");
    check_gpu(dloss, w, op, "dloss");
    check_gpu(state, w, op, "state");
    TORCH_CHECK(dloss.dtype() == torch::kFloat && dloss.numel() == (reduction == FA2_REDUCE_NONE ? rows : 1), op,
                ": dloss must be fp32 with the loss's shape");
    TORCH_CHECK(state.dtype() == torch::kByte && state.is_contiguous(), op, ": state must be the bytes xent_fwd returned");
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

}  // namespace

void bind_token_ops(pybind11::module_ &m) {
    m.def("rms_norm_fwd", &rms_norm_fwd, "residual addition and RMS norm");
    m.def("rms_norm_fp8", &rms_norm_fp8, "residual addition and RMS norm, 8-bit output with scales");
    m.def("rms_norm_bwd", &rms_norm_bwd, "backward of rms_norm_fwd");
    m.def("dropout", &dropout, "dropout from the counter-based generator");
    m.def("xent_fwd", &xent_fwd, "language model head with cross entropy");
    m.def("xent_bwd", &xent_bwd, "backward of xent_fwd");
}
