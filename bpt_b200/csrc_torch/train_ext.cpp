// The differentiable training operators as a thin torch C++ extension over the C-ABI library: tensor checks, output and
// workspace allocation, one bpt_* call per direction, and the autograd nodes.  Compiled because a training step of small
// tensors is host time: the same nodes written in Python cost 150 us a forward and backward, these about a third.
// bpt_b200/norm.py and bpt_b200/loss.py document the functions.
#include <ATen/Functions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "../../include/bpt_b200.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

int dtype_code(const at::Tensor &t, const char *what) {
    switch (t.scalar_type()) {
        case at::kFloat: return BPT_F32;
        case at::kBFloat16: return BPT_BF16;
        case at::kHalf: return BPT_F16;
        default: TORCH_CHECK(false, "bpt_b200: ", what, ": unsupported dtype ", t.scalar_type());
    }
    return -1;
}
void check_rc(int rc) { TORCH_CHECK(rc == BPT_OK, "bpt_b200 error ", rc, ": ", bpt_last_error()); }
bpt_stream_t stream_of(const at::Tensor &t) {
    return reinterpret_cast<bpt_stream_t>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
}
const void *ptr(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
void *mutable_ptr(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
float *f32(const at::Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
at::Tensor workspace(size_t bytes, const at::Tensor &like) {
    return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}
at::Tensor or_undefined(const OptTensor &t) { return t.has_value() ? *t : at::Tensor(); }
// An autograd node takes tensors that may be missing as optionals; its edges count the ones that are there.
OptTensor if_defined(const at::Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }
// A view whose memory holds the negatives (the imaginary part of a conjugate) is written out: kernels read memory.
at::Tensor as_stored(const at::Tensor &t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }
at::Tensor contiguous(const at::Tensor &t) { return t.defined() ? as_stored(t).contiguous() : t; }
bool wants_grad(const at::Tensor &t) { return t.defined() && t.requires_grad(); }
// There are no forward-mode derivatives.  The autograd nodes would say so, but calls without a node would drop the tangent.
void refuse_tangents(const char *name, std::initializer_list<const at::Tensor *> inputs) {
    for (const at::Tensor *t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), "bpt_b200: ", name, " has no forward-mode derivative");
}

// Results of a backward that has no derivative of its own: asking for one is an error, as with once_differentiable.
variable_list once(variable_list grads, const char *what) {
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string("bpt_b200: ") + what + " is differentiable once only",
                                                                static_cast<int64_t>(grads.size()));
    for (at::Tensor &g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    return (*error)(std::move(grads));
}

// ---------------------------------------------------------------------------------- layer norm
constexpr int64_t kMaxDim = 8192;

at::Tensor norm_forward(const at::Tensor &x, const at::Tensor &residual, const at::Tensor &weight, const at::Tensor &bias, double eps,
                        at::Tensor *mean_rstd) {
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t dim = x.size(-1), rows = x.numel() / dim;
    at::Tensor y = at::empty_like(x);
    if (mean_rstd) *mean_rstd = at::empty({2, rows}, x.options().dtype(at::kFloat));
    float *mean = mean_rstd ? f32(*mean_rstd) : nullptr;
    check_rc(bpt_layer_norm_forward(ptr(x), ptr(residual), ptr(weight), ptr(bias), eps, mutable_ptr(y), mean, mean ? mean + rows : nullptr,
                                    rows, static_cast<int>(dim), dtype_code(x, "layer_norm"), stream_of(x)));
    return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const OptTensor &residual_, const OptTensor &weight_,
                              const OptTensor &bias_, double eps) {
        const at::Tensor residual = or_undefined(residual_), weight = or_undefined(weight_), bias = or_undefined(bias_);
        at::Tensor mean_rstd;
        at::Tensor y = norm_forward(x, residual, weight, bias, eps, &mean_rstd);
        ctx->save_for_backward({x, residual, weight, mean_rstd});
        ctx->saved_data["bias"] = bias.defined();
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grad) {
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &residual = saved[1], &weight = saved[2], &mean_rstd = saved[3];
        const c10::cuda::CUDAGuard guard(x.device());
        const int64_t dim = x.size(-1), rows = x.numel() / dim;
        const at::Tensor gy = contiguous(grad[0]);
        size_t edge = 0;
        auto needed = [&](bool there) { return there && ctx->needs_input_grad(edge++); };
        const bool need_x = needed(true), need_r = needed(residual.defined()), need_w = needed(weight.defined());
        const bool need_b = needed(ctx->saved_data["bias"].toBool());
        at::Tensor da, dw, db, ws;
        if (need_x || need_r) da = at::empty_like(x);
        if (need_w) dw = at::empty({dim}, x.options());
        if (need_b) db = at::empty({dim}, x.options());
        const size_t bytes = need_w || need_b ? bpt_layer_norm_backward_workspace_bytes(rows, static_cast<int>(dim)) : 0;
        if (bytes) ws = workspace(bytes, x);
        const float *mean = f32(mean_rstd);
        check_rc(bpt_layer_norm_backward(ptr(gy), ptr(x), ptr(residual), ptr(weight), mean, mean + rows, mutable_ptr(da), mutable_ptr(dw),
                                         mutable_ptr(db), rows, static_cast<int>(dim), dtype_code(x, "layer_norm"), mutable_ptr(ws), bytes,
                                         stream_of(x)));
        return once({need_x ? da : at::Tensor(), need_r ? da : at::Tensor(), dw, db, at::Tensor()}, "layer_norm");
    }
};

at::Tensor layer_norm(const at::Tensor &x_, const OptTensor &weight_, const OptTensor &bias_, double eps, const OptTensor &residual_) {
    TORCH_CHECK(x_.is_cuda(), "bpt_b200: expected a CUDA tensor (there is no CPU path)");
    dtype_code(x_, "layer_norm");
    TORCH_CHECK(x_.dim() >= 1 && x_.size(-1) >= 1 && x_.size(-1) <= kMaxDim, "bpt_b200: layer_norm: the last dimension must be in [1, ", kMaxDim, "]");
    const at::Tensor weight_in = or_undefined(weight_), bias_in = or_undefined(bias_), residual_in = or_undefined(residual_);
    refuse_tangents("layer_norm", {&x_, &weight_in, &bias_in, &residual_in});
    auto check = [&](const at::Tensor &t, const char *name, at::IntArrayRef shape) {
        TORCH_CHECK(!t.defined() || (t.device() == x_.device() && t.scalar_type() == x_.scalar_type() && t.sizes() == shape),
                    "bpt_b200: layer_norm: ", name, " must be a ", x_.scalar_type(), " tensor of shape ", shape, " on ", x_.device());
    };
    check(weight_in, "weight", x_.sizes().slice(x_.dim() - 1));
    check(bias_in, "bias", x_.sizes().slice(x_.dim() - 1));
    check(residual_in, "residual", x_.sizes());
    const at::Tensor x = contiguous(x_), weight = contiguous(weight_in), bias = contiguous(bias_in), residual = contiguous(residual_in);
    if (at::GradMode::is_enabled() && (x.requires_grad() || wants_grad(residual) || wants_grad(weight) || wants_grad(bias)))
        return LayerNorm::apply(x, if_defined(residual), if_defined(weight), if_defined(bias), eps);
    return norm_forward(x, residual, weight, bias, eps, nullptr);
}

// ---------------------------------------------------------------------------------- projection + cross entropy
// A matrix whose rows are contiguous (a copy if need be) and its row stride in elements.  That of a single row is free.
struct Rows {
    at::Tensor t;
    int64_t ld;
    explicit Rows(const at::Tensor &m) : t(m) {
        if (m.size(0) == 1 && (m.size(1) == 1 || m.stride(1) == 1)) {
            ld = (m.size(1) + 7) / 8 * 8;
            return;
        }
        if ((m.stride(1) != 1 && m.size(1) != 1) || m.stride(0) < m.size(1)) t = m.contiguous();
        ld = std::max(t.stride(0), t.size(1));
    }
};

struct CeOptions {
    int64_t ignore_index;
    double smoothing;
    int64_t reduction;
};

at::Tensor ce_forward(const at::Tensor &x_, const at::Tensor &weight_, const at::Tensor &bias, const at::Tensor &target, const CeOptions &o,
                      at::Tensor *lse, at::Tensor *count) {
    const c10::cuda::CUDAGuard guard(x_.device());
    const Rows x(x_), w(weight_);
    const int64_t n = x.t.size(0);
    const int dim = static_cast<int>(x.t.size(1)), vocab = static_cast<int>(w.t.size(0)), dtype = dtype_code(x_, "linear_cross_entropy");
    const at::TensorOptions f = x_.options().dtype(at::kFloat);
    at::Tensor loss = o.reduction == BPT_LOSS_NONE ? at::empty({n}, f) : at::empty({}, f);
    if (lse) {
        *lse = at::empty({n}, f);
        *count = at::empty({}, f);
    }
    const size_t bytes = bpt_linear_ce_forward_workspace_bytes(ptr(x.t), x.ld, ptr(w.t), w.ld, n, vocab, dim, dtype);
    const at::Tensor ws = workspace(bytes, x_);
    check_rc(bpt_linear_ce_forward(ptr(x.t), x.ld, ptr(w.t), w.ld, ptr(bias), target.data_ptr<int64_t>(), o.ignore_index, o.smoothing,
                                   static_cast<int>(o.reduction), f32(loss), lse ? f32(*lse) : nullptr, lse ? f32(*count) : nullptr, n, vocab,
                                   dim, dtype, mutable_ptr(ws), bytes, stream_of(x_)));
    return loss;
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
    static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &weight, const OptTensor &bias_,
                              const at::Tensor &target, int64_t ignore_index, double smoothing, int64_t reduction) {
        const at::Tensor bias = or_undefined(bias_);
        at::Tensor lse, count;
        at::Tensor loss = ce_forward(x, weight, bias, target, {ignore_index, smoothing, reduction}, &lse, &count);
        ctx->save_for_backward({x, weight, bias, target, lse, count});
        ctx->saved_data["ignore_index"] = ignore_index;
        ctx->saved_data["smoothing"] = smoothing;
        ctx->saved_data["reduction"] = reduction;
        return loss;
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const at::Tensor &bias = saved[2], &target = saved[3], &lse = saved[4], &count = saved[5];
        const c10::cuda::CUDAGuard guard(saved[0].device());
        const Rows x(saved[0]), w(saved[1]);
        const int64_t n = x.t.size(0);
        const int dim = static_cast<int>(x.t.size(1)), vocab = static_cast<int>(w.t.size(0)), dtype = dtype_code(x.t, "linear_cross_entropy");
        const at::Tensor grad = contiguous(grads[0]);
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = bias.defined() && ctx->needs_input_grad(2);
        at::Tensor dx, dw, db;
        if (need_x) dx = at::empty({n, dim}, x.t.options());
        if (need_w) dw = at::empty({vocab, dim}, x.t.options());
        if (need_b) db = at::empty({vocab}, x.t.options());
        const size_t bytes = bpt_linear_ce_backward_workspace_bytes(ptr(x.t), x.ld, ptr(w.t), w.ld, n, vocab, dim, dtype, need_x, need_w, need_b);
        const at::Tensor ws = workspace(bytes, x.t);
        check_rc(bpt_linear_ce_backward(ptr(x.t), x.ld, ptr(w.t), w.ld, ptr(bias), target.data_ptr<int64_t>(),
                                        ctx->saved_data["ignore_index"].toInt(), ctx->saved_data["smoothing"].toDouble(),
                                        static_cast<int>(ctx->saved_data["reduction"].toInt()), f32(lse), f32(count), f32(grad), mutable_ptr(dx),
                                        mutable_ptr(dw), mutable_ptr(db), n, vocab, dim, dtype, mutable_ptr(ws), bytes, stream_of(x.t)));
        return once({dx, dw, db, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()}, "linear_cross_entropy");
    }
};

at::Tensor linear_cross_entropy(const at::Tensor &x_, const at::Tensor &weight_, const at::Tensor &target_, const OptTensor &bias_,
                                int64_t ignore_index, double smoothing, int64_t reduction) {
    const char *const name = "linear_cross_entropy";
    const at::Tensor weight = as_stored(weight_);
    TORCH_CHECK(x_.is_cuda(), "bpt_b200: expected a CUDA tensor (there is no CPU path)");
    dtype_code(x_, name);
    TORCH_CHECK(weight.dim() == 2 && x_.dim() >= 1 && weight.size(0) >= 1 && weight.size(1) >= 1 && x_.size(-1) == weight.size(1), "bpt_b200: ",
                name, ": x must be (..., dim) and weight (vocab, dim), got ", x_.sizes(), " and ", weight.sizes());
    TORCH_CHECK(weight.scalar_type() == x_.scalar_type() && weight.device() == x_.device(), "bpt_b200: ", name, ": weight must be a ",
                x_.scalar_type(), " tensor on ", x_.device());
    TORCH_CHECK(weight.size(0) <= (1 << 30) && weight.size(1) <= (1 << 20), "bpt_b200: ", name, ": weight is too large");
    const at::Tensor bias_in = or_undefined(bias_);
    refuse_tangents(name, {&x_, &weight, &bias_in});
    TORCH_CHECK(!bias_in.defined() || (bias_in.scalar_type() == x_.scalar_type() && bias_in.device() == x_.device() && bias_in.dim() == 1 &&
                                       bias_in.size(0) == weight.size(0)),
                "bpt_b200: ", name, ": bias must be a ", x_.scalar_type(), " tensor of shape [", weight.size(0), "] on ", x_.device());
    TORCH_CHECK(target_.scalar_type() == at::kLong && target_.device() == x_.device() && target_.sizes() == x_.sizes().slice(0, x_.dim() - 1),
                "bpt_b200: ", name, ": target must be an int64 tensor of shape ", x_.sizes().slice(0, x_.dim() - 1), " on ", x_.device());
    TORCH_CHECK(smoothing >= 0.0 && smoothing <= 1.0, "bpt_b200: ", name, ": label_smoothing must be in [0, 1]");
    const at::Tensor x = as_stored(x_.dim() == 2 ? x_ : x_.reshape({x_.numel() / x_.size(-1), x_.size(-1)}));
    const at::Tensor target = contiguous(target_.reshape({-1})), bias = contiguous(bias_in);
    at::Tensor loss;
    if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || wants_grad(bias)))
        loss = LinearCrossEntropy::apply(x, weight, if_defined(bias), target, ignore_index, smoothing, reduction);
    else
        loss = ce_forward(x, weight, bias, target, {ignore_index, smoothing, reduction}, nullptr, nullptr);
    return reduction == BPT_LOSS_NONE && target_.dim() != 1 ? loss.view(target_.sizes()) : loss;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "Differentiable training operators on libbpt_b200.so";
    m.def("layer_norm", &layer_norm, "LayerNorm(x + residual) over the last dimension");
    m.def("linear_cross_entropy", &linear_cross_entropy, "cross_entropy(x @ weight.T + bias, target) without the logits");
}
