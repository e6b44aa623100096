// abx_torch.cpp -- libabx's norms and device-resident AdamW step for torch tensors, as a Python module.
//
// The other entry points of libabx are called through ctypes, once per launch of many tensors.  These are called
// once per layer (a norm and its backward pass, which torch runs on a thread of its own) or look at every parameter
// at every call, and in Python that took longer than the kernels: 150 us for a norm forward and backward, 140 us to
// check and describe 184 parameters.  Nothing is computed here: checks, allocations and the C calls of include/abx.h.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <ATen/TensorUtils.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>

#include <memory>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/abx.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

void succeeded(int rc, const char* what)
{
    TORCH_CHECK(rc == ABX_OK, what, " failed (code ", rc, rc == ABX_E_CUDA ? std::string(": ") + abx_last_error() : "", ")");
}

bool known(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }
int32_t code_of(at::ScalarType t) { return t == at::kBFloat16 ? ABX_DT_BF16 : ABX_DT_F32; }

// ---- norms -----------------------------------------------------------------------------------------

struct Rows {
    Tensor t;          // the tensor itself where its rows lie evenly spaced, else a contiguous copy
    int64_t count;
    int64_t stride;    // elements between rows
};

// The memory of a lazily negated view holds the other sign.  (Asked first: resolving goes through torch's dispatcher.)
Tensor signed_as_read(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }

Rows rows_of(const Tensor& given)
{
    const Tensor t = signed_as_read(given);
    const int64_t cols = t.size(-1);
    if (!t.is_contiguous()) {
        const int64_t count = t.numel() / cols;
        const at::DimVector shape{count, cols};
        const auto strides = at::detail::computeStride(t.sizes(), t.strides(), shape);
        if (strides && (cols == 1 || (*strides)[1] == 1)) return {t, count, count > 1 ? (*strides)[0] : cols};
        const Tensor copy = t.contiguous();
        return {copy, count, cols};
    }
    return {t, t.numel() / cols, cols};
}

void check_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps)
{
    TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "a norm needs at least one value along the last axis, got the shape ",
                      x.sizes());
    TORCH_CHECK_VALUE(x.is_cuda(), "adambridge_b200's norms run on CUDA tensors only");
    TORCH_CHECK_TYPE(known(x.scalar_type()), "x must be float32 or bfloat16, got ", x.scalar_type());
    TORCH_CHECK_VALUE(eps >= 0.0, "invalid epsilon: ", eps);
    for (const auto& [name, t] : {std::pair{"weight", &weight}, std::pair{"bias", &bias}}) {
        if (!t->has_value()) continue;
        const Tensor& w = **t;
        TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == x.size(-1), name, " has the shape ", w.sizes(), ", the last axis ",
                          x.size(-1), " values");
        TORCH_CHECK_TYPE(known(w.scalar_type()), name, " must be float32 or bfloat16, got ", w.scalar_type());
        TORCH_CHECK_VALUE(w.device() == x.device(), name, " is on ", w.device(), ", x on ", x.device());
    }
    TORCH_CHECK_TYPE(!weight || !bias || weight->scalar_type() == bias->scalar_type(),
                     "weight and bias must have one dtype, got ", weight->scalar_type(), " and ", bias->scalar_type());
}

abx_norm describe(const Rows& x, const Tensor& weight, const Tensor& bias, double eps, bool rms)
{
    abx_norm n{};
    n.x = x.t.const_data_ptr();
    n.w = weight.defined() ? weight.const_data_ptr() : nullptr;
    n.b = bias.defined() ? bias.const_data_ptr() : nullptr;
    n.rows = x.count;
    n.cols = x.t.size(-1);
    n.x_stride = x.stride;
    n.dtype = code_of(x.t.scalar_type());
    n.w_dtype = weight.defined() ? code_of(weight.scalar_type()) : bias.defined() ? code_of(bias.scalar_type()) : n.dtype;
    n.rms = rms;
    n.eps = (float)eps;
    return n;
}

Tensor contiguous(const Tensor& t) { return t.defined() ? signed_as_read(t).contiguous() : t; }
Tensor contiguous(const std::optional<Tensor>& t) { return t ? contiguous(*t) : Tensor(); }

// y, x as the kernels read it, and where `keep`, the rows' statistics: rstd, then the mean (not for RMS norm)
std::tuple<Tensor, Tensor, Tensor> forward_norm(const Tensor& x, const std::optional<Tensor>& weight,
                                                const std::optional<Tensor>& bias, double eps, bool rms, bool keep)
{
    const c10::DeviceGuard guard(x.device());
    const Rows rows = rows_of(x);
    const Tensor w = contiguous(weight), b = contiguous(bias);
    Tensor y = at::empty(x.sizes(), x.options()), stats;
    float* rstd = nullptr;
    if (keep) {
        stats = at::empty({rms ? 1 : 2, rows.count}, x.options().dtype(at::kFloat));
        rstd = stats.mutable_data_ptr<float>();
    }
    const abx_norm n = describe(rows, w, b, eps, rms);
    succeeded(abx_norm_forward(stream_of(x), &n, y.mutable_data_ptr(), keep && !rms ? rstd + rows.count : nullptr, rstd),
              "abx_norm_forward");
    return {y, rows.t, stats};
}

// Level 0 is torch's only one.
void check_tangent(const Tensor& t)
{
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "layer_norm and rms_norm have no forward-mode derivatives");
}

class Norm : public torch::autograd::Function<Norm> {
public:
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& weight,
                          const std::optional<Tensor>& bias, double eps, bool rms)
    {
        auto [y, kept, stats] = forward_norm(x, weight, bias, eps, rms, true);
        ctx->save_for_backward({kept, weight.value_or(Tensor()), bias.value_or(Tensor()), stats});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["rms"] = rms;
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads)
    {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &weight = saved[1], &bias = saved[2], &stats = saved[3], &dy = grads[0];
        variable_list out(5);
        if (!dy.defined()) return out;
        check_tangent(dy);
        // edges are counted over the tensors that were given
        const bool want_x = ctx->needs_input_grad(0);
        const bool want_w = weight.defined() && ctx->needs_input_grad(1);
        const bool want_b = bias.defined() && ctx->needs_input_grad(weight.defined() ? 2 : 1);
        const bool twice = at::GradMode::is_enabled();
        {
            const at::AutoGradMode no_grad(false);
            const c10::DeviceGuard guard(x.device());
            const bool rms = ctx->saved_data["rms"].toBool();
            const Rows rows = rows_of(x), given = rows_of(dy);
            const Tensor w = contiguous(weight), b = contiguous(bias);
            const abx_norm n = describe(rows, w, b, ctx->saved_data["eps"].toDouble(), rms);
            if (want_x) out[0] = at::empty(x.sizes(), x.options());
            if (want_w) out[1] = at::empty(weight.sizes(), weight.options());
            if (want_b) out[2] = at::empty(bias.sizes(), bias.options());
            Tensor ws;
            size_t bytes = 0;
            if (want_w || want_b) {
                bytes = abx_norm_backward_workspace_bytes(&n);
                ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
            }
            const auto to = [](const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; };
            const float* rstd = stats.const_data_ptr<float>();
            succeeded(abx_norm_backward(stream_of(x), &n, given.t.const_data_ptr(), given.stride,
                                        rms ? nullptr : rstd + rows.count, rstd, to(out[0]), to(out[1]), to(out[2]), to(ws),
                                        bytes), "abx_norm_backward");
        }
        if (twice) {   // a graph of the gradients is being built: differentiating them says so instead of giving 0
            variable_list found;
            for (const Tensor& t : out) if (t.defined()) found.push_back(t.set_requires_grad(true));
            const auto error = std::make_shared<torch::autograd::DelayedError>(
                "layer_norm and rms_norm are once_differentiable: gradients of their gradients are not available",
                (int64_t)found.size());
            found = (*error)(std::move(found));
            size_t i = 0;
            for (Tensor& t : out) if (t.defined()) t = found[i++];
        }
        return out;
    }
};

// What follows a program through torch's dispatcher does not see a norm: it would take the result for one that nothing
// computes, or for one that does not depend on x.
void check_seen(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias)
{
    using Mode = c10::impl::TorchDispatchModeKey;
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing()
                                    && !c10::impl::TorchDispatchModeTLS::get_mode(Mode::PROXY)
                                    && !c10::impl::TorchDispatchModeTLS::get_mode(Mode::FAKE),
                                "layer_norm and rms_norm are not operators of torch's dispatcher: a trace does not see them");
    check_tangent(x);
    if (weight) check_tangent(*weight);
    if (bias) check_tangent(*bias);
}

Tensor norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, double eps, bool rms)
{
    check_norm(x, weight, bias, eps);
    check_seen(x, weight, bias);
    if (at::GradMode::is_enabled() && (x.requires_grad() || (weight && weight->requires_grad()) || (bias && bias->requires_grad())))
        return Norm::apply(x, weight, bias, eps, rms);
    return std::get<0>(forward_norm(x, weight, bias, eps, rms, false));
}

// ---- the AdamW step ----------------------------------------------------------------------------------

// The kernel descriptions of one arena's parameters that have a gradient, with the tensors they point at.
struct Described {
    std::vector<abx_graph_tensor> tensors;
    std::vector<Tensor> params;   // undefined where there is no gradient
    std::vector<Tensor> keep;
    c10::Device device{c10::kCUDA, 0};
};

// `rows`: the arena's descriptions without the addresses of weights and gradients (host, one abx_graph_tensor a row).
std::unique_ptr<Described> describe_step(std::vector<Tensor> params, const Tensor& rows, int64_t device)
{
    TORCH_CHECK_VALUE(rows.scalar_type() == at::kLong && rows.is_cpu() && rows.is_contiguous() && rows.dim() == 2
                          && rows.size(0) == (int64_t)params.size() && rows.size(1) * 8 == (int64_t)sizeof(abx_graph_tensor),
                      "one row of ", sizeof(abx_graph_tensor) / 8, " words per parameter is needed");
    auto d = std::make_unique<Described>();
    d->device = c10::Device(c10::kCUDA, (c10::DeviceIndex)device);
    d->tensors.reserve(params.size());
    d->keep.reserve(params.size());
    const auto* row = reinterpret_cast<const abx_graph_tensor*>(rows.const_data_ptr());
    d->params = std::move(params);
    for (size_t i = 0; i < d->params.size(); ++i, ++row) {
        Tensor& p = d->params[i];
        Tensor g = p.grad();
        if (!g.defined()) {
            p.reset();
            continue;
        }
        TORCH_CHECK(p.numel() == row->n && known(p.scalar_type()) && code_of(p.scalar_type()) == row->dtype
                        && p.device() == d->device,
                    "a parameter changed after its state was made (", row->n, " values of dtype code ", row->dtype, " on ",
                    d->device, ", now ", p.numel(), " x ", p.scalar_type(), " on ", p.device(), ")");
        TORCH_CHECK_VALUE(p.is_contiguous() && !p.is_neg(), "non-contiguous parameters are not supported, nor negated views");
        TORCH_CHECK(!g.is_sparse() && g.layout() == at::kStrided, "GraphAdamW does not support sparse gradients");
        TORCH_CHECK_TYPE(g.scalar_type() == p.scalar_type(), "the gradient of a ", p.scalar_type(), " parameter must be ",
                         p.scalar_type(), ", got ", g.scalar_type());
        TORCH_CHECK_VALUE(g.numel() == row->n && g.device() == d->device, "a gradient has ", g.numel(), " elements on ",
                          g.device(), ", its parameter ", row->n, " on ", d->device);
        if (!g.is_contiguous() || g.is_neg()) {
            const c10::DeviceGuard guard(d->device);
            g = signed_as_read(g).contiguous();
        }
        abx_graph_tensor t = *row;
        t.w = p.data_ptr();
        t.g = g.const_data_ptr();
        d->tensors.push_back(t);
        d->keep.push_back(std::move(g));
    }
    return d;
}

// `shared`: the address of an abx_graph_step.
void launch_step(const Described& d, uintptr_t shared, const Tensor& ticket, int64_t max_ctas)
{
    if (d.tensors.empty()) return;
    TORCH_CHECK_VALUE(ticket.device() == d.device && ticket.scalar_type() == at::kInt && ticket.numel() == 1,
                      "ticket must be a one-element int32 tensor on ", d.device);
    const c10::DeviceGuard guard(d.device);
    succeeded(abx_graph_adamw(stream_of(ticket), d.tensors.data(), (int32_t)d.tensors.size(),
                              reinterpret_cast<const abx_graph_step*>(shared), reinterpret_cast<uint32_t*>(ticket.data_ptr()),
                              (int32_t)max_ctas), "abx_graph_adamw");
    // as an operation in place says to autograd: a graph that saved a weight may no longer run backward
    for (const Tensor& p : d.params)
        if (p.defined() && !p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
}

// ---- 8-bit moments -----------------------------------------------------------------------------------

void check_i8(const Tensor& codes, const Tensor& scales, int64_t n)
{
    const int64_t blocks = (n + ABX_I8_BLOCK - 1) / ABX_I8_BLOCK;
    TORCH_CHECK_VALUE(codes.is_cuda() && scales.is_cuda() && codes.device() == scales.device() && codes.is_contiguous()
                          && scales.is_contiguous(), "codes and scales must be contiguous CUDA tensors of one device");
    TORCH_CHECK_TYPE(codes.element_size() == 1 && scales.scalar_type() == at::kFloat, "8-bit codes and float32 scales are needed");
    TORCH_CHECK_VALUE(n >= 0 && codes.numel() >= blocks * ABX_I8_BLOCK && scales.numel() >= blocks, n, " values need ", blocks,
                      " whole blocks of codes and as many scales");
}

// The first n values of 8-bit moments (second: of the second moment) as a new fp32 tensor.
Tensor i8_decode(const Tensor& codes, const Tensor& scales, int64_t n, bool second)
{
    check_i8(codes, scales, n);
    const c10::DeviceGuard guard(codes.device());
    Tensor out = at::empty({n}, scales.options());
    succeeded(abx_i8_decode(stream_of(codes), codes.const_data_ptr(), scales.const_data_ptr<float>(),
                            out.mutable_data_ptr<float>(), n, second), "abx_i8_decode");
    return out;
}

void i8_encode(const Tensor& values, const Tensor& codes, const Tensor& scales, bool second)
{
    check_i8(codes, scales, values.numel());
    TORCH_CHECK_VALUE(values.device() == codes.device() && values.is_contiguous() && values.scalar_type() == at::kFloat,
                      "values must be a contiguous float32 tensor on ", codes.device());
    const c10::DeviceGuard guard(codes.device());
    succeeded(abx_i8_encode(stream_of(codes), values.const_data_ptr<float>(), codes.mutable_data_ptr(),
                            scales.mutable_data_ptr<float>(), values.numel(), second), "abx_i8_encode");
}

}  // namespace

PYBIND11_MODULE(_abx_torch, m)
{
    m.def("norm", torch::wrap_pybind_function(norm));
    pybind11::class_<Described>(m, "Described").def("__len__", [](const Described& d) { return d.tensors.size(); });
    m.def("describe_step", torch::wrap_pybind_function(describe_step));
    m.def("launch_step", torch::wrap_pybind_function(launch_step));
    m.def("i8_decode", torch::wrap_pybind_function(i8_decode));
    m.def("i8_encode", torch::wrap_pybind_function(i8_encode));
}
