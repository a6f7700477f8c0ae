// The training operators of the C ABI as PyTorch calls: checks of the tensors, allocation on PyTorch's current stream, and the
// autograd node of the layer norm.  A training step of a small network is bound by the host: through ctypes the checks and
// pointer tables of an AdamW step over 93 tensors took 116 us and a layer norm's forward and backward 50, more than the
// kernels of a 24 M parameter network.
#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <string>
#include <vector>

#include "../../include/az_engine.h"

namespace {

[[noreturn]] void value_error(const std::string &s) { throw py::value_error(s); }
[[noreturn]] void type_error(const std::string &s) { throw py::type_error(s); }

std::string name_of(at::ScalarType t) { return std::string("torch.") + (t == at::kBFloat16 ? "bfloat16" : t == at::kHalf ? "float16" : t == at::kFloat ? "float32" : c10::toString(t)); }

int32_t type_id(at::ScalarType t) { return t == at::kFloat ? AZ_TYPE_F32 : t == at::kBFloat16 ? AZ_TYPE_BF16 : t == at::kHalf ? AZ_TYPE_F16 : -1; }

hipStream_t stream_of(const at::Tensor &t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.get_device()).stream(); }

bool capturing(const at::Tensor &t)
{
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream_of(t), &status) == hipSuccess) return status != hipStreamCaptureStatusNone;
    (void)hipGetLastError();   // (the default stream cannot be asked while another thread captures)
    return true;
}

// A tracer records PyTorch's own operations only: what is launched here would be missing from the graph, its result a constant.
void not_traced(const char *what)
{
    if (torch::jit::tracer::isTracing() || c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY))
        throw std::runtime_error(std::string(what) + " cannot be traced on the GPU");
}

void launched(int rc)
{
    if (rc) throw std::runtime_error("az_engine error " + std::to_string(rc) + ": " + az_last_error(nullptr));
}

// ---- layer norm -----------------------------------------------------------------------------------------------------------
// x as rows of `cols` neighbouring elements, and the elements from one row to the next; copied only if it is not one
std::pair<at::Tensor, int64_t> as_rows(const at::Tensor &x_, int64_t cols)
{
    const at::Tensor x = x_.is_neg() ? x_.resolve_neg() : x_;     // (a sign that is not in memory yet)
    if (x.is_contiguous()) return {x, cols};
    if (x.dim() > 1 && (x.stride(-1) == 1 || cols == 1)) {
        int64_t step = -1, next = 0;   // of the leading axes, from the last one: the stride that continues the ones so far
        bool merge = true;
        for (int64_t d = x.dim() - 2; d >= 0 && merge; d--) {
            if (x.size(d) == 1) continue;
            if (step < 0) step = x.stride(d);
            else merge = x.stride(d) == next;
            next = x.stride(d) * x.size(d);
        }
        if (merge) return {x, step < 0 ? cols : step};
    }
    return {x.contiguous(), cols};
}

// a weight or bias as its elements lie in memory
at::Tensor plain(const at::Tensor &t) { return !t.defined() ? t : t.is_neg() ? t.resolve_neg().contiguous() : t.contiguous(); }

const void *pointer(const at::Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }

at::Tensor norm_forward(const at::Tensor &x, const at::Tensor &weight, const at::Tensor &bias, double eps, float *mean, float *rstd)
{
    const int64_t cols = x.size(-1), rows = x.numel() / cols;
    const auto [v, stride] = as_rows(x, cols);
    const at::Tensor w = plain(weight), b = plain(bias);
    const at::ScalarType affine = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat;
    const int32_t type = type_id(x.scalar_type());
    at::Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous)), space;
    const int64_t n = az_layer_norm_fwd_workspace(type, rows, cols);
    if (n) space = at::empty({n}, x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
    launched(az_layer_norm_fwd_dev(x.get_device(), stream_of(x), type, type_id(affine), rows, cols, eps, v.const_data_ptr(), stride,
                                   pointer(w), pointer(b), y.data_ptr(), cols, mean, rstd, n ? static_cast<float *>(space.data_ptr()) : nullptr, n));
    return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &x, const std::optional<at::Tensor> &weight_, const std::optional<at::Tensor> &bias_, double eps)
    {
        const at::Tensor weight = weight_ ? *weight_ : at::Tensor(), bias = bias_ ? *bias_ : at::Tensor();
        const int64_t rows = x.numel() / x.size(-1);
        const at::Tensor stats = at::empty({2 * rows}, x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
        float *at = static_cast<float *>(stats.data_ptr());
        const at::Tensor y = norm_forward(x, weight, bias, eps, at, at + rows);
        ctx->save_for_backward({x, weight, stats});
        ctx->saved_data["bias"] = bias.defined();
        ctx->saved_data["affine"] = (int64_t)(weight.defined() ? weight.scalar_type() : bias.defined() ? bias.scalar_type() : at::kFloat);
        return y;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list grads)
    {
        // (grad mode is on in a backward pass that is to be differentiated itself)
        TORCH_CHECK(!at::GradMode::is_enabled(), "layer_norm can be differentiated once only");
        const auto saved = ctx->get_saved_variables();
        const at::Tensor &x = saved[0], &stats = saved[2];
        const at::Tensor w = plain(saved[1]);
        const int64_t cols = x.size(-1), rows = x.numel() / cols;
        const auto affine = (at::ScalarType)ctx->saved_data["affine"].toInt();
        const auto [v, x_stride] = as_rows(x, cols);
        const auto [g, dy_stride] = as_rows(grads[0], cols);
        const int32_t type = type_id(x.scalar_type());
        const auto options = x.options().memory_format(at::MemoryFormat::Contiguous);
        at::Tensor dx, dw, db, space;
        // (needs_input_grad counts the tensors that were given)
        if (ctx->needs_input_grad(0)) dx = at::empty(x.sizes(), options);
        if (w.defined() && ctx->needs_input_grad(1)) dw = at::empty({cols}, options.dtype(affine));
        if (ctx->saved_data["bias"].toBool() && ctx->needs_input_grad(w.defined() ? 2 : 1)) db = at::empty({cols}, options.dtype(affine));
        const int64_t n = dw.defined() || db.defined() ? az_layer_norm_bwd_workspace(type, rows, cols) : az_layer_norm_fwd_workspace(type, rows, cols);
        if (n) space = at::empty({n}, options.dtype(at::kFloat));
        const float *at = static_cast<const float *>(stats.const_data_ptr());
        launched(az_layer_norm_bwd_dev(x.get_device(), stream_of(x), type, type_id(affine), rows, cols, g.const_data_ptr(), dy_stride, v.const_data_ptr(), x_stride,
                                       pointer(w), at, at + rows, dx.defined() ? dx.data_ptr() : nullptr, cols, dw.defined() ? dw.data_ptr() : nullptr,
                                       db.defined() ? db.data_ptr() : nullptr, n ? static_cast<float *>(space.data_ptr()) : nullptr, n));
        return {dx, dw, db, at::Tensor()};
    }
};

// layer_norm of network/layer_norm.py; nothing comes back for checked tensors on the CPU
std::optional<at::Tensor> layer_norm(const at::Tensor &x, const std::optional<at::Tensor> &weight, const std::optional<at::Tensor> &bias, double eps)
{
    const at::ScalarType type = x.scalar_type();
    if (type_id(type) < 0) type_error("layer_norm takes float32, bfloat16 or float16, not " + name_of(type));
    if (x.dim() == 0 || x.size(-1) == 0) value_error("layer_norm needs a last axis of at least one element");
    if (!(eps >= 0.0 && eps < std::numeric_limits<double>::infinity())) value_error("eps must be a non-negative number");
    const auto check = [&](const std::optional<at::Tensor> &t, const char *name) {
        if (!t) return;
        if (t->dim() != 1 || t->size(0) != x.size(-1))
            value_error(std::string(name) + " must have one axis of " + std::to_string(x.size(-1)) + " elements, as the last axis of x");
        if (t->scalar_type() != type && t->scalar_type() != at::kFloat) type_error(std::string(name) + " must be float32 or of x's type, not " + name_of(t->scalar_type()));
        if (t->device() != x.device()) value_error(std::string(name) + " is on " + t->device().str() + ", x on " + x.device().str());
    };
    check(weight, "weight");
    check(bias, "bias");
    if (weight && bias && weight->scalar_type() != bias->scalar_type()) type_error("weight and bias must have one type");
    if (x.is_cpu()) return std::nullopt;
    if (!x.is_cuda()) value_error("layer_norm runs on the GPU or the CPU, not on " + x.device().str());
    not_traced("layer_norm");
    for (const at::Tensor *t : {&x, weight ? &*weight : nullptr, bias ? &*bias : nullptr})
        if (t && t->_fw_grad(0).defined()) throw std::runtime_error("layer_norm has no forward-mode derivative on the GPU");
    const bool record = at::GradMode::is_enabled() && (x.requires_grad() || (weight && weight->requires_grad()) || (bias && bias->requires_grad()));
    py::gil_scoped_release nogil;
    if (!record) return norm_forward(x, weight ? *weight : at::Tensor(), bias ? *bias : at::Tensor(), eps, nullptr, nullptr);
    // The gradients of leaves are added on the stream on which the leaf was first used; where that is not the captured one
    // the capture breaks in the autograd thread and takes the process with it.
    if (capturing(x)) throw std::runtime_error("layer_norm cannot record gradients while a HIP graph is captured: use torch.no_grad()");
    return LayerNorm::apply(x, weight, bias, eps);
}

// ---- AdamW ----------------------------------------------------------------------------------------------------------------
std::vector<at::Tensor> tensors_of(const py::sequence &list, const char *what)
{
    std::vector<at::Tensor> out;
    out.reserve(list.size());
    for (const py::handle h : list) {
        if (!THPVariable_Check(h.ptr())) type_error(std::string(what) + " is not a tensor");
        out.push_back(THPVariable_Unpack(h.ptr()));
    }
    return out;
}

// adamw_step of network/adamw.py: 0 or the C ABI's error; 1 for checked tensors on the CPU, with nothing done
int adamw_step(const py::sequence &params_, const py::sequence &grads_, const py::sequence &m_, const py::sequence &v_, int64_t step, double lr, double beta1,
               double beta2, double eps, double weight_decay, const std::optional<py::sequence> &m_scales_, const std::optional<py::sequence> &v_scales_)
{
    if (!(lr >= 0.0) || !(eps >= 0.0) || !(weight_decay >= 0.0)) value_error("lr, eps and weight_decay must not be negative");
    if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0)) value_error("betas must lie in [0, 1)");
    if (step < 1) value_error("steps are counted from 1");
    if (m_scales_.has_value() != v_scales_.has_value()) value_error("8-bit states need the scales of both");
    const bool eight = m_scales_.has_value();
    const auto params = tensors_of(params_, "a parameter"), m = tensors_of(m_, "exp_avg"), v = tensors_of(v_, "exp_avg_sq");
    const auto ms = eight ? tensors_of(*m_scales_, "a scale") : std::vector<at::Tensor>(), vs = eight ? tensors_of(*v_scales_, "a scale") : std::vector<at::Tensor>();
    auto grads = tensors_of(grads_, "a gradient");
    const size_t n = params.size();
    if (grads.size() != n || m.size() != n || v.size() != n || (eight && (ms.size() != n || vs.size() != n)))
        value_error("one gradient, two states and their scales for every parameter");
    if (n == 0) return 0;
    const at::ScalarType type = params[0].scalar_type();
    const at::Device device = params[0].device();
    if (type_id(type) < 0) type_error("adamw_step takes float32, bfloat16 or float16 parameters, not " + name_of(type));
    std::vector<int64_t> numels(n);
    std::vector<void *> pp(n), mp(n), vp(n);
    std::vector<const void *> gp(n);
    std::vector<float *> msp(eight ? n : 0), vsp(eight ? n : 0);
    const bool there = device.is_cuda();
    const auto check = [&](const at::Tensor &t, at::ScalarType kind, const char *what) {
        if (t.layout() != at::kStrided) type_error(std::string(what) + " is not a strided tensor");
        if (t.scalar_type() != kind) type_error(std::string(what) + " is not " + name_of(kind));
        if (t.device() != device) value_error(std::string(what) + " is not on " + device.str());
        if (there && t.is_neg()) type_error(std::string(what) + " is negated in name only: resolve_neg() it");
    };
    for (size_t i = 0; i < n; i++) {
        const at::Tensor &p = params[i];
        check(p, type, "a parameter");
        const auto alike = [&](const at::Tensor &t, at::ScalarType kind, const char *what) {
            check(t, kind, what);
            if (t.sizes() != p.sizes()) value_error(std::string("the shape of a parameter and of its ") + what + " differ");
            if (!(p.is_contiguous() && t.is_contiguous()) && !(p.is_non_overlapping_and_dense() && p.strides() == t.strides()))
                value_error(std::string(what) + " does not lie in memory as its parameter does (or the parameter is not dense)");
        };
        if (there && grads[i].is_neg()) grads[i] = grads[i].resolve_neg();      // (read only: a copy does)
        alike(grads[i], type, "gradient");
        alike(m[i], eight ? at::kChar : at::kFloat, "exp_avg");
        alike(v[i], eight ? at::kByte : at::kFloat, "exp_avg_sq");
        numels[i] = p.numel();
        if (eight) {
            for (const at::Tensor *s : {&ms[i], &vs[i]}) {
                check(*s, at::kFloat, "a scale");
                if (s->numel() != (numels[i] + AZ_STATE_BLOCK - 1) / AZ_STATE_BLOCK || !s->is_contiguous())
                    value_error("one contiguous scale for every " + std::to_string(AZ_STATE_BLOCK) + " elements");
            }
        }
        if (!there) continue;
        pp[i] = p.data_ptr(); gp[i] = grads[i].const_data_ptr(); mp[i] = m[i].data_ptr(); vp[i] = v[i].data_ptr();
        if (eight) { msp[i] = static_cast<float *>(ms[i].data_ptr()); vsp[i] = static_cast<float *>(vs[i].data_ptr()); }
    }
    if (device.is_cpu()) return 1;
    if (!there) value_error("adamw_step runs on the GPU or the CPU, not on " + device.str());
    not_traced("an AdamW step");
    if (capturing(params[0])) throw std::runtime_error("an AdamW step cannot be captured into a HIP graph: every replay would be the same step");
    int rc;
    {
        py::gil_scoped_release nogil;
        rc = az_adamw_step_dev(params[0].get_device(), stream_of(params[0]), (int64_t)n, pp.data(), gp.data(), mp.data(), vp.data(), eight ? msp.data() : nullptr,
                               eight ? vsp.data() : nullptr, numels.data(), type_id(type), lr, beta1, beta2, eps, weight_decay, step);
    }
    if (rc) return rc;
    // autograd learns that these were written, as from any operation in place: a backward pass that saved one before refuses
    for (const auto *list : {&params, &m, &v, &ms, &vs})
        for (const at::Tensor &t : *list)
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    return 0;
}

// dequantize_state of network/adamw.py; nothing comes back for checked tensors on the CPU
std::optional<at::Tensor> dequantize_state(const at::Tensor &codes, const at::Tensor &scales)
{
    const at::ScalarType type = codes.scalar_type();
    if ((type != at::kChar && type != at::kByte) || scales.scalar_type() != at::kFloat)
        type_error("a state in 8 bits is int8 or uint8 codes with float32 scales, not " + name_of(type) + " with " + name_of(scales.scalar_type()));
    if (codes.device() != scales.device()) value_error("codes are on " + codes.device().str() + ", scales on " + scales.device().str());
    const int64_t n = codes.numel(), blocks = (n + AZ_STATE_BLOCK - 1) / AZ_STATE_BLOCK;
    if (!codes.is_non_overlapping_and_dense() || !scales.is_contiguous() || scales.numel() != blocks)
        value_error(std::to_string(n) + " codes need dense memory and " + std::to_string(blocks) + " scales, not " + std::to_string(scales.numel()));
    if (codes.is_cpu()) return std::nullopt;
    if (!codes.is_cuda()) value_error("dequantize_state runs on the GPU or the CPU, not on " + codes.device().str());
    if (scales.is_neg()) type_error("scales are negated in name only: resolve_neg() them");
    not_traced("dequantize_state");
    at::Tensor out = at::empty_strided(codes.sizes(), codes.strides(), codes.options().dtype(at::kFloat));
    launched(az_dequantize_state_dev(codes.get_device(), stream_of(codes), codes.const_data_ptr(), static_cast<const float *>(scales.const_data_ptr()), n,
                                     type == at::kChar, static_cast<float *>(out.data_ptr())));
    return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.def("layer_norm", &layer_norm);
    m.def("adamw_step", &adamw_step);
    m.def("dequantize_state", &dequantize_state);
}
