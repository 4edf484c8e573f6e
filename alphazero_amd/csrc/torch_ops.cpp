// The training operators as torch sees them: autograd nodes and the optimiser's walk over its tensors, on top of the
// C entries of libazamd.so (bound by address, so that a diagnostic build of the library is used where one is loaded).
//
// Why this is native: a Python autograd node costs 30 us in the backward pass and 25 us of argument handling per call,
// and a step over 216 parameters 100 us of list building, where the kernels themselves take 40 to 100 us.  Measured on the
// host: norm_gate_residual forward + backward 152 us with a Python node, 104 with this one, of which torch's own engine
// takes some 60 (it hands the node and each of its eight gradients from thread to thread); FusedAdam.step 150 and 25 us.
#include <mutex>

#include <pybind11/pybind11.h>
#include <pybind11/stl.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/azamd.h"

namespace py = pybind11;
using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct Entries {
    decltype(&az_last_error) last_error;
    decltype(&az_norm_sizes) norm_sizes;
    decltype(&az_norm_forward) norm_forward;
    decltype(&az_norm_backward) norm_backward;
    decltype(&az_policy_value_loss_ready) loss_ready;
    decltype(&az_policy_value_loss_forward) loss_forward;
    decltype(&az_policy_value_loss_backward) loss_backward;
    decltype(&az_adam_plan) adam_plan;
    decltype(&az_adam_scratch) adam_scratch;
    decltype(&az_adam_step) adam_step;
} lib;

PyObject* az_error = nullptr;        // the package's exception for a library error

void check(int rc) {
    if (rc == AZ_OK) return;
    const std::string what = "libazamd error " + std::to_string(rc) + ": " + lib.last_error();
    if (!PyGILState_Check()) throw std::runtime_error(what);       // autograd's own threads: torch hands it on
    PyErr_SetString(az_error, what.c_str());
    throw py::error_already_set();
}

void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

template <typename T>
T* ptr(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }

int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return AZ_F32;
        case at::kBFloat16: return AZ_BF16;
        case at::kHalf: return AZ_F16;
        default: return -1;
    }
}

// What a call may leave out.  (torch's autograd takes no undefined tensors among a node's arguments.)
typedef optional<Tensor> MaybeTensor;
Tensor held(const MaybeTensor& t) { return t ? *t : Tensor(); }

// A buffer of the device's current stream.
Tensor bytes(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kByte)); }
Tensor floats(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kFloat)); }

// `like`, at element `at` of a buffer: a tensor of its own, not a view that autograd knows of (those refuse to be changed in
// place when a node returns several).
Tensor part_of(const Tensor& all, int64_t at, at::IntArrayRef sizes, at::IntArrayRef strides) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(all.storage()), all.key_set(), all.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(at);
    t.unsafeGetTensorImpl()->set_sizes_and_strides(sizes, strides);
    return t;
}

// Float tensors like these in one allocation, each at a multiple of 256 bytes: six small gradients cost what one does (1.4 us
// instead of 8 us of a backward pass that takes 50 us of host time).  They share that memory: whoever keeps one keeps all of
// them, a few KB to 16 MB (a gate of 1024 x 1024).
std::vector<Tensor> together(const std::vector<Tensor>& like, const Tensor& device) {
    std::vector<int64_t> at;
    int64_t total = 0;
    for (const Tensor& t : like) {
        at.push_back(total);
        if (t.defined()) total += (t.numel() + 63) / 64 * 64;
    }
    const Tensor all = floats(total, device);
    std::vector<Tensor> out(like.size());
    for (size_t i = 0; i < like.size(); ++i)
        if (like[i].defined()) out[i] = part_of(all, at[i], like[i].sizes(), like[i].strides());
    return out;
}

// Gradients of a backward pass that was asked for a graph of its own: using them again is an error, not a silent zero.
variable_list first_derivatives_only(variable_list grads, const char* name) {
    if (!at::GradMode::is_enabled()) return grads;
    for (auto& g : grads)
        if (g.defined()) g = g.detach().set_requires_grad(true);
    auto node = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " has first derivatives only", (int64_t)grads.size());
    return (*node)(std::move(grads));
}

// A backward pass under capture that comes to a leaf whose eager graph on the default stream is still alive would accumulate
// there, on a stream that cannot take part in a capture, and end the process: refused while it is still a forward pass.
void refuse_eager_graph(std::initializer_list<const Tensor*> inputs) {
    if (!at::GradMode::is_enabled() || c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
    for (const Tensor* t : inputs) {
        if (!t->defined() || !t->requires_grad() || !t->is_leaf()) continue;
        const auto node = torch::autograd::impl::try_get_grad_accumulator(*t);
        const auto stream = node ? node->stream() : std::nullopt;
        TORCH_CHECK_VALUE(!stream || stream->id() != 0, "a forward pass is captured while an eager graph of the same leaf (shape ",
                          t->sizes(), ") is alive on the default stream: drop its outputs first, or run it on another stream");
    }
}

// ------------------------------------------------------------------------------------------------- norms
struct NormHead {
    int64_t n;
    int c, hw, hidden, dtype, last, training;
    double eps, momentum;
    void fill(az_norm_args& a) const {
        a = az_norm_args{};
        a.n = n;
        a.c = c;
        a.hw = hw;
        a.hidden = hidden;
        a.dtype = dtype;
        a.channels_last = last;
        a.training = training;
        a.eps = eps;
        a.momentum = momentum;
    }
};

struct NormFunction : torch::autograd::Function<NormFunction> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x_, const MaybeTensor& residual_, const Tensor& weight, const Tensor& bias,
                          const MaybeTensor& fc1_weight, const MaybeTensor& fc1_bias, const MaybeTensor& fc2_weight,
                          const MaybeTensor& fc2_bias, const MaybeTensor& mean, const MaybeTensor& var, const MaybeTensor& batches,
                          bool training, double momentum, double eps) {
        const Tensor w1 = held(fc1_weight), b1 = held(fc1_bias), w2 = held(fc2_weight), b2 = held(fc2_bias);
        const Tensor running_mean = held(mean), running_var = held(var), num_batches = held(batches);
        const c10::DeviceGuard guard(x_.device());
        // a tensor that is contiguous both ways counts as contiguous
        const bool last = !x_.is_contiguous() && x_.is_contiguous(at::MemoryFormat::ChannelsLast);
        const auto format = last ? at::MemoryFormat::ChannelsLast : at::MemoryFormat::Contiguous;
        const Tensor x = x_.contiguous(format);
        const bool gated = w1.defined();
        const Tensor residual = gated ? residual_->contiguous(format) : Tensor();
        NormHead head = {x.size(0), (int)x.size(1), (int)(x.size(2) * x.size(3)), gated ? (int)w1.size(0) : 0, dtype_code(x), last,
                         training, eps, momentum};
        az_norm_args a;
        head.fill(a);
        int64_t sizes[3];
        check(lib.norm_sizes(&a, sizes));
        const Tensor saved = bytes(sizes[0], x), workspace = bytes(sizes[1], x);
        const Tensor out = at::empty_like(x);
        a.x_dev = x.data_ptr();
        a.residual_dev = ptr<void>(residual);
        a.weight_dev = ptr<float>(weight);
        a.bias_dev = ptr<float>(bias);
        a.running_mean_dev = ptr<float>(running_mean);
        a.running_var_dev = ptr<float>(running_var);
        a.num_batches_dev = ptr<int64_t>(num_batches);
        a.fc1_weight_dev = ptr<float>(w1);
        a.fc1_bias_dev = ptr<float>(b1);
        a.fc2_weight_dev = ptr<float>(w2);
        a.fc2_bias_dev = ptr<float>(b2);
        a.saved_dev = saved.data_ptr();
        a.workspace_dev = workspace.data_ptr();
        a.out_dev = out.data_ptr();
        check(lib.norm_forward(&a, stream_of(x)));
        if (training)                 // written behind torch's back: whoever watches version counters has to see it
            for (const Tensor* t : {&running_mean, &running_var, &num_batches})
                if (t->defined()) t->unsafeGetTensorImpl()->bump_version();
        ctx->save_for_backward({x, weight, bias, w1, b1, w2, b2, saved});
        ctx->saved_data["head"] = std::vector<int64_t>{head.n, head.c, head.hw, head.hidden, head.dtype, last, training, sizes[2]};
        ctx->saved_data["eps"] = eps;
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved_tensors = ctx->get_saved_variables();
        const Tensor &x = saved_tensors[0], &saved = saved_tensors[7];
        const auto h = ctx->saved_data["head"].toIntVector();
        const NormHead head = {h[0], (int)h[1], (int)h[2], (int)h[3], (int)h[4], (int)h[5], (int)h[6], ctx->saved_data["eps"].toDouble(), 0.0};
        const c10::DeviceGuard guard(x.device());
        variable_list out(14);
        {
            const at::NoGradGuard no_grad;
            const Tensor grad = grads[0].contiguous(head.last ? at::MemoryFormat::ChannelsLast : at::MemoryFormat::Contiguous);
            const Tensor workspace = bytes(h[7], x);
            out[0] = at::empty_like(x);
            if (head.hidden) out[1] = at::empty_like(x);
            const auto small = together({saved_tensors.begin() + 1, saved_tensors.begin() + 7}, x);
            std::copy(small.begin(), small.end(), out.begin() + 2);
            az_norm_args a;
            head.fill(a);
            a.x_dev = x.data_ptr();
            a.weight_dev = ptr<float>(saved_tensors[1]);
            a.bias_dev = ptr<float>(saved_tensors[2]);
            a.fc1_weight_dev = ptr<float>(saved_tensors[3]);
            a.fc1_bias_dev = ptr<float>(saved_tensors[4]);
            a.fc2_weight_dev = ptr<float>(saved_tensors[5]);
            a.fc2_bias_dev = ptr<float>(saved_tensors[6]);
            a.saved_dev = saved.data_ptr();
            a.workspace_dev = workspace.data_ptr();
            a.grad_dev = grad.data_ptr();
            a.dx_dev = out[0].data_ptr();
            a.dresidual_dev = ptr<void>(out[1]);
            a.dweight_dev = ptr<float>(out[2]);
            a.dbias_dev = ptr<float>(out[3]);
            a.dfc1_weight_dev = ptr<float>(out[4]);
            a.dfc1_bias_dev = ptr<float>(out[5]);
            a.dfc2_weight_dev = ptr<float>(out[6]);
            a.dfc2_bias_dev = ptr<float>(out[7]);
            check(lib.norm_backward(&a, stream_of(x)));
        }
        return first_derivatives_only(std::move(out), "a fused norm");
    }
};

Tensor parameter(const char* name, const Tensor& t, at::IntArrayRef want, const Tensor& x) {
    TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, name, " must be float32, got ", t.scalar_type());
    TORCH_CHECK_VALUE(t.sizes() == want, name, " must have shape ", want, ", got ", t.sizes());
    TORCH_CHECK_VALUE(t.device() == x.device(), name, " is on ", t.device(), ", the activations on ", x.device());
    return t.contiguous();
}

void statistic(const char* name, const MaybeTensor& t, at::IntArrayRef want, at::ScalarType type, const Tensor& x) {
    if (t.has_value())
        TORCH_CHECK_VALUE(t->scalar_type() == type && t->sizes() == want && t->device() == x.device() && t->is_contiguous(), name,
                          " must be a contiguous ", type, " tensor of shape ", want, " on ", x.device());
}

Tensor norm(const Tensor& x, const MaybeTensor& residual, const Tensor& weight, const Tensor& bias,
            const MaybeTensor& running_mean, const MaybeTensor& running_var, const MaybeTensor& w1,
            const MaybeTensor& b1, const MaybeTensor& w2, const MaybeTensor& b2, const MaybeTensor& num_batches,
            bool training, double momentum, double eps) {
    TORCH_CHECK_VALUE(residual.has_value() == w1.has_value() && residual.has_value() == b1.has_value() &&
                          residual.has_value() == w2.has_value() && residual.has_value() == b2.has_value(),
                      "a gate needs residual, fc1_weight, fc1_bias, fc2_weight and fc2_bias");
    TORCH_CHECK_VALUE(x.is_cuda(), "the fused norms need a GPU tensor, got one on ", x.device());
    TORCH_CHECK_TYPE(dtype_code(x) >= 0, "activations must be float32, bfloat16 or float16, got ", x.scalar_type());
    TORCH_CHECK_VALUE(x.dim() == 4, "activations must have shape [boards, channels, height, width], got ", x.sizes());
    TORCH_CHECK_VALUE(x.numel() > 0, "no values to normalise in shape ", x.sizes());
    const int64_t c = x.size(1);
    TORCH_CHECK_VALUE(x.size(0) <= INT32_MAX && c <= INT32_MAX && x.size(0) * c <= INT32_MAX && x.numel() / x.size(0) / c <= 1 << 24,
                      "a norm takes up to 2^31 - 1 boards times channels and 2^24 places, got shape ", x.sizes());
    TORCH_CHECK_VALUE(!training || x.numel() / c > 1, "the batch's statistics need more than one value per channel, got shape ", x.sizes());
    TORCH_CHECK_VALUE(training || (running_mean.has_value() && running_var.has_value()), "evaluation needs running statistics");
    statistic("running_mean", running_mean, {c}, at::kFloat, x);
    statistic("running_var", running_var, {c}, at::kFloat, x);
    statistic("num_batches_tracked", num_batches, {}, at::kLong, x);
    const Tensor w = parameter("weight", weight, {c}, x), b = parameter("bias", bias, {c}, x);
    refuse_eager_graph({&x, &weight, &bias});
    if (!residual)
        return NormFunction::apply(x, residual, w, b, w1, b1, w2, b2, running_mean, running_var, num_batches, training, momentum, eps);
    TORCH_CHECK_VALUE(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type() && residual->device() == x.device(),
                      "residual must be like x (", x.sizes(), ", ", x.scalar_type(), ", ", x.device(), "), got ", residual->sizes(), ", ",
                      residual->scalar_type(), ", ", residual->device());
    TORCH_CHECK_VALUE(w1->dim() == 2, "fc1_weight must have shape [hidden, channels], got ", w1->sizes());
    const int64_t hidden = w1->size(0);
    TORCH_CHECK_VALUE(hidden >= 1 && hidden <= 1024 && c <= 1024, "a gate takes up to 1024 channels and 1 to 1024 hidden units, got ", c,
                      " and ", hidden);
    refuse_eager_graph({&*residual, &*w1, &*b1, &*w2, &*b2});
    const MaybeTensor p1 = parameter("fc1_weight", *w1, {hidden, c}, x), p2 = parameter("fc1_bias", *b1, {hidden}, x);
    const MaybeTensor p3 = parameter("fc2_weight", *w2, {2 * c, hidden}, x), p4 = parameter("fc2_bias", *b2, {2 * c}, x);
    return NormFunction::apply(x, residual, w, b, p1, p2, p3, p4, running_mean, running_var, num_batches, training, momentum, eps);
}

// -------------------------------------------------------------------------------------------------- loss
struct LossFunction : torch::autograd::Function<LossFunction> {
    static az_loss_args arguments(const Tensor& policy, const Tensor& wl, const Tensor& target_pi, const Tensor& target_wl,
                                  const Tensor& mask, const Tensor& stats) {
        az_loss_args a{};
        a.n = policy.size(0);
        a.actions = (int)policy.size(1);
        a.outcomes = (int)wl.size(1);
        a.dtype = dtype_code(policy);
        a.policy_dev = policy.data_ptr();
        a.wl_dev = wl.data_ptr();
        a.target_pi_dev = ptr<float>(target_pi);
        a.target_wl_dev = ptr<float>(target_wl);
        a.mask_dev = ptr<uint8_t>(mask);
        a.stats_dev = ptr<float>(stats);
        return a;
    }

    static variable_list forward(AutogradContext* ctx, const Tensor& policy, const Tensor& wl, const Tensor& target_pi,
                                 const Tensor& target_wl, const MaybeTensor& mask_, bool differentiated) {
        const Tensor mask = held(mask_);
        const c10::DeviceGuard guard(policy.device());
        const Tensor losses = floats(3, policy), stats = floats(8 * policy.size(0), policy);
        az_loss_args a = arguments(policy, wl, target_pi, target_wl, mask, stats);
        a.losses_dev = ptr<float>(losses);
        if (differentiated && lib.loss_ready(&a)) {
            const Tensor dpolicy = at::empty_like(policy), dwl = at::empty_like(wl);
            a.dpolicy_dev = dpolicy.data_ptr();
            a.dwl_dev = dwl.data_ptr();
            ctx->saved_data["grads"] = std::vector<Tensor>{dpolicy, dwl};
        }
        check(lib.loss_forward(&a, stream_of(policy)));
        ctx->save_for_backward({policy, wl, target_pi, target_wl, mask, stats});
        ctx->set_materialize_grads(false);
        return {part_of(losses, 0, {}, {}), part_of(losses, 1, {}, {}), part_of(losses, 2, {}, {})};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const c10::DeviceGuard guard(s[0].device());
        variable_list out(6);
        {
            const at::NoGradGuard no_grad;
            az_loss_args a = arguments(s[0], s[1], s[2], s[3], s[4], s[5]);
            // the forward pass's gradients serve one backward pass (they belong to whoever gets them)
            static std::mutex taking;
            {
                const std::lock_guard<std::mutex> lock(taking);
                const auto ready = ctx->saved_data.find("grads");
                if (ready != ctx->saved_data.end()) {
                    const auto held = ready->second.toTensorVector();
                    out[0] = held[0];
                    out[1] = held[1];
                    a.grads_ready = 1;
                    ctx->saved_data.erase(ready);
                }
            }
            if (!a.grads_ready) {
                out[0] = at::empty_like(s[0]);
                out[1] = at::empty_like(s[1]);
            }
            for (int i = 0; i < 3; ++i) a.upstream_dev[i] = ptr<float>(grads[i]);
            a.dpolicy_dev = out[0].data_ptr();
            a.dwl_dev = out[1].data_ptr();
            check(lib.loss_backward(&a, stream_of(s[0])));
            if (!grads[0].defined()) {           // a head whose loss is not used gets none (and no 0 times NaN)
                if (!grads[1].defined()) out[0] = Tensor();
                if (!grads[2].defined()) out[1] = Tensor();
            }
        }
        return first_derivatives_only(std::move(out), "policy_value_loss");
    }
};

py::tuple policy_value_loss(const Tensor& policy, const Tensor& wl, const Tensor& target_pi, const Tensor& target_wl,
                            const MaybeTensor& mask) {
    TORCH_CHECK_VALUE(policy.is_cuda(), "policy_value_loss needs GPU tensors, got one on ", policy.device());
    TORCH_CHECK_TYPE(dtype_code(policy) >= 0 && wl.scalar_type() == policy.scalar_type(),
                     "logits must be both float32, both bfloat16 or both float16, got ", policy.scalar_type(), " and ", wl.scalar_type());
    TORCH_CHECK_VALUE(policy.dim() == 2 && wl.dim() == 2 && policy.size(0) == wl.size(0), "logits must be [n, actions] and [n, outcomes], got ",
                      policy.sizes(), " and ", wl.sizes());
    TORCH_CHECK_VALUE(policy.numel() > 0 && wl.numel() > 0, "policy_value_loss of no rows or no classes");
    TORCH_CHECK_VALUE(wl.size(1) <= 4096, "up to 4096 outcomes, got ", wl.size(1));
    TORCH_CHECK_VALUE(policy.size(0) <= 1 << 28 && policy.size(1) <= 1 << 28, "up to 2^28 rows and actions, got ", policy.sizes());
    const std::tuple<const char*, const Tensor*, const Tensor*> targets[] = {{"target_pis", &target_pi, &policy}, {"target_wls", &target_wl, &wl}};
    for (const auto& [name, t, like] : targets) {
        TORCH_CHECK_TYPE(t->scalar_type() == at::kFloat, name, " must be float32, got ", t->scalar_type());
        TORCH_CHECK_VALUE(t->sizes() == like->sizes(), name, " must have the logits' shape ", like->sizes(), ", got ", t->sizes());
        TORCH_CHECK_VALUE(!t->requires_grad(), name, " must not require a gradient");
    }
    if (mask)
        TORCH_CHECK_VALUE((mask->scalar_type() == at::kBool || mask->scalar_type() == at::kByte) && mask->sizes() == policy.sizes(),
                          "mask must be bool or uint8 of shape ", policy.sizes(), ", got ", mask->scalar_type(), " ", mask->sizes());
    TORCH_CHECK_VALUE(wl.device() == policy.device() && target_pi.device() == policy.device() && target_wl.device() == policy.device() &&
                          (!mask || mask->device() == policy.device()),
                      "all tensors must be on ", policy.device());
    refuse_eager_graph({&policy, &wl});
    const auto r = LossFunction::apply(policy.contiguous(), wl.contiguous(), target_pi.contiguous(), target_wl.contiguous(),
                                       mask ? MaybeTensor(mask->contiguous()) : mask,
                                       at::GradMode::is_enabled() && (policy.requires_grad() || wl.requires_grad()));
    return py::make_tuple(r[0], r[1], r[2]);
}

// --------------------------------------------------------------------------------------------- optimiser
// Whether two layouts of one shape put every element at the same place.
bool same_places(const Tensor& a, at::IntArrayRef strides) {
    if (a.strides() == strides) return true;
    for (int64_t i = 0; i < a.dim(); ++i)
        if (a.size(i) > 1 && a.stride(i) != strides[i]) return false;
    return true;
}

class AdamPlan {
  public:
    // Lays out the moments of the parameters; attach() gives it the buffers.
    explicit AdamPlan(std::vector<Tensor> params) : params_(std::move(params)), offsets_(params_.size() + 1) {
        for (const Tensor& p : params_) {
            sizes_.push_back(p.numel());
            strides_.push_back(p.strides().vec());
        }
        const int32_t count = (int32_t)params_.size();
        const int64_t n = lib.adam_plan(count, sizes_.data(), offsets_.data(), nullptr);
        check(n < 0 ? (int)n : AZ_OK);
        Tensor pieces = at::empty({n * (int64_t)sizeof(az_adam_piece)}, at::kByte);
        lib.adam_plan(count, sizes_.data(), nullptr, (az_adam_piece*)pieces.data_ptr());
        n_pieces_ = n;
        pieces_ = pieces.to(params_.at(0).device());
    }

    std::vector<int64_t> offsets() const { return offsets_; }

    void attach(int bits, uint64_t seed, Tensor step, Tensor m, Tensor v, MaybeTensor m_scale, MaybeTensor v_scale, Tensor norm) {
        bits_ = bits;
        seed_ = seed;
        step_ = step;
        m_ = m;
        v_ = v;
        m_scale_ = held(m_scale);
        v_scale_ = held(v_scale);
        norm_ = norm;
    }

    // One step over every parameter that has a gradient.
    void step(const std::vector<az_adam_group>& groups, double max_norm) {
        const at::NoGradGuard no_grad;
        const c10::DeviceGuard guard(step_.device());
        void* stream = stream_of(step_);
        const size_t count = params_.size();
        std::vector<uint64_t> params(count), grads(count);
        std::vector<Tensor> copies;                  // gradients brought into their parameter's memory order
        bool any = false;
        for (size_t i = 0; i < count; ++i) {
            const Tensor& p = params_[i];
            TORCH_CHECK_VALUE(p.scalar_type() == at::kFloat && p.device() == step_.device() && p.numel() == sizes_[i], "a parameter became ",
                              p.scalar_type(), " ", p.sizes(), " on ", p.device(), " after FusedAdam was built");
            TORCH_CHECK_VALUE(p.dim() == (int64_t)strides_[i].size() && same_places(p, strides_[i]),
                              "a parameter's strides changed after FusedAdam was built: its moments are in the old order");
            const Tensor& held_grad = p.grad();
            if (!held_grad.defined() || sizes_[i] == 0) continue;
            Tensor g = held_grad;
            TORCH_CHECK_VALUE(g.layout() == at::kStrided, "FusedAdam takes dense gradients");
            TORCH_CHECK_VALUE(g.scalar_type() == at::kFloat && g.device() == step_.device() && g.sizes() == p.sizes(),
                              "the gradient of a parameter of shape ", p.sizes(), " is ", g.scalar_type(), " ", g.sizes(), " on ", g.device());
            if (!same_places(g, p.strides())) {
                g = at::empty_strided(p.sizes(), p.strides(), g.options()).copy_(g);
                copies.push_back(g);
            }
            params[i] = (uint64_t)p.data_ptr();
            grads[i] = (uint64_t)g.data_ptr();
            any = true;
        }
        if (!any) return;
        const Tensor scratch = bytes(lib.adam_scratch((int32_t)count), step_);
        az_adam_config c{};
        c.max_norm = max_norm > 0 ? max_norm : 0.0;
        c.state_bits = bits_;
        c.seed = seed_;
        c.pieces_dev = (const az_adam_piece*)pieces_.data_ptr();
        c.m_dev = m_.data_ptr();
        c.v_dev = v_.data_ptr();
        c.m_scale_dev = ptr<float>(m_scale_);
        c.v_scale_dev = ptr<float>(v_scale_);
        c.steps_dev = ptr<float>(step_);
        c.norm_dev = ptr<float>(norm_);
        c.scratch_dev = scratch.data_ptr();
        check(lib.adam_step(&c, (int32_t)groups.size(), groups.data(), (int32_t)count, params.data(), grads.data(), sizes_.data(), stream));
        // written behind torch's back: whoever watches version counters has to see it
        for (size_t i = 0; i < count; ++i)
            if (grads[i]) params_[i].unsafeGetTensorImpl()->bump_version();
        for (const Tensor* t : {&step_, &m_, &v_, &m_scale_, &v_scale_, &norm_})
            if (t->defined()) t->unsafeGetTensorImpl()->bump_version();
    }

  private:
    std::vector<Tensor> params_;
    std::vector<int64_t> sizes_, offsets_;
    std::vector<std::vector<int64_t>> strides_;
    int64_t n_pieces_ = 0;
    Tensor pieces_;
    int bits_ = 32;
    uint64_t seed_ = 0;
    Tensor step_, m_, v_, m_scale_, v_scale_, norm_;
};

template <typename F>
void set(F& f, const py::dict& addresses, const char* name) { f = (F)addresses[name].cast<uintptr_t>(); }

}  // namespace

PYBIND11_MODULE(_azops, m) {
    // addresses of the library's entries, and the exception that their errors become
    m.def("bind", [](const py::dict& a, py::object error) {
        set(lib.last_error, a, "az_last_error");
        set(lib.norm_sizes, a, "az_norm_sizes");
        set(lib.norm_forward, a, "az_norm_forward");
        set(lib.norm_backward, a, "az_norm_backward");
        set(lib.loss_ready, a, "az_policy_value_loss_ready");
        set(lib.loss_forward, a, "az_policy_value_loss_forward");
        set(lib.loss_backward, a, "az_policy_value_loss_backward");
        set(lib.adam_plan, a, "az_adam_plan");
        set(lib.adam_scratch, a, "az_adam_scratch");
        set(lib.adam_step, a, "az_adam_step");
        az_error = error.release().ptr();
    });
    m.def("norm", torch::wrap_pybind_function(norm));
    m.def("policy_value_loss", torch::wrap_pybind_function(policy_value_loss));
    py::class_<AdamPlan>(m, "AdamPlan")
        .def(py::init<std::vector<Tensor>>())
        .def("offsets", &AdamPlan::offsets)
        .def("attach", &AdamPlan::attach)
        .def("step", [](AdamPlan& self, const std::vector<std::tuple<double, double, double, double, double, bool, int>>& groups,
                        double max_norm) {          // (lr, beta1, beta2, eps, weight_decay, decoupled, end)
            std::vector<az_adam_group> g;
            for (const auto& t : groups) g.push_back(std::apply([](auto... v) { return az_adam_group{v...}; }, t));
            torch::wrap_pybind_function([&] { self.step(g, max_norm); })();
        });
}
