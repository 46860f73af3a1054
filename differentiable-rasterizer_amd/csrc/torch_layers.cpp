// The network layers as torch operations: argument checks, outputs and workspaces from
// torch's allocator, torch's current stream, and the autograd nodes, over the C ABI
// (include/diffrast_hip.h). diffrast/layers.py documents them.
//
// Native, because a training step of small layers is bound by the host: the autograd
// engine runs a backward pass on a thread of its own, where a Python function starts with
// cold caches and waits for the interpreter's lock. A layer norm's forward and backward
// (16384 x 1024, 40 us on the GPU) took 146 us as a torch.autograd.Function and take 67 so.

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <mutex>
#include <optional>
#include <string>
#include <vector>

#include "diffrast_hip.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using Optional = std::optional<Tensor>;

const Tensor& undefined() {
    static const Tensor none;
    return none;
}
const Tensor& of(const Optional& t) { return t.has_value() ? *t : undefined(); }

// diffrast._lib.DiffrastError where there is a Python caller to see it, else (the
// autograd engine's threads) a runtime error of the same text.
void check(int rc) {
    if (rc == DRH_OK) return;
    static const char* names[] = {"", "NoDevice", "Timeout", "Device", "Readback", "TooLarge", "InvalidArgument"};
    const std::string text = drh_last_error();
    if (PyGILState_Check()) {
        py::object type = py::module_::import("diffrast._lib").attr("DiffrastError");
        PyErr_SetObject(type.ptr(), type(rc, text).ptr());
        throw py::error_already_set();
    }
    throw std::runtime_error(std::string(rc >= 1 && rc <= 6 ? names[rc] : "error") + ": " + text);
}

// The layers' context on a device. They keep no state in it, so one per device lives as
// long as the process.
drh_ctx* context(c10::DeviceIndex device) {
    static std::mutex mu;
    static std::vector<drh_ctx*> all;
    std::lock_guard<std::mutex> g(mu);
    if ((size_t)device >= all.size()) all.resize(device + 1, nullptr);
    if (!all[device]) check(drh_create(&all[device]));  // binds the current device: the caller's guard
    return all[device];
}

struct Call {
    c10::DeviceGuard guard;
    drh_ctx* ctx;
    void* stream;
    explicit Call(const Tensor& x)
        : guard(x.device()),
          ctx(context(x.device().index())),
          stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream()) {}
};

int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return DRH_F32;
        case at::kBFloat16: return DRH_BF16;
        case at::kHalf: return DRH_F16;
        default:
            TORCH_CHECK_VALUE(false, "expected float32, bfloat16 or float16, got ", t.scalar_type());
    }
}

// t as (rows, features) with contiguous features: a view where its strides allow.
Tensor as_rows(const Tensor& t) {
    if (t.dim() == 2 && t.is_contiguous()) return t;
    Tensor v = t;
    if (t.dim() != 2) {
        int64_t rows = 1;
        for (int64_t i = 0; i + 1 < t.dim(); i++) rows *= t.size(i);
        v = t.reshape({rows, t.size(-1)});
    }
    if (v.stride(1) != 1 || (v.size(0) > 1 && v.stride(0) < v.size(1))) v = v.contiguous();
    return v;
}

// Elements between the rows of as_rows' view; one row has no stride of its own.
int64_t row_stride(const Tensor& v) { return v.size(0) > 1 ? v.stride(0) : v.size(1); }

const void* in(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor flat(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

Tensor workspace(uint64_t bytes, const Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

bool wants_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// The layers are no operators that torch's dispatcher sees: a trace would record the output's
// allocation alone.
void refuse_tracing() {
    using c10::impl::TorchDispatchModeKey;
    using c10::impl::TorchDispatchModeTLS;
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() && !TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY) &&
                                    !TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::FAKE) &&
                                    !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch),
                                "the network layers cannot be traced (torch.jit.trace, make_fx, fake tensors)");
}

// Nor have they tangents: without this a derivative in forward mode would be zero.
void refuse_transforms(std::initializer_list<const Tensor*> ts) {
    refuse_tracing();
    if (!at::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor* t : ts)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(),
                                    "the network layers have no forward-mode derivative");
}

// Whether every tensor is on the GPU that x is on; if not, they are moved there (to the
// current GPU where x is on none). A tensor that torch negates when it is read (the imaginary
// part of a conjugate) is negated here: kernels read memory as it stands.
bool together(std::initializer_list<Tensor*> ts) {
    Tensor& x = **ts.begin();
    for (Tensor* t : ts)
        if (t->defined() && t->is_neg()) *t = t->resolve_neg();
    bool same = x.is_cuda();
    for (Tensor* t : ts) same = same && (!t->defined() || t->device() == x.device());
    if (same) return true;
    at::Device dev = x.device();
    if (!x.is_cuda()) {
        if (!at::hasCUDA() || c10::impl::VirtualGuardImpl(at::kCUDA).deviceCount() == 0)
            throw std::runtime_error("no HIP device is visible; there is no CPU path");
        dev = at::Device(at::kCUDA, c10::impl::VirtualGuardImpl(at::kCUDA).getDevice().index());
    }
    for (Tensor* t : ts)
        if (t->defined()) *t = t->to(dev);
    return false;
}

// A tensor kept for the backward pass. What comes back may be a user's (a saved-tensor hook's): a
// kernel is given nothing but what went in's type, shape and GPU.
class Kept {
    SavedVariable saved_;
    at::TensorOptions options_;
    c10::DimVector sizes_;
    bool holds_ = false;

public:
    void keep(const Tensor& t) {
        saved_ = SavedVariable(t, false);
        options_ = t.options();
        sizes_ = c10::DimVector(t.sizes());
        holds_ = true;
    }
    // Undefined where nothing was kept.
    Tensor get() const {
        if (!holds_) return Tensor();
        const Tensor t = saved_.unpack();
        TORCH_CHECK(t.defined() && t.sizes() == c10::IntArrayRef(sizes_) && t.scalar_type() == options_.dtype().toScalarType() &&
                        t.device() == options_.device() && t.layout() == at::kStrided,
                    "a tensor saved for a layer's backward pass came back as another type, shape or device");
        return t.resolve_neg();
    }
    void release() { saved_.reset_data(); }
};

// The history of a gradient that was made with a graph asked for: raises for whoever
// differentiates it. It leads to all that the gradient depends on (the layer's inputs and the
// gradient that came in), since the engine skips what is on no path to the inputs asked for.
struct DifferentiatedAgain : Node {
    std::string name() const override { return "DiffrastDifferentiatedAgain"; }
    variable_list apply(variable_list&&) final {
        throw std::runtime_error("this layer can be differentiated once only");
    }
};

// A node of a layer that is differentiable once.
struct OnceNode : Node {
    variable_list apply(variable_list&& grads) final {
        std::lock_guard<std::mutex> lock(mutex_);
        refuse_transforms({&grads[0]});
        if (grads[0].defined()) {  // the engine sees to this, but a node's own hooks come after it
            const auto& meta = input_metadata(0);
            TORCH_CHECK(meta.is_same_shape(grads[0]) && grads[0].device() == meta.device() && grads[0].layout() == at::kStrided &&
                            grads[0].scalar_type() == meta.dtype().toScalarType(),
                        "the gradient of a layer's output is of another type, shape or device than the output");
        }
        variable_list r;
        {
            at::NoGradGuard no;
            r = grads[0].defined() ? gradients(grads[0].resolve_neg()) : variable_list(num_outputs());
        }
        if (at::GradMode::is_enabled() && grads[0].defined()) {
            torch::autograd::edge_list edges = next_edges();
            edges.push_back(torch::autograd::impl::gradient_edge(grads[0]));
            auto error = std::shared_ptr<Node>(new DifferentiatedAgain(), torch::autograd::deleteNode);
            error->set_next_edges(std::move(edges));
            for (Tensor& t : r)
                if (t.defined()) {
                    t = t.detach();
                    torch::autograd::set_history(t, error);
                }
        }
        return r;
    }
    virtual variable_list gradients(const Tensor& g) = 0;
};

// y as the output of `node`, whose inputs are `inputs` in the order of its gradients.
template <class N>
Tensor attach(Tensor y, std::shared_ptr<N> node, std::initializer_list<const Tensor*> inputs) {
    torch::autograd::edge_list edges;
    for (const Tensor* t : inputs)
        edges.push_back(t->defined() ? torch::autograd::impl::gradient_edge(*t) : torch::autograd::Edge());
    node->set_next_edges(std::move(edges));
    torch::autograd::set_history(y, node);
    return y;
}

template <class N>
std::shared_ptr<N> new_node() {
    return std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
}

// ---------------------------------------------------------------- layer norm

// Keeps what the gradients that are wanted need: weight where dx is, never the bias.
struct LayerNormBackward : OnceNode {
    Kept x_, weight_, stats_;
    at::ScalarType weight_type = at::kFloat;  // and the bias's
    int weight_code = DRH_F32;

    std::string name() const override { return "DiffrastLayerNormBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x_.release();
        weight_.release();
        stats_.release();
    }

    variable_list gradients(const Tensor& g) override {
        const Tensor x = x_.get(), stats = stats_.get().contiguous(), w = weight_.get();
        const Tensor xv = as_rows(x), gv = as_rows(g), wv = flat(w);
        const int64_t rows = xv.size(0), cols = xv.size(1);
        variable_list r(3);
        if (task_should_compute_output(0)) r[0] = at::empty(g.sizes(), x.options());
        for (int i : {1, 2})
            if (task_should_compute_output(i)) r[i] = at::empty({cols}, x.options().dtype(weight_type));
        uint64_t bytes = 0;
        if (r[1].defined() || r[2].defined()) check(drh_layer_norm_backward_bytes(rows, cols, dtype_code(x), &bytes));
        const Tensor ws = workspace(bytes, x);
        const float* mean = stats.const_data_ptr<float>();
        Call call(x);
        check(drh_layer_norm_backward(call.ctx, in(xv), in(wv), mean, mean + rows, in(gv), rows, cols, row_stride(xv),
                                      row_stride(gv), dtype_code(x), weight_code, out(r[0]), out(r[1]), out(r[2]), out(ws),
                                      bytes, call.stream, 0));
        return r;
    }
};

Tensor layer_norm(Tensor x, const Optional& weight, const Optional& bias, double eps) {
    Tensor w = of(weight), b = of(bias);
    const int code = dtype_code(x);
    const int64_t cols = x.dim() ? x.size(-1) : 0;
    TORCH_CHECK_VALUE(cols > 0, "expected x of shape (..., D), got ", x.sizes());
    TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative");
    auto vector = [&](const Tensor& t, const char* name) {
        if (!t.defined()) return;
        TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == cols, "expected ", name, " of shape (", cols, ",), got ", t.sizes());
        TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat, "expected ", name, " in ",
                          x.scalar_type(), " or float32, got ", t.scalar_type());
    };
    vector(w, "weight");
    vector(b, "bias");
    TORCH_CHECK_VALUE(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), "weight is ", w.scalar_type(),
                      " but bias ", b.scalar_type());
    refuse_transforms({&x, &w, &b});
    const at::Device home = x.device();
    if (!together({&x, &w, &b})) return layer_norm(x, w.defined() ? Optional(w) : std::nullopt,
                                                   b.defined() ? Optional(b) : std::nullopt, eps).to(home);
    const bool grad = wants_grad({&x, &w, &b});
    const at::ScalarType wtype = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type();
    const int wcode = w.defined() ? dtype_code(w) : b.defined() ? dtype_code(b) : code;
    Tensor y, stats;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor xv = as_rows(x), wv = flat(w), bv = flat(b);
        const int64_t rows = xv.size(0);
        y = at::empty(x.sizes(), x.options());
        float* mean = nullptr;
        if (grad) {
            stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
            mean = stats.mutable_data_ptr<float>();
        }
        Call call(x);
        check(drh_layer_norm(call.ctx, in(xv), in(wv), in(bv), rows, cols, row_stride(xv), code, wcode, (float)eps, out(y),
                             mean, mean ? mean + rows : nullptr, call.stream, 0));
    }
    if (!grad) return y;
    auto node = new_node<LayerNormBackward>();
    node->x_.keep(x);
    node->stats_.keep(stats);
    if (w.defined() && x.requires_grad()) node->weight_.keep(w);
    node->weight_type = wtype;
    node->weight_code = wcode;
    return attach(std::move(y), std::move(node), {&x, &w, &b});
}

// ---------------------------------------------------------------- linear

// Keeps what the gradients that are wanted need: x where dW is, the weight where dx is, the
// slopes where any is but the residual's.
struct LinearBackward : OnceNode {
    Kept x_, weight_, slopes_;
    std::vector<int64_t> x_sizes;
    at::TensorOptions options;
    int64_t rows = 0, n_out = 0, n_in = 0;
    int act = 0, code = 0;

    std::string name() const override { return "DiffrastLinearBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x_.release();
        weight_.release();
        slopes_.release();
    }

    variable_list gradients(const Tensor& grad) override {
        const Tensor x = x_.get(), w = weight_.get(), kept = flat(slopes_.get());
        const Tensor xv = x.defined() ? as_rows(x) : x, wv = w.defined() ? as_rows(w) : w;
        const Tensor g = flat(grad);
        variable_list r(4);
        if (task_should_compute_output(0)) r[0] = at::empty(x_sizes, options);
        if (task_should_compute_output(1)) r[1] = at::empty({n_out, n_in}, options);
        if (task_should_compute_output(2)) r[2] = at::empty({n_out}, options);
        if (task_should_compute_output(3)) r[3] = grad;
        if (!r[0].defined() && !r[1].defined() && !r[2].defined()) return r;
        const int64_t xs = xv.defined() ? row_stride(xv) : n_in, ws = wv.defined() ? row_stride(wv) : n_in;
        uint64_t bytes = 0;
        check(drh_linear_backward_bytes(rows, n_out, n_in, xs, ws, code, act, &bytes));
        const Tensor space = workspace(bytes, g);
        Call call(g);
        check(drh_linear_backward(call.ctx, in(xv), in(wv), in(kept), in(g), rows, n_out, n_in, xs, ws, code, act, out(r[0]),
                                  out(r[1]), out(r[2]), out(space), bytes, call.stream, 0));
        return r;
    }
};

Tensor linear(Tensor x, Tensor w, const Optional& bias, int act, const Optional& residual) {
    Tensor b = of(bias), res = of(residual);
    const int code = dtype_code(x);
    TORCH_CHECK_VALUE(x.dim() >= 1 && w.dim() == 2 && w.size(1) == x.size(-1) && w.size(0) > 0,
                      "expected x (..., K) and weight (N, K), got ", x.sizes(), " and ", w.sizes());
    const int64_t n_out = w.size(0), n_in = w.size(1);
    c10::DimVector shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n_out;
    TORCH_CHECK_VALUE(!b.defined() || (b.dim() == 1 && b.size(0) == n_out), "expected bias of shape (", n_out, ",), got ",
                      b.sizes());
    TORCH_CHECK_VALUE(!res.defined() || res.sizes() == c10::IntArrayRef(shape), "expected residual of shape ",
                      c10::IntArrayRef(shape), ", got ", res.sizes());
    auto typed = [&](const Tensor& t, const char* name) {
        TORCH_CHECK_VALUE(!t.defined() || t.scalar_type() == x.scalar_type(), "x is ", x.scalar_type(), " but ", name, " ",
                          t.scalar_type());
    };
    typed(w, "weight");
    typed(b, "bias");
    typed(res, "residual");
    refuse_transforms({&x, &w, &b, &res});
    const at::Device home = x.device();
    if (!together({&x, &w, &b, &res}))
        return linear(x, w, b.defined() ? Optional(b) : std::nullopt, act, res.defined() ? Optional(res) : std::nullopt)
            .to(home);
    const bool grad = wants_grad({&x, &w, &b, &res}), keep = act != DRH_ACT_NONE && wants_grad({&x, &w, &b});
    Tensor y, kept;
    int64_t rows = 0;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        const Tensor xv = as_rows(x), wv = as_rows(w), bv = flat(b), rv = flat(res);
        rows = xv.size(0);
        const int64_t xs = row_stride(xv), ws = row_stride(wv);
        y = at::empty(shape, x.options());
        if (keep) kept = at::empty({rows, n_out}, x.options().dtype(code == DRH_F32 ? at::kFloat : at::kHalf));
        uint64_t bytes = 0;
        check(drh_linear_bytes(rows, n_out, n_in, xs, ws, code, &bytes));
        const Tensor space = workspace(bytes, x);
        Call call(x);
        check(drh_linear(call.ctx, in(xv), in(wv), in(bv), in(rv), rows, n_out, n_in, xs, ws, code, act, out(y), out(kept),
                         out(space), bytes, call.stream, 0));
    }
    if (!grad) return y;
    auto node = new_node<LinearBackward>();
    if (w.requires_grad()) node->x_.keep(x);
    if (x.requires_grad()) node->weight_.keep(w);
    node->x_sizes = x.sizes().vec();
    node->options = x.options();
    node->rows = rows, node->n_out = n_out, node->n_in = n_in;
    node->act = act, node->code = code;
    if (keep) node->slopes_.keep(kept);
    return attach(std::move(y), std::move(node), {&x, &w, &b, &res});
}

// ---------------------------------------------------------------- dropout

Tensor drop(const Tensor& x_, const Tensor& res, double p, uint64_t seed, uint64_t offset) {
    const Tensor x = x_.contiguous(), r = flat(res);
    Tensor y = at::empty(x.sizes(), x.options());
    Call call(x);
    check(drh_dropout(call.ctx, in(x), in(r), x.numel(), dtype_code(x), p, seed, offset, out(y), call.stream, 0));
    return y;
}

struct DropoutBackward : OnceNode {
    double p = 0;
    uint64_t seed = 0, offset = 0;
    std::string name() const override { return "DiffrastDropoutBackward"; }
    variable_list gradients(const Tensor& g) override {
        variable_list r(2);
        if (task_should_compute_output(0)) r[0] = drop(g, undefined(), p, seed, offset);
        if (task_should_compute_output(1)) r[1] = g;
        return r;
    }
};

Tensor dropout(Tensor x, double p, uint64_t seed, uint64_t offset, const Optional& residual) {
    Tensor res = of(residual);
    dtype_code(x);
    TORCH_CHECK_VALUE(p >= 0.0 && p < 1.0, "p must be in [0, 1)");
    TORCH_CHECK_VALUE(!res.defined() || (res.sizes() == x.sizes() && res.scalar_type() == x.scalar_type()),
                      "expected a residual of shape ", x.sizes(), " in ", x.scalar_type(), ", got ",
                      res.defined() ? res.sizes() : x.sizes(), " in ", res.defined() ? res.scalar_type() : x.scalar_type());
    refuse_transforms({&x, &res});
    const at::Device home = x.device();
    if (!together({&x, &res})) return dropout(x, p, seed, offset, res.defined() ? Optional(res) : std::nullopt).to(home);
    const bool grad = wants_grad({&x, &res});
    Tensor y;
    {
        at::AutoDispatchBelowADInplaceOrView below;
        y = drop(x, res, p, seed, offset);
    }
    if (!grad) return y;
    auto node = new_node<DropoutBackward>();
    node->p = p;
    node->seed = seed;
    node->offset = offset;
    return attach(std::move(y), std::move(node), {&x, &res});
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.def("layer_norm", &layer_norm);
    m.def("linear", &linear);
    m.def("dropout", &dropout);
}
