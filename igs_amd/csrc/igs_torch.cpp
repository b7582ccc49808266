// igs_torch.cpp -- torch side of the feature operators: allocation, the current stream and the autograd
// nodes, around the C ABI of libigs_hip.so (include/igs_hip.h).
//
// A training step of a small problem is bound by the host, and most of that by the backward: the engine
// runs it on a thread of its own, where every Python-level step costs two to three times what it does on
// the caller's (embedding lookup with gradient, 8 x 64: 85 us a step with autograd nodes in Python, layer
// norm 112 us; 50 and 68 us for torch's own nodes).  So these nodes are native.  The library is not linked
// but resolved from the handle that the ctypes binding has open, so both use the same one.
#include <torch/extension.h>

#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <optional>
#include <tuple>

#include "igs_hip.h"

namespace {
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct Library {
    decltype(&igs_status_string) status_string = nullptr;
    decltype(&igs_embedding_forward) embedding_forward = nullptr;
    decltype(&igs_embedding_plan) embedding_plan = nullptr;
    decltype(&igs_embedding_backward) embedding_backward = nullptr;
    decltype(&igs_dropout) dropout = nullptr;
    decltype(&igs_layer_norm_forward) layer_norm_forward = nullptr;
    decltype(&igs_layer_norm_plan) layer_norm_plan = nullptr;
    decltype(&igs_layer_norm_backward) layer_norm_backward = nullptr;
} lib;

template <class F>
void resolve(void* handle, const char* name, F& f) {
    f = reinterpret_cast<F>(dlsym(handle, name));
    TORCH_CHECK(f, "the library does not export ", name);
}

void bind(int64_t handle) {
    void* h = reinterpret_cast<void*>(handle);
    resolve(h, "igs_status_string", lib.status_string);
    resolve(h, "igs_embedding_forward", lib.embedding_forward);
    resolve(h, "igs_embedding_plan", lib.embedding_plan);
    resolve(h, "igs_embedding_backward", lib.embedding_backward);
    resolve(h, "igs_dropout", lib.dropout);
    resolve(h, "igs_layer_norm_forward", lib.layer_norm_forward);
    resolve(h, "igs_layer_norm_plan", lib.layer_norm_plan);
    resolve(h, "igs_layer_norm_backward", lib.layer_norm_backward);
}

void check(int rc, const char* what) {
    TORCH_CHECK(rc == 0, what, " failed: ", lib.status_string(rc), " (status ", rc, ")");
}

int dtype_code(at::ScalarType type) {
    switch (type) {
        case at::kFloat: return IGS_F32;
        case at::kHalf: return IGS_F16;
        case at::kBFloat16: return IGS_BF16;
        default: return -1;  // the library refuses it
    }
}
int dtype_code(const Tensor& t) { return dtype_code(t.scalar_type()); }

const void* address(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* writable(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor value(const OptTensor& t) { return t ? *t : Tensor(); }
const uint64_t* seed_address(const Tensor& t) { return static_cast<const uint64_t*>(address(t)); }
void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// A row length as the library takes it; one beyond its range is refused there.
int width(int64_t D) { return D > 0x7FFFFFFF ? -1 : static_cast<int>(D); }

Tensor workspace(uint64_t bytes, const Tensor& like) {
    return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}

// What the kernels read are a tensor's bytes: a negation that is yet to be done (the imaginary part of a conjugate) is
// done first.  contiguous() leaves it where it copies nothing.
Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous().resolve_neg() : t; }

// (x or a contiguous copy, distance of its rows in elements): rows of the last axis are taken where they are if they
// are dense and evenly spaced (slices of the last axis, expanded batches).
std::tuple<Tensor, int64_t> rows_of(const Tensor& x) {
    const int64_t D = x.size(-1);
    if (x.is_neg()) return {dense(x), D};
    if (x.is_contiguous()) return {x, D};
    if (D != 1 && x.stride(-1) != 1) return {x.contiguous(), D};
    int64_t step = -1, span = -1;
    for (int64_t d = x.dim() - 2; d >= 0; --d) {
        const int64_t n = x.size(d), s = x.stride(d);
        if (n == 1) continue;
        if (span < 0) step = s;
        else if (s != span) return {x.contiguous(), D};
        span = s * n;
    }
    return {x, step < 0 ? D : step};
}

// The registered operators can be called directly, so what would make a kernel read beside a tensor is checked here.
void same_device(const Tensor& a, const Tensor& b, const char* what) {
    TORCH_CHECK(!b.defined() || b.device() == a.device(), "Expected all tensors to be on the same device, but ", what, " is on ",
                b.defined() ? b.device() : a.device(), " and the first tensor on ", a.device());
}
void check_tokens(const Tensor& tokens) {
    TORCH_CHECK(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt, "tokens must be int32 or int64");
}
void check_weights(const Tensor& x, const Tensor& weight, const Tensor& bias) {
    for (const Tensor* t : {&weight, &bias})
        if (t->defined()) {
            same_device(x, *t, "a weight");
            TORCH_CHECK(t->dim() == 1 && t->size(0) == x.size(-1), "weight and bias must be [", x.size(-1), "]");
        }
    TORCH_CHECK(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(),
                "weight and bias must have one type");
}
void check_grad(const Tensor& grad, const Tensor& like, int64_t numel) {
    same_device(like, grad, "the upstream gradient");
    TORCH_CHECK(grad.scalar_type() == like.scalar_type() && grad.numel() == numel, "the upstream gradient has another type or size");
}

// ---------------------------------------------------------------------------------- library calls
Tensor embedding_fwd(const Tensor& tokens_, const Tensor& weight_, double scale) {
    const c10::OptionalDeviceGuard guard(weight_.device());
    check_tokens(tokens_);
    same_device(weight_, tokens_, "tokens");
    TORCH_CHECK(weight_.dim() == 2, "weight must be [V, D]");
    const Tensor tokens = dense(tokens_);
    const int64_t vocab = weight_.size(0), D = weight_.size(1);
    const Tensor weight = weight_.is_neg() || (D > 1 && weight_.stride(1) != 1) ? dense(weight_) : weight_;
    at::DimVector shape(tokens.sizes());
    shape.push_back(D);
    const Tensor out = at::empty(shape, weight.options());
    check(lib.embedding_forward(address(weight), weight.stride(0), dtype_code(weight), vocab, width(D),
                                address(tokens), static_cast<int>(tokens.element_size()), tokens.numel(),
                                static_cast<float>(scale), writable(out), stream_of(weight)),
          "igs_embedding_forward");
    return out;
}

Tensor embedding_bwd(const Tensor& grad_, const Tensor& tokens_, int64_t vocab, double scale, int64_t padding) {
    const c10::OptionalDeviceGuard guard(grad_.device());
    check_tokens(tokens_);
    same_device(grad_, tokens_, "tokens");
    TORCH_CHECK(grad_.dim() > 0 && grad_.numel() == tokens_.numel() * grad_.size(-1), "one gradient row per token");
    const Tensor grad = dense(grad_), tokens = dense(tokens_);
    const int64_t D = grad.size(-1), n = tokens.numel();
    const int code = dtype_code(grad);
    igs_embedding_plan_t plan;
    check(lib.embedding_plan(vocab, width(D), code, n, &plan), "igs_embedding_plan");
    const Tensor out = at::empty({vocab, D}, grad.options()), ws = workspace(plan.ws_bytes, grad);
    check(lib.embedding_backward(address(grad), code, address(tokens), static_cast<int>(tokens.element_size()), n, vocab,
                                 width(D), static_cast<float>(scale), padding, writable(out), writable(ws),
                                 plan.ws_bytes, stream_of(grad)),
          "igs_embedding_backward");
    return out;
}

struct DropoutArgs {
    int64_t threshold, seed;
    Tensor seed_tensor;
    int64_t offset;
    void check(const Tensor& x) const {
        TORCH_CHECK(threshold >= 0 && threshold <= 65536, "a dropout threshold is in 0..65536; got ", threshold);  // 64 bits here
        same_device(x, seed_tensor, "the seed");
        TORCH_CHECK(!seed_tensor.defined() || (seed_tensor.scalar_type() == at::kLong && seed_tensor.numel() == 1 && !seed_tensor.is_neg()),
                    "a seed tensor holds one int64 element");
    }
};

std::tuple<Tensor, Tensor> norm_fwd(const Tensor& x_, const Tensor& weight_, const Tensor& bias_, double eps,
                                    const DropoutArgs& d, bool want_stats) {
    const c10::OptionalDeviceGuard guard(x_.device());
    TORCH_CHECK(x_.dim() > 0 && x_.size(-1) > 0, "x must have a last axis of one element or more");
    check_weights(x_, weight_, bias_);
    d.check(x_);
    const auto [x, step] = rows_of(x_);
    const Tensor weight = dense(weight_), bias = dense(bias_);
    const int64_t D = x.size(-1), rows = x.numel() / D;
    const Tensor y = at::empty(x.sizes(), x.options());
    const Tensor stats = want_stats ? at::empty({rows, 2}, x.options().dtype(at::kFloat)) : Tensor();
    check(lib.layer_norm_forward(address(x), step, dtype_code(x), address(weight), address(bias),
                                 dtype_code(weight.defined() ? weight : bias.defined() ? bias : x), rows, width(D),
                                 static_cast<float>(eps), static_cast<int>(d.threshold), static_cast<uint64_t>(d.seed),
                                 seed_address(d.seed_tensor), static_cast<uint64_t>(d.offset), writable(y),
                                 static_cast<float*>(writable(stats)), stream_of(x)),
          "igs_layer_norm_forward");
    return {y, stats};
}

std::tuple<Tensor, Tensor, Tensor> norm_bwd(const Tensor& grad_, const Tensor& x_, const Tensor& weight_,
                                            at::ScalarType wtype, const Tensor& stats, const DropoutArgs& d, bool want_x,
                                            bool want_w, bool want_b) {
    const c10::OptionalDeviceGuard guard(x_.device());
    TORCH_CHECK(x_.dim() > 0 && x_.size(-1) > 0, "x must have a last axis of one element or more");
    check_weights(x_, weight_, Tensor());
    check_grad(grad_, x_, x_.numel());
    d.check(x_);
    same_device(x_, stats, "the statistics");
    TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.numel() == 2 * (x_.numel() / x_.size(-1)),
                "the statistics are the forward's");
    const auto [x, step] = rows_of(x_);
    const Tensor grad = dense(grad_), weight = dense(weight_);
    const int64_t D = x.size(-1), rows = x.numel() / D;
    const auto wopts = x.options().dtype(wtype);
    const Tensor gx = want_x ? at::empty(x.sizes(), x.options()) : Tensor();
    const Tensor gw = want_w ? at::empty({D}, wopts) : Tensor(), gb = want_b ? at::empty({D}, wopts) : Tensor();
    const int code = dtype_code(x);
    const int wcode = dtype_code(wtype);
    igs_layer_norm_plan_t plan;
    check(lib.layer_norm_plan(rows, width(D), code, wcode, &plan), "igs_layer_norm_plan");
    const Tensor ws = workspace(plan.ws_bytes, x);
    check(lib.layer_norm_backward(address(grad), address(x), step, code, address(weight), wcode,
                                  static_cast<const float*>(address(stats)), rows, width(D),
                                  static_cast<int>(d.threshold), static_cast<uint64_t>(d.seed), seed_address(d.seed_tensor),
                                  static_cast<uint64_t>(d.offset), writable(gx), writable(gw), writable(gb), writable(ws),
                                  plan.ws_bytes, stream_of(x)),
          "igs_layer_norm_backward");
    return {gx, gw, gb};
}

Tensor dropout_call(const Tensor& x_, const DropoutArgs& d) {
    const c10::OptionalDeviceGuard guard(x_.device());
    d.check(x_);
    const Tensor x = dense(x_), y = at::empty(x.sizes(), x.options());
    check(lib.dropout(address(x), dtype_code(x), x.numel(), static_cast<int>(d.threshold), static_cast<uint64_t>(d.seed),
                      seed_address(d.seed_tensor), static_cast<uint64_t>(d.offset), writable(y), stream_of(x)),
          "igs_dropout");
    return y;
}

// ---------------------------------------------------------------------------------- tracers and dispatch modes
// torch.jit.trace and make_fx record the operators that torch dispatches, and a dispatch mode may replace them.  Of the
// calls here they see the allocation of the result and nothing else: a traced function would return memory that nothing
// wrote.  The registered operators are taken then: by the caller in Python where a differentiable operator returns
// nothing, and in the nodes below for a backward of what was called before.
bool dispatch_mode() { return c10::impl::TorchDispatchModeTLS::any_modes_set(); }
bool recorded() { return torch::jit::tracer::isTracing() || dispatch_mode(); }

// Fake tensors and other subclasses hold no memory, and the operators have no rule for them.
void plain_tensors(std::initializer_list<const Tensor*> tensors) {
    for (const Tensor* t : tensors)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->key_set().has(c10::DispatchKey::Python),
                                    "the feature operators take plain tensors; got a fake tensor or another subclass "
                                    "(under torch.compile and torch.export they are registered operators)");
}

template <class F>
c10::TypedOperatorHandle<F> registered(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}
OptTensor optional(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

Tensor embedding_bwd_recorded(const Tensor& grad, const Tensor& tokens, int64_t vocab, double scale, int64_t padding) {
    return registered<Tensor(const Tensor&, const Tensor&, c10::SymInt, double, c10::SymInt)>("igs_amd::embedding_bwd")
        .call(grad, tokens, vocab, scale, padding);
}
variable_list norm_bwd_recorded(const Tensor& grad, const Tensor& x, const Tensor& weight, at::ScalarType wtype,
                                const Tensor& stats, const DropoutArgs& d, bool want_w, bool want_b) {
    // of the bias the operator takes the type and the length alone
    const Tensor bias = !want_b ? Tensor() : weight.defined() ? weight : at::empty({x.size(-1)}, x.options().dtype(wtype));
    const std::vector<Tensor> g =
        registered<std::vector<Tensor>(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, const Tensor&, c10::SymInt,
                                       c10::SymInt, const OptTensor&, c10::SymInt)>("igs_amd::layer_norm_bwd")
            .call(grad, x, optional(weight), optional(bias), stats, d.threshold, d.seed, optional(d.seed_tensor), d.offset);
    const size_t at_b = weight.defined() ? 2 : 1;
    return {g[0], want_w ? g[1] : Tensor(), want_b ? g[at_b] : Tensor()};
}
Tensor dropout_recorded(const Tensor& x, const DropoutArgs& d) {
    return registered<Tensor(const Tensor&, c10::SymInt, c10::SymInt, const OptTensor&, c10::SymInt)>("igs_amd::dropout")
        .call(x, d.threshold, d.seed, optional(d.seed_tensor), d.offset);
}

// ---------------------------------------------------------------------------------- autograd nodes
// Gradients as the engine gets them.  The nodes differentiate once: where the backward is itself being recorded
// (create_graph), what it returns raises when it is differentiated.
variable_list once(variable_list grads, bool recorded) {
    if (!recorded || !at::GradMode::is_enabled()) return grads;
    for (Tensor& g : grads)
        if (g.defined()) g = g.detach().requires_grad_();
    torch::autograd::DelayedError error("trying to differentiate twice an operator whose backward is not differentiable",
                                        static_cast<int64_t>(grads.size()));
    return error.apply(std::move(grads));
}

struct EmbeddingNode : torch::autograd::Node {
    SavedVariable tokens;
    int64_t vocab = 0, padding = -1;
    double scale = 1.0;

    std::string name() const override { return "IgsEmbeddingBackward"; }
    variable_list apply(variable_list&& grads) override {
        if (!grads[0].defined() || !task_should_compute_output(0)) return {Tensor()};
        const Tensor t = tokens.unpack();
        Tensor g;
        {
            const at::AutoDispatchBelowADInplaceOrView below;
            g = (dispatch_mode() ? embedding_bwd_recorded : embedding_bwd)(grads[0], t, vocab, scale, padding);
        }
        return once({g}, grads[0].requires_grad());
    }
    void release_variables() override { tokens.reset_data(); }
};

struct NormNode : torch::autograd::Node {
    SavedVariable x, weight, stats, seed_tensor;
    at::ScalarType wtype = at::kFloat;
    int64_t threshold = 0, seed = 0, offset = 0;

    std::string name() const override { return "IgsLayerNormBackward"; }
    variable_list apply(variable_list&& grads) override {
        const bool need[3] = {task_should_compute_output(0), task_should_compute_output(1), task_should_compute_output(2)};
        if (!grads[0].defined() || !(need[0] || need[1] || need[2])) return {Tensor(), Tensor(), Tensor()};
        const Tensor xs = x.unpack(), ws = weight.unpack(), st = stats.unpack();
        const DropoutArgs d{threshold, seed, seed_tensor.unpack(), offset};
        variable_list out(3);
        {
            const at::AutoDispatchBelowADInplaceOrView below;
            if (dispatch_mode()) out = norm_bwd_recorded(grads[0], xs, ws, wtype, st, d, need[1], need[2]);
            else std::tie(out[0], out[1], out[2]) = norm_bwd(grads[0], xs, ws, wtype, st, d, need[0], need[1], need[2]);
        }
        return once(std::move(out), grads[0].requires_grad() || xs.requires_grad() || (ws.defined() && ws.requires_grad()));
    }
    void release_variables() override {
        x.reset_data();
        weight.reset_data();
        stats.reset_data();
        seed_tensor.reset_data();
    }
};

struct DropoutNode : torch::autograd::Node {
    SavedVariable seed_tensor;
    int64_t threshold = 0, seed = 0, offset = 0;

    std::string name() const override { return "IgsDropoutBackward"; }
    variable_list apply(variable_list&& grads) override {
        if (!grads[0].defined() || !task_should_compute_output(0)) return {Tensor()};
        const DropoutArgs d{threshold, seed, seed_tensor.unpack(), offset};
        Tensor g;
        {
            const at::AutoDispatchBelowADInplaceOrView below;
            g = (dispatch_mode() ? dropout_recorded : dropout_call)(grads[0], d);
        }
        return once({g}, grads[0].requires_grad());
    }
    void release_variables() override { seed_tensor.reset_data(); }
};

// Forward-mode derivatives would be dropped without a word.
void no_tangent(const Tensor& t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(),
                                "the feature operators have no forward-mode derivative");
}

template <class N, class... Inputs>
std::shared_ptr<N> node_for(const Inputs&... inputs) {
    std::shared_ptr<N> node(new N(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(inputs...));
    return node;
}

// ---------------------------------------------------------------------------------- differentiable operators
// What a caller gets wrong is refused here (a call on a small tensor takes 5 us, and each Python-level check adds to it).
void on_gpu(const Tensor& first) {
    TORCH_CHECK(first.device().is_cuda(), "the feature operators run on the GPU only (HIP kernels); got a tensor on ", first.device(),
                ". The naive_* functions are the plain-torch expressions.");
}
void supported(const Tensor& t, const char* what) {
    TORCH_CHECK_TYPE(dtype_code(t) >= 0, what, " must be float32, float16 or bfloat16; got ", t.scalar_type());
}

// The row of padding_idx, which may count from the end of the table (-1: none).
int64_t padding_row(const Tensor& weight, std::optional<int64_t> padding_idx) {
    if (!padding_idx) return -1;
    const int64_t vocab = weight.size(0), row = *padding_idx;
    TORCH_CHECK_VALUE(row >= -vocab && row < vocab, "padding_idx ", row, " is outside the table of ", vocab, " rows");
    return row < 0 ? row + vocab : row;
}

// These return nothing under a tracer or a dispatch mode: the caller takes the registered operator.
OptTensor embedding(const Tensor& tokens, const Tensor& weight, double scale, std::optional<int64_t> padding_idx) {
    TORCH_CHECK_VALUE(weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0,
                      "weight must be [V, D] with V, D >= 1; got ", weight.sizes());
    TORCH_CHECK_TYPE(tokens.scalar_type() == at::kLong || tokens.scalar_type() == at::kInt, "tokens must be int32 or int64; got ",
                     tokens.scalar_type());
    supported(weight, "weight");
    TORCH_CHECK_VALUE(std::isfinite(scale), "scale must be finite");
    const int64_t padding = padding_row(weight, padding_idx);
    on_gpu(weight);
    no_tangent(weight);
    if (recorded()) return plain_tensors({&tokens, &weight}), OptTensor();
    std::shared_ptr<EmbeddingNode> node;
    if (torch::autograd::compute_requires_grad(weight)) {
        node = node_for<EmbeddingNode>(weight);
        node->tokens = SavedVariable(tokens, false);
        node->vocab = weight.size(0);
        node->padding = padding;
        node->scale = scale;
    }
    Tensor y;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        y = embedding_fwd(tokens, weight, scale);
    }
    if (node) torch::autograd::set_history(y, node);
    return y;
}

OptTensor layer_norm(const Tensor& x, const OptTensor& weight_, const OptTensor& bias_, double eps, int64_t threshold,
                     int64_t seed, const OptTensor& seed_tensor, int64_t offset) {
    TORCH_CHECK_VALUE(x.dim() > 0 && x.size(-1) > 0, "x must have a last axis of one element or more; got ", x.sizes());
    supported(x, "x");
    Tensor weight = value(weight_), bias = value(bias_);
    bool other = false;
    for (const Tensor* t : {&weight, &bias})
        if (t->defined()) {
            const char* name = t == &weight ? "weight" : "bias";
            TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == x.size(-1), name, " must be [", x.size(-1), "]; got ", t->sizes());
            TORCH_CHECK_TYPE(t->is_floating_point(), name, " must be a floating-point tensor; got ", t->scalar_type());
            other |= t->scalar_type() != x.scalar_type();
        }
    TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "eps must be finite and not negative; got ", eps);
    on_gpu(x);
    if (recorded()) {
        for (const Tensor* t : std::initializer_list<const Tensor*>{&x, &weight, &bias}) no_tangent(*t);
        return plain_tensors({&x, &weight, &bias}), OptTensor();
    }
    if (other) {  // weights of another type than x's are taken in fp32
        if (weight.defined()) weight = weight.to(at::kFloat);
        if (bias.defined()) bias = bias.to(at::kFloat);
    }
    for (const Tensor* t : std::initializer_list<const Tensor*>{&x, &weight, &bias}) no_tangent(*t);
    const DropoutArgs d{threshold, seed, value(seed_tensor), offset};
    std::shared_ptr<NormNode> node;
    if (torch::autograd::compute_requires_grad(x, weight, bias)) node = node_for<NormNode>(x, weight, bias);
    Tensor y, stats;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        std::tie(y, stats) = norm_fwd(x, weight, bias, eps, d, node != nullptr);
    }
    if (node) {
        node->x = SavedVariable(x, false);
        node->weight = SavedVariable(weight, false);
        node->stats = SavedVariable(stats, false);
        node->seed_tensor = SavedVariable(d.seed_tensor, false);
        node->wtype = (weight.defined() ? weight : bias.defined() ? bias : x).scalar_type();
        node->threshold = threshold;
        node->seed = seed;
        node->offset = offset;
        torch::autograd::set_history(y, node);
    }
    return y;
}

OptTensor dropout(const Tensor& x, int64_t threshold, int64_t seed, const OptTensor& seed_tensor, int64_t offset) {
    supported(x, "x");
    on_gpu(x);
    no_tangent(x);
    if (recorded()) return plain_tensors({&x}), OptTensor();
    const DropoutArgs d{threshold, seed, value(seed_tensor), offset};
    std::shared_ptr<DropoutNode> node;
    if (torch::autograd::compute_requires_grad(x)) {
        node = node_for<DropoutNode>(x);
        node->seed_tensor = SavedVariable(d.seed_tensor, false);
        node->threshold = threshold;
        node->seed = seed;
        node->offset = offset;
    }
    Tensor y;
    {
        const at::AutoDispatchBelowADInplaceOrView below;
        y = dropout_call(x, d);
    }
    if (node) torch::autograd::set_history(y, node);
    return y;
}
}  // namespace

PYBIND11_MODULE(_igs_torch, m) {
    const auto nogil = py::call_guard<py::gil_scoped_release>();
    m.def("bind", &bind);
    m.def("embedding", &embedding, nogil);
    m.def("layer_norm", &layer_norm, nogil);
    m.def("dropout", &dropout, nogil);
    m.def("padding_row", &padding_row);
    // without autograd, for the registered operators
    m.def("embedding_fwd", &embedding_fwd, nogil);
    m.def("embedding_bwd", &embedding_bwd, nogil);
    m.def(
        "layer_norm_fwd",
        [](const Tensor& x, const OptTensor& w, const OptTensor& b, double eps, int64_t threshold, int64_t seed,
           const OptTensor& seed_tensor, int64_t offset) {
            return norm_fwd(x, value(w), value(b), eps, DropoutArgs{threshold, seed, value(seed_tensor), offset}, true);
        },
        nogil);
    m.def(
        "layer_norm_bwd",
        [](const Tensor& grad, const Tensor& x, const OptTensor& w, const OptTensor& b, const Tensor& stats,
           int64_t threshold, int64_t seed, const OptTensor& seed_tensor, int64_t offset) {
            const Tensor weight = value(w), bias = value(b);
            check_weights(x, weight, bias);
            auto [gx, gw, gb] = norm_bwd(grad, x, weight, (w ? weight : b ? bias : x).scalar_type(), stats,
                                         DropoutArgs{threshold, seed, value(seed_tensor), offset}, true, w.has_value(), b.has_value());
            std::vector<Tensor> out{gx};
            if (w) out.push_back(gw);
            if (b) out.push_back(gb);
            return out;
        },
        nogil);
    m.def(
        "dropout_plain",
        [](const Tensor& x, int64_t threshold, int64_t seed, const OptTensor& seed_tensor, int64_t offset) {
            return dropout_call(x, DropoutArgs{threshold, seed, value(seed_tensor), offset});
        },
        nogil);
    m.def("rows_of", &rows_of);
}
