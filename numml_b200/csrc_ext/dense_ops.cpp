// Compiled per-call path of the dense operators of the graph layers (numml_b200/functional.py): argument
// checks, allocation, the C-ABI call and the autograd node in C++.  The Python module holds the same
// logic for when the extension has not been built; results are identical.
#include "dense_ops.h"

#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>

#include "../../include/numml_b200.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check_rc(int rc, const char* fn) { TORCH_CHECK(rc == NB200_OK, fn, " failed: status ", rc, " (", nb200_status_string(rc), ")"); }

int dense_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return NB200_F32;
        case at::kDouble: return NB200_F64;
        case at::kBFloat16: return NB200_BF16;
        case at::kHalf: return NB200_F16;
        default: TORCH_CHECK(false, "the dense operators support float32, float64, bfloat16 and float16, got ", t.scalar_type());
    }
}

void check_operand(const Tensor& X, const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), "numml_b200 operators run on CUDA tensors only (there is no CPU path); move the operands to a CUDA device");
    TORCH_CHECK(t.device() == X.device(), "all operands must be on the same device, got ", X.device(), " and ", t.device());
    TORCH_CHECK(t.scalar_type() == X.scalar_type(), "operands must share one floating type, got ", X.scalar_type(), " and ",
                t.scalar_type(), " (", name, ")");
}
void check_first(const Tensor& X) {
    TORCH_CHECK(X.is_cuda(), "numml_b200 operators run on CUDA tensors only (there is no CPU path); move the operands to a CUDA device");
    dense_code(X);
}

const void* ptr(const Tensor& t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }
void* mutable_ptr(const Tensor& t) { return const_cast<void*>(ptr(t)); }

struct Matrix {
    Tensor t;
    int64_t ld;
};
// A [rows, cols] matrix over t's memory (a copy only where rows are not evenly strided runs) and its row stride.
// Lazily negated values (the imaginary part of a conjugate) are negated first, here and below.
Matrix rows_of(const Tensor& given, int64_t cols) {
    const Tensor t = given.resolve_neg();
    if (t.dim() == 2 && (cols <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= cols)) return {t, t.size(0) > 1 ? t.stride(0) : cols};
    return {t.contiguous(), cols};
}
Tensor aligned(const Tensor& t) {
    Tensor c = t.resolve_neg().contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
int64_t row_count(const Tensor& X) {
    int64_t n = 1;
    for (int64_t d = 0; d + 1 < X.dim(); ++d) n *= X.size(d);
    return n;
}
Tensor or_empty(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
Tensor contiguous_or_empty(const Tensor& t) { return t.defined() ? t.resolve_neg().contiguous() : t; }
// Tangents of forward-mode differentiation are refused: no operator passes them on, and a result without one reads as zero.
void refuse_tangents(std::initializer_list<std::reference_wrapper<const Tensor>> operands) {
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (const Tensor& t : operands)
        TORCH_CHECK(!t.defined() || !t._fw_grad(/*level=*/0).defined(), "the dense operators have no forward-mode derivative; an operand carries a tangent");
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

// The device's int32 status word, into which kernels with bounded waits report a failure and which
// numml_torch_cpp.check_status reads: the Python module owns one per GPU for good and hands it over at the first call.
py::function* status_source = nullptr;                   // device index -> tensor; never destroyed, like the words

Tensor* known_status_words() {
    static Tensor* words = new Tensor[64];               // never destroyed: the context may be gone by then
    return words;
}

int32_t* status_word(const Tensor& like) {
    static std::mutex mutex;
    const auto device = static_cast<size_t>(like.get_device());
    if (device >= 64 || status_source == nullptr) return nullptr;
    Tensor& w = known_status_words()[device];
    {
        std::lock_guard<std::mutex> lock(mutex);
        if (w.defined()) return w.data_ptr<int32_t>();
    }
    // a capture may not come to own it: left out until the first call outside one
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(at::cuda::getCurrentCUDAStream(like.get_device()), &capturing) != cudaSuccess ||
        capturing != cudaStreamCaptureStatusNone)
        return nullptr;
    Tensor word;
    {
        py::gil_scoped_acquire gil;                      // not under the mutex
        word = (*status_source)(like.get_device()).cast<Tensor>();
    }
    std::lock_guard<std::mutex> lock(mutex);
    if (!w.defined()) w = word;
    return w.data_ptr<int32_t>();
}

// Gradients of gradients are refused instead of being silently left out.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", static_cast<int64_t>(grads.size()));
    for (auto& g : grads)
        if (g.defined()) g = g.detach().requires_grad_(true);
    return (*error)(std::move(grads));
}

// Absent operands of an autograd node are empty options; needs_input_grad counts only those that are there.
OptTensor option(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }
struct Needs {
    AutogradContext* ctx;
    size_t next = 0;
    bool operator()(bool present) { return present && ctx->needs_input_grad(next++); }
};

// A backward pass under capture may not hand a gradient to a leaf that a live eager graph holds on the default stream: the
// engine would make that stream wait for the capture, which invalidates it or ends the process.  Raised here instead.
// (Another stream that waits becomes part of the capture, and the engine joins it again: warming up on a side stream and
// keeping the results is fine.)
void refuse_foreign_accumulation() {
    const auto current = at::cuda::getCurrentCUDAStream();
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(current, &capturing) != cudaSuccess || capturing == cudaStreamCaptureStatusNone) return;
    const auto node = torch::autograd::get_current_node();
    if (!node) return;
    const auto* info = torch::autograd::get_current_graph_task_exec_info();
    for (const auto& edge : node->next_edges()) {
        if (!edge.is_valid() || dynamic_cast<torch::autograd::AccumulateGrad*>(edge.function.get()) == nullptr) continue;
        if (info != nullptr && !info->empty()) {                 // torch.autograd.grad: only the leaves that were asked for
            const auto it = info->find(edge.function.get());
            if (it == info->end() || !it->second.should_execute()) continue;
        }
        const auto stream = edge.function->stream();
        TORCH_CHECK(!stream.has_value() || *stream == current.unwrap() || at::cuda::CUDAStream(*stream).stream() != nullptr,
                    "a backward pass is being captured into a CUDA graph while an eager graph of the same leaf is alive on the default "
                    "stream; drop the eager results first, run them on another stream, or make the leaf inside the capture");
    }
}

// ---- linear ---------------------------------------------------------------------------------------------
std::pair<Tensor, Tensor> linear_forward(const Tensor& X, const Tensor& W, const Tensor& bias, const Tensor& residual, int act, bool keep_z) {
    const int64_t M = row_count(X), K = W.size(0), N = W.size(1);
    const Matrix x = rows_of(X, K), w = rows_of(W, N), r = residual.defined() ? rows_of(residual, N) : Matrix{Tensor(), 0};
    const Tensor b = contiguous_or_empty(bias);
    c10::cuda::CUDAGuard guard(X.device());
    auto shape = X.sizes().vec();
    shape.back() = N;
    Tensor y = at::empty(shape, X.options()), z;
    if (keep_z && act != NB200_ACT_NONE) z = at::empty({M, N}, X.options());
    check_rc(nb200_linear_forward(M, K, N, ptr(x.t), x.ld, ptr(w.t), w.ld, ptr(b), ptr(r.t), r.ld, act, mutable_ptr(z), mutable_ptr(y),
                                  status_word(X), dense_code(X), at::cuda::getCurrentCUDAStream()), "nb200_linear_forward");
    return {y, z};
}

struct LinearNode : torch::autograd::Function<LinearNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& X, const Tensor& W, const OptTensor& bias, const OptTensor& residual, int64_t act) {
        auto [y, z] = linear_forward(X, W, or_empty(bias), or_empty(residual), static_cast<int>(act), true);
        ctx->save_for_backward({X, W, z});
        ctx->saved_data["act"] = act;
        ctx->saved_data["bias"] = bias.has_value();
        ctx->saved_data["residual"] = residual.has_value();
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        refuse_foreign_accumulation();
        const auto saved = ctx->get_saved_variables();
        const Tensor &X = saved[0], &W = saved[1], &z = saved[2], &dY = grads[0];
        const int act = static_cast<int>(ctx->saved_data["act"].toInt());
        Needs needs{ctx};
        const bool want_x = needs(true), want_w = needs(true), want_b = needs(ctx->saved_data["bias"].toBool()),
                   want_r = needs(ctx->saved_data["residual"].toBool());
        Tensor dx, dw, db;
        if (dY.defined() && (want_x || want_w || want_b)) {
            const int64_t M = row_count(X), K = W.size(0), N = W.size(1);
            const Matrix x = rows_of(X, K), w = rows_of(W, N), g = rows_of(dY, N);
            c10::cuda::CUDAGuard guard(X.device());
            if (want_x) dx = at::empty(X.sizes(), X.options());
            if (want_w) dw = at::empty({K, N}, X.options());
            if (want_b) db = at::empty({N}, X.options());
            const size_t bytes = nb200_linear_backward_workspace_bytes(M, K, N, act, dense_code(X));
            Tensor work = at::empty({static_cast<int64_t>(bytes)}, X.options().dtype(at::kByte));
            check_rc(nb200_linear_backward(M, K, N, ptr(g.t), g.ld, ptr(x.t), x.ld, ptr(w.t), w.ld, ptr(z), act, mutable_ptr(dx), mutable_ptr(dw),
                                           mutable_ptr(db), mutable_ptr(work), bytes, status_word(X), dense_code(X),
                                           at::cuda::getCurrentCUDAStream()), "nb200_linear_backward");
        }
        return once({dx, dw, db, want_r ? dY : Tensor(), Tensor()});
    }
};

Tensor linear(const Tensor& X, const Tensor& W, const OptTensor& bias_, const OptTensor& residual_, int64_t act) {
    const Tensor bias = or_empty(bias_), residual = or_empty(residual_);
    check_first(X);
    check_operand(X, W, "weights");
    if (bias.defined()) check_operand(X, bias, "bias");
    if (residual.defined()) check_operand(X, residual, "residual");
    TORCH_CHECK(X.dim() >= 2, "expected node features [..., channels] with at least 2 dimensions, got ", X.dim());
    TORCH_CHECK(W.dim() == 2 && W.size(0) == X.size(-1), "weights must be [", X.size(-1), ", out_channels], got ", W.sizes());
    TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == W.size(1)), "bias must be [", W.size(1), "], got ", bias.sizes());
    if (residual.defined()) {
        bool same = residual.dim() == X.dim() && residual.size(-1) == W.size(1);
        for (int64_t d = 0; same && d + 1 < X.dim(); ++d) same = residual.size(d) == X.size(d);
        TORCH_CHECK(same, "residual must have the output's shape ", X.sizes().slice(0, X.dim() - 1), " + ", W.size(1), ", got ", residual.sizes());
    }
    refuse_tangents({X, W, bias, residual});
    if (at::GradMode::is_enabled() && (wants_grad(X) || wants_grad(W) || wants_grad(bias) || wants_grad(residual)))
        return LinearNode::apply(X, W, option(bias), option(residual), act);
    return linear_forward(X, W, bias, residual, static_cast<int>(act), false).first;
}

// ---- group norm -----------------------------------------------------------------------------------------
int64_t segment_count(const Tensor& X, const Tensor& p) { return p.defined() ? p.numel() - 1 : (X.dim() == 2 ? 1 : X.size(0)); }

std::pair<Tensor, Tensor> norm_forward(const Tensor& X, int64_t groups, const Tensor& weight, const Tensor& bias, double eps, int act,
                                       const Tensor& p_) {
    const Tensor x = aligned(X), w = contiguous_or_empty(weight), b = contiguous_or_empty(bias), p = contiguous_or_empty(p_);
    const int64_t rows = row_count(X), C = X.size(-1), segments = segment_count(X, p);
    const int code = dense_code(X);
    c10::cuda::CUDAGuard guard(X.device());
    Tensor y = at::empty(X.sizes(), X.options());
    Tensor stats = at::empty({2, segments, groups}, X.options().dtype(code == NB200_F64 ? at::kDouble : at::kFloat));
    const size_t bytes = nb200_group_norm_workspace_bytes(rows, C, groups, segments, code);
    Tensor work = at::empty({static_cast<int64_t>(bytes)}, X.options().dtype(at::kByte));
    char* s = static_cast<char*>(mutable_ptr(stats));
    check_rc(nb200_group_norm_forward(rows, C, groups, segments, static_cast<const int64_t*>(ptr(p)), ptr(x), ptr(w), ptr(b), eps, act,
                                      mutable_ptr(y), s, s ? s + stats.nbytes() / 2 : nullptr, mutable_ptr(work), bytes, code,
                                      at::cuda::getCurrentCUDAStream()), "nb200_group_norm_forward");
    return {y, stats};
}

struct NormNode : torch::autograd::Function<NormNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& X, const OptTensor& weight, const OptTensor& bias, const OptTensor& p,
                          int64_t groups, double eps, int64_t act) {
        auto [y, stats] = norm_forward(X, groups, or_empty(weight), or_empty(bias), eps, static_cast<int>(act), or_empty(p));
        ctx->save_for_backward({X, or_empty(weight), or_empty(bias), or_empty(p), stats});
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        refuse_foreign_accumulation();
        const auto saved = ctx->get_saved_variables();
        const Tensor &X = saved[0], &stats = saved[4];
        const int64_t groups = ctx->saved_data["groups"].toInt();
        const int act = static_cast<int>(ctx->saved_data["act"].toInt());
        Tensor dx, dw, db;
        if (grads[0].defined()) {
            const Tensor x = aligned(X), g = aligned(grads[0]), w = contiguous_or_empty(saved[1]), b = contiguous_or_empty(saved[2]),
                         p = contiguous_or_empty(saved[3]);
            const int64_t rows = row_count(X), C = X.size(-1), segments = segment_count(X, p);
            const int code = dense_code(X);
            c10::cuda::CUDAGuard guard(X.device());
            Needs needs{ctx};
            if (needs(true)) dx = at::empty(X.sizes(), X.options());
            if (needs(saved[1].defined())) dw = at::empty({C}, X.options());
            if (needs(saved[2].defined())) db = at::empty({C}, X.options());
            const size_t bytes = nb200_group_norm_workspace_bytes(rows, C, groups, segments, code);
            Tensor work = at::empty({static_cast<int64_t>(bytes)}, X.options().dtype(at::kByte));
            const char* s = static_cast<const char*>(ptr(stats));
            check_rc(nb200_group_norm_backward(rows, C, groups, segments, static_cast<const int64_t*>(ptr(p)), ptr(g), ptr(x), ptr(w), ptr(b),
                                               s, s ? s + stats.nbytes() / 2 : nullptr, act, mutable_ptr(dx), mutable_ptr(dw), mutable_ptr(db),
                                               mutable_ptr(work), bytes, code, at::cuda::getCurrentCUDAStream()),
                     "nb200_group_norm_backward");
        }
        return once({dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

Tensor group_norm(const Tensor& X, int64_t groups, const OptTensor& weight_, const OptTensor& bias_, double eps, int64_t act,
                  const OptTensor& ptr_) {
    const Tensor weight = or_empty(weight_), bias = or_empty(bias_), p = or_empty(ptr_);
    check_first(X);
    if (weight.defined()) check_operand(X, weight, "weight");
    if (bias.defined()) check_operand(X, bias, "bias");
    TORCH_CHECK(X.dim() >= 2 && X.size(-1) >= 1, "expected features [..., channels] with at least 2 dimensions and one channel, got ", X.sizes());
    const int64_t C = X.size(-1);
    TORCH_CHECK(groups >= 1 && C % groups == 0, C, " channels cannot be split into ", groups, " groups");
    TORCH_CHECK(!weight.defined() || (weight.dim() == 1 && weight.size(0) == C), "weight must be [", C, "], got ", weight.sizes());
    TORCH_CHECK(!bias.defined() || (bias.dim() == 1 && bias.size(0) == C), "bias must be [", C, "], got ", bias.sizes());
    TORCH_CHECK(eps >= 0.0, "eps must not be negative, got ", eps);
    if (p.defined()) {
        TORCH_CHECK(p.is_cuda(), "numml_b200 operators run on CUDA tensors only (there is no CPU path); move the operands to a CUDA device");
        TORCH_CHECK(p.device() == X.device(), "all operands must be on the same device, got ", X.device(), " and ", p.device());
        TORCH_CHECK(p.scalar_type() == at::kLong && p.dim() == 1 && p.numel() >= 1,
                    "ptr must be a 1-D int64 tensor of graphs + 1 row numbers, got ", p.scalar_type(), " ", p.sizes());
        TORCH_CHECK(X.dim() == 2, "with ptr the features must be [nodes, channels], got ", X.sizes());
    }
    refuse_tangents({X, weight, bias});
    if (at::GradMode::is_enabled() && (wants_grad(X) || wants_grad(weight) || wants_grad(bias)))
        return NormNode::apply(X, option(weight), option(bias), option(p), groups, eps, act);
    return norm_forward(X, groups, weight, bias, eps, static_cast<int>(act), p).first;
}

// ---- dropout --------------------------------------------------------------------------------------------
Tensor dropout_run(const Tensor& X, double p, uint64_t seed, uint64_t offset, const Tensor& state, const Tensor& residual) {
    const Tensor x = aligned(X), r = residual.defined() ? aligned(residual) : residual;
    c10::cuda::CUDAGuard guard(X.device());
    Tensor y = at::empty(X.sizes(), X.options());
    check_rc(nb200_dropout(x.numel(), ptr(x), ptr(r), mutable_ptr(y), p, seed, offset, static_cast<const int64_t*>(ptr(state)), dense_code(X),
                           at::cuda::getCurrentCUDAStream()), "nb200_dropout");
    return y;
}

struct DropoutNode : torch::autograd::Function<DropoutNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& X, const OptTensor& residual, const OptTensor& state, double p, int64_t seed,
                          int64_t offset) {
        ctx->save_for_backward({or_empty(state)});
        ctx->saved_data["residual"] = residual.has_value();
        ctx->saved_data["p"] = p;
        ctx->saved_data["seed"] = seed;              // the 64 bits, whatever their sign
        ctx->saved_data["offset"] = offset;
        return dropout_run(X, p, static_cast<uint64_t>(seed), static_cast<uint64_t>(offset), or_empty(state), or_empty(residual));
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        refuse_foreign_accumulation();
        const Tensor state = ctx->get_saved_variables()[0];
        Tensor dx;
        Needs needs{ctx};
        const bool want_x = needs(true), want_r = needs(ctx->saved_data["residual"].toBool());
        if (want_x && grads[0].defined())
            dx = dropout_run(grads[0], ctx->saved_data["p"].toDouble(), static_cast<uint64_t>(ctx->saved_data["seed"].toInt()),
                             static_cast<uint64_t>(ctx->saved_data["offset"].toInt()), state, Tensor());
        return once({dx, want_r ? grads[0] : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

Tensor dropout(const Tensor& X, double p, uint64_t seed, uint64_t offset, const OptTensor& state_, const OptTensor& residual_) {
    const Tensor state = or_empty(state_), residual = or_empty(residual_);
    check_first(X);
    if (residual.defined()) {
        check_operand(X, residual, "residual");
        TORCH_CHECK(residual.sizes() == X.sizes(), "residual must have the shape ", X.sizes(), ", got ", residual.sizes());
    }
    TORCH_CHECK(p >= 0.0 && p <= 1.0, "dropout probability must be in [0, 1], got ", p);
    if (state.defined()) {
        TORCH_CHECK(state.is_cuda(), "numml_b200 operators run on CUDA tensors only (there is no CPU path); move the operands to a CUDA device");
        TORCH_CHECK(state.device() == X.device(), "all operands must be on the same device, got ", X.device(), " and ", state.device());
        TORCH_CHECK(state.scalar_type() == at::kLong && state.dim() == 1 && state.numel() == 2 && state.is_contiguous(),
                    "a seed tensor must hold two int64 words [seed, offset], got ", state.scalar_type(), " ", state.sizes());
    }
    refuse_tangents({X, residual});
    if (at::GradMode::is_enabled() && (wants_grad(X) || wants_grad(residual)))
        return DropoutNode::apply(X, option(residual), option(state), p, static_cast<int64_t>(seed), static_cast<int64_t>(offset));
    return dropout_run(X, p, seed, offset, state, residual);
}

}  // namespace

void register_dense_ops(py::module_& m) {
    const auto free_gil = py::call_guard<py::gil_scoped_release>();
    m.def("linear", &linear, free_gil);
    m.def("group_norm", &group_norm, free_gil);
    m.def("dropout", &dropout, free_gil);
    m.def("set_status_source", [](py::function f) { status_source = new py::function(std::move(f)); });
    m.def("known_status_word", [](int64_t device) { return device >= 0 && device < 64 ? known_status_words()[device] : Tensor(); });
}
