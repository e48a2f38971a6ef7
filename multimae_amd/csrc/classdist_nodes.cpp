// Autograd nodes of the class distributions for calls whose tensors need no copy: the same calls of the C ABI as the Python nodes
// make, without the interpreter in the backward pass, which runs on autograd's own thread and finds cold caches there.  On one host,
// log probabilities and gradient of 512 x 1000 fp32: 63 us a step, 112 us with the Python nodes; distillation of 16 x 32000 bf16 68
// and 119 us; log probabilities of 1 x 32000 bf16 10 and 21 us.  (44 us of the steps are autograd's: log_softmax and its gradient.)
// A call that is anything else (another layout, type or device, a wrong argument, a mode that does not see the kernels) is answered
// with None: the Python side copies, or refuses it by name.
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "../../include/mmae.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The package's own error: what a backward pass throws reaches the caller of backward() as this type.
PyObject* error_type = nullptr;
struct Refused : torch::PyTorchError {
    using PyTorchError::PyTorchError;
    PyObject* python_type() override { return error_type; }
};

int dtype_code(const Tensor& t) {
    const auto s = t.scalar_type();
    return s == at::kFloat ? MMAE_DT_F32 : s == at::kBFloat16 ? MMAE_DT_BF16 : s == at::kHalf ? MMAE_DT_F16 : -1;
}

struct Geometry { int outer, classes, inner; };

// Forward-mode derivatives and traces do not see what the kernels write.
bool passed_by(const Tensor& logits) {
    return logits._fw_grad(0).defined() || torch::jit::tracer::isTracing() ||
           c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value();
}

// Logits [B, C, ...] as they are in most calls: contiguous, not empty, on the current device.
bool plain_logits(const Tensor& t, Geometry& g) {
    if (!t.is_cuda() || t.layout() != at::kStrided || dtype_code(t) < 0 || t.dim() < 2 || !t.is_contiguous() || t.numel() == 0) return false;
    if (t.device().index() != c10::hip::current_device()) return false;
    const int64_t outer = t.size(0), classes = t.size(1), inner = t.numel() / (outer * classes);
    if (outer > INT_MAX || classes > INT_MAX || inner > INT_MAX) return false;
    g = {(int)outer, (int)classes, (int)inner};
    return true;
}
// t: contiguous, [B, k, ...] (or [B, ...] for k = 0) beside the logits.
bool beside(const Tensor& t, const Tensor& logits, int64_t k) {
    if (!t.is_cuda() || t.layout() != at::kStrided || t.device() != logits.device() || !t.is_contiguous() || t.dim() != logits.dim() - (k == 0)) return false;
    for (int64_t i = 0; i < t.dim(); ++i) {
        const int64_t want = i == 0 ? logits.size(0) : k && i == 1 ? k : logits.size(k ? i : i + 1);
        if (t.size(i) != want) return false;
    }
    return true;
}

// What a distillation call points to.
bool fits(const Tensor& logits, const Tensor& top_class, const Tensor& top_value, const Tensor& mask, int64_t patch, Geometry& g) {
    if (!plain_logits(logits, g) || top_class.dim() < 2) return false;
    const int64_t k = top_class.size(1);
    const auto kind = top_class.scalar_type();
    if (k < 1 || k > 64 || (kind != at::kLong && kind != at::kInt) || dtype_code(top_value) < 0 || !beside(top_class, logits, k) || !beside(top_value, logits, k)) return false;
    if (!mask.defined()) return true;
    const int64_t width = logits.dim() > 2 ? logits.size(-1) : 1;
    if (patch < 1 || (patch > 1 && logits.dim() != 4) || width % patch || g.inner / width % patch) return false;
    return mask.is_cuda() && mask.device() == logits.device() && mask.scalar_type() == at::kLong && mask.is_contiguous() && mask.dim() == 2 &&
           mask.size(0) == g.outer && mask.size(1) == g.inner / (patch * patch);
}
// The tensors that a backward pass gets back: as they were saved, or what a hook made of them, in any layout.  Whatever else the hook
// changed is refused.
variable_list unpacked(AutogradContext* ctx) {
    at::AutoGradMode off(false);
    auto saved = ctx->get_saved_variables();
    for (auto& t : saved)
        if (t.defined()) t = t.contiguous();
    return saved;
}
bool floats(const Tensor& t, const Tensor& like, int64_t n) { return t.device() == like.device() && t.scalar_type() == at::kFloat && t.numel() == n; }
void require_unpacked(bool as_saved) {
    if (!as_saved) throw Refused("class distributions: a saved tensor came back with another shape, type or device");
}

mmae_stream_t stream_of(const Tensor& t) { return (mmae_stream_t)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
void check(int rc) {
    if (rc != MMAE_OK) throw Refused(mmae_last_error());
}

// What a backward pass hands out: a gradient of it is refused, not taken for zero.
Tensor once(const Tensor& grad) {
    if (!at::GradMode::is_enabled()) return grad;
    auto refuse = std::make_shared<torch::autograd::DelayedError>("class distributions: differentiated once, a gradient of the gradient is not there", 1);
    return (*refuse)({grad.detach().requires_grad_(true)})[0];
}

struct Scores { Tensor log_prob, entropy, top_log_prob, top_class, stats; };

Scores scores(const Tensor& logits, const Geometry& g, const Tensor& target, int64_t k, double temperature, bool want_stats) {
    const auto f32 = logits.options().dtype(at::kFloat);
    Scores s;
    s.log_prob = at::empty(target.sizes(), f32);
    s.entropy = at::empty(target.sizes(), f32);
    const int64_t n = target.numel();
    if (want_stats) s.stats = at::empty({2, n}, f32);
    if (k) {
        auto shape = logits.sizes().vec();
        shape[1] = k;
        s.top_log_prob = at::empty(shape, f32);
        s.top_class = at::empty(shape, f32.dtype(at::kLong));
    }
    const int code = dtype_code(logits);
    const size_t bytes = mmae_class_log_probs_workspace_bytes(code, g.outer, g.classes, g.inner, (int)k);
    const Tensor ws = bytes ? at::empty({(int64_t)bytes}, f32.dtype(at::kByte)) : Tensor();
    float* stats = want_stats ? s.stats.data_ptr<float>() : nullptr;
    check(mmae_class_log_probs(logits.data_ptr(), code, g.outer, g.classes, g.inner, (long)g.classes * g.inner, target.data_ptr<int64_t>(), (int)k,
                               (float)temperature, s.log_prob.data_ptr<float>(), s.entropy.data_ptr<float>(), stats, stats ? stats + n : nullptr,
                               k ? s.top_log_prob.data_ptr<float>() : nullptr, k ? s.top_class.data_ptr<int64_t>() : nullptr,
                               bytes ? ws.data_ptr() : nullptr, bytes, stream_of(logits)));
    return s;
}

struct LogProbs : torch::autograd::Function<LogProbs> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& target, int64_t k, double temperature) {
        Geometry g;
        plain_logits(logits, g);
        const Scores s = scores(logits, g, target, k, temperature, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({logits, target, s.entropy, s.stats});
        ctx->saved_data["temperature"] = temperature;
        if (!k) return {s.log_prob, s.entropy};
        ctx->mark_non_differentiable({s.top_log_prob, s.top_class});
        return {s.log_prob, s.entropy, s.top_log_prob, s.top_class};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const auto saved = unpacked(ctx);
        const Tensor &logits = saved[0], &target = saved[1];
        Geometry g;
        require_unpacked(plain_logits(logits, g) && target.scalar_type() == at::kLong && beside(target, logits, 0) && floats(saved[2], logits, target.numel()) &&
                         floats(saved[3], logits, 2 * target.numel()));
        Tensor d[2], d_logits;
        {
            at::AutoGradMode off(false);
            for (int i = 0; i < 2; ++i)
                if (grads[i].defined()) d[i] = grads[i].contiguous();  // (fp32, as the outputs: autograd sees to it)
            d_logits = at::empty(logits.sizes(), logits.options());
        }
        const float* stats = saved[3].data_ptr<float>();
        check(mmae_class_log_probs_bwd(logits.data_ptr(), dtype_code(logits), g.outer, g.classes, g.inner, (long)g.classes * g.inner,
                                       target.data_ptr<int64_t>(), (float)ctx->saved_data["temperature"].toDouble(), saved[2].data_ptr<float>(), stats,
                                       stats + target.numel(), d[0].defined() ? d[0].data_ptr<float>() : nullptr,
                                       d[1].defined() ? d[1].data_ptr<float>() : nullptr, d_logits.data_ptr(), stream_of(logits)));
        return {once(d_logits), Tensor(), Tensor(), Tensor()};
    }
};

// One call of mmae_distill: what it points to, and how a map's positions meet the mask.
struct Distillation {
    Tensor logits, top_class, top_value, mask, workspace;
    int64_t patch;
    double temperature;
    bool log_probs;
    void run(const float* upstream, bool again, bool skip_unit, float* loss, void* d_logits) const {
        Geometry g;
        plain_logits(logits, g);
        const int64_t width = logits.dim() > 2 ? logits.size(-1) : 1;
        check(mmae_distill(logits.data_ptr(), dtype_code(logits), g.outer, g.classes, g.inner, (long)g.classes * g.inner, top_class.data_ptr(),
                           (int)top_class.element_size(), top_value.data_ptr(), dtype_code(top_value), (int)top_class.size(1), log_probs, (float)temperature,
                           mask.defined() ? mask.data_ptr<int64_t>() : nullptr, (int)width, mask.defined() ? (int)patch : 1, upstream, again, skip_unit,
                           loss, d_logits, workspace.data_ptr(), (size_t)workspace.numel(), stream_of(logits)));
    }
};

// The gradient for an upstream gradient of 1 is made with the loss; the backward pass looks at the real one on the device and makes it
// again only where it differs.  The buffer goes to the caller of the first backward pass, a further one fills a buffer of its own.
struct Distill : torch::autograd::Function<Distill> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& top_class, const Tensor& top_value, const std::optional<Tensor>& given,
                          const Tensor& workspace, int64_t patch, double temperature, bool log_probs) {
        const Tensor mask = given ? *given : Tensor();
        const Tensor loss = at::empty({}, logits.options().dtype(at::kFloat)), d_logits = at::empty(logits.sizes(), logits.options());
        Distillation{logits, top_class, top_value, mask, workspace, patch, temperature, log_probs}.run(nullptr, false, false, loss.data_ptr<float>(), d_logits.data_ptr());
        ctx->save_for_backward({logits, top_class, top_value, mask, workspace});
        auto& d = ctx->saved_data;
        d["patch"] = patch;
        d["temperature"] = temperature;
        d["log_probs"] = log_probs;
        d["d_logits"] = d_logits;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        auto& d = ctx->saved_data;
        const auto first = d.find("d_logits");
        Tensor d_logits;
        if (first != d.end()) {
            d_logits = first->second.toTensor();
            d.erase(first);
        }
        const bool made = d_logits.defined();
        if (!made || !d.count("unit")) {
            const auto saved = unpacked(ctx);  // (refused if an input was changed since, or the graph is freed)
            at::AutoGradMode off(false);
            Geometry g;
            require_unpacked(fits(saved[0], saved[1], saved[2], saved[3], d["patch"].toInt(), g) && saved[4].device() == saved[0].device() &&
                             saved[4].scalar_type() == at::kByte && (!made || (d_logits.sizes() == saved[0].sizes() && d_logits.scalar_type() == saved[0].scalar_type())));
            if (!made) d_logits = at::empty(saved[0].sizes(), saved[0].options());
            const Tensor upstream = grads[0].contiguous();
            Distillation{saved[0], saved[1], saved[2], saved[3], saved[4], d["patch"].toInt(), d["temperature"].toDouble(), d["log_probs"].toBool()}.run(
                upstream.data_ptr<float>(), true, made, nullptr, d_logits.data_ptr());
        }
        variable_list out(8);
        out[0] = once(d_logits);
        return out;
    }
};

// What the library refuses is left to the Python side too, which raises its error.
template <class F>
pybind11::object unless_refused(F call) {
    try {
        return call();
    } catch (const Refused&) {
        return pybind11::none();
    }
}

pybind11::object class_log_probs(const Tensor& logits, const Tensor& target, int64_t k, double temperature) {
    Geometry g;
    if (passed_by(logits) || !plain_logits(logits, g) || target.scalar_type() != at::kLong || !beside(target, logits, 0) || k < 0 || k > 64 || k > g.classes || !(temperature > 0) ||
        temperature > 1e30)
        return pybind11::none();
    const auto give = [](const Tensor& a, const Tensor& b, const Tensor& c, const Tensor& e) {
        const auto none = [](const Tensor& t) { return t.defined() ? pybind11::cast(t) : pybind11::none(); };
        return pybind11::make_tuple(a, b, none(c), none(e));
    };
    return unless_refused([&]() -> pybind11::object {
        if (at::GradMode::is_enabled() && logits.requires_grad()) {
            const variable_list out = LogProbs::apply(logits, target, k, temperature);
            return give(out[0], out[1], k ? out[2] : Tensor(), k ? out[3] : Tensor());
        }
        const Scores s = scores(logits, g, target, k, temperature, false);
        return give(s.log_prob, s.entropy, s.top_log_prob, s.top_class);
    });
}

pybind11::object distill(const Tensor& logits, const Tensor& top_class, const Tensor& top_value, const std::optional<Tensor>& mask_, int64_t patch,
                         double temperature, bool log_probs) {
    Geometry g;
    const Tensor mask = mask_ ? *mask_ : Tensor();
    if (passed_by(logits) || !fits(logits, top_class, top_value, mask, patch, g) || !(temperature > 0) || temperature > 1e30) return pybind11::none();
    const size_t bytes = mmae_distill_workspace_bytes(dtype_code(logits), g.outer, g.classes, g.inner, (int)top_class.size(1));
    const Tensor workspace = at::empty({(int64_t)bytes}, logits.options().dtype(at::kByte).requires_grad(false));
    return unless_refused([&]() -> pybind11::object {
        if (at::GradMode::is_enabled() && logits.requires_grad())
            return pybind11::cast(Distill::apply(logits, top_class, top_value, mask_, workspace, patch, temperature, log_probs));
        const Tensor loss = at::empty({}, logits.options().dtype(at::kFloat).requires_grad(false));
        Distillation{logits, top_class, top_value, mask, workspace, patch, temperature, log_probs}.run(nullptr, false, false, loss.data_ptr<float>(), nullptr);
        return pybind11::cast(loss);
    });
}

// The gradient that arrives at this loss will be exactly 1.
bool mark_unit_upstream(const Tensor& loss) {
    const auto fn = loss.grad_fn();
    auto* node = dynamic_cast<torch::autograd::CppNode<Distill>*>(fn.get());
    if (node) node->ctx_.saved_data["unit"] = true;
    return node != nullptr;
}

}  // namespace

PYBIND11_MODULE(_nodes, m) {
    error_type = pybind11::object(pybind11::module_::import("multimae_amd._lib").attr("MmaeError")).release().ptr();
    m.def("class_log_probs", &class_log_probs);
    m.def("distill", &distill);
    m.def("mark_unit_upstream", &mark_unit_upstream);
}
