// swarm_torch.cpp — the sequence-policy operators of include/swarmseq.h as differentiable torch functions (module
// SwarmACB_isaac._seqops, called by agents/sequence_ops.py, which checks every argument first).
//
// Their kernels take a few microseconds at the trainers' own sizes, where the host decides how long a training pass
// takes. With the backward passes written in Python it took 113 us, of which the operators' own Python was half: the
// autograd engine runs them on a thread of its own, so interpreter state moves between two cores on every pass.
//
// The C ABI is looked up in the library that the package has loaded (bind()), not linked, so that both always use
// one and the same build.
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPStream.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/swarmseq.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Optional = std::optional<Tensor>;

// The functions of the C ABI, in order of declaration.
#define SEQ_FUNCTIONS(X)              \
    X(swarm_gated_scan_workspace)     \
    X(swarm_gated_scan_forward)       \
    X(swarm_gated_scan_backward)      \
    X(swarm_gated_step)               \
    X(swarm_residual_norm_workspace)  \
    X(swarm_residual_norm_forward)    \
    X(swarm_residual_norm_backward)   \
    X(swarm_log_probs_workspace)      \
    X(swarm_log_probs)                \
    X(swarm_policy_loss_forward)      \
    X(swarm_policy_loss_backward)

struct Abi {
#define X(name) decltype(&::name) name = nullptr;
    SEQ_FUNCTIONS(X)
#undef X
    const char* (*strerror)(int32_t) = nullptr;
    int32_t (*last_hip_error)() = nullptr;
    decltype(&hipStreamGetCaptureInfo) capture_info = nullptr;
};
Abi abi;

void bind(const std::string& path) {
    void* lib = dlopen(path.c_str(), RTLD_NOW | RTLD_NOLOAD);
    if (!lib) throw std::runtime_error("_seqops: " + path + " is not loaded");
    auto find = [&](const char* name) {
        void* f = dlsym(lib, name);
        if (!f) throw std::runtime_error(std::string("_seqops: ") + path + " has no " + name);
        return f;
    };
#define X(name) abi.name = reinterpret_cast<decltype(abi.name)>(find(#name));
    SEQ_FUNCTIONS(X)
#undef X
    abi.strerror = reinterpret_cast<decltype(abi.strerror)>(find("swarm_strerror"));
    abi.last_hip_error = reinterpret_cast<decltype(abi.last_hip_error)>(find("swarm_last_hip_error"));
    abi.capture_info = reinterpret_cast<decltype(abi.capture_info)>(find("hipStreamGetCaptureInfo"));
}

void check(int32_t rc, const char* what) {
    if (rc != 0)
        throw std::runtime_error(std::string(what) + " failed: " + abi.strerror(rc) + " (status " + std::to_string(rc) +
                                 ", hip error " + std::to_string(abi.last_hip_error()) + ")");
}

int32_t type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return SWARM_F32;
        case at::kBFloat16: return SWARM_BF16;
        case at::kHalf: return SWARM_F16;
        default: throw std::runtime_error("_seqops: float32, bfloat16 or float16 is needed");
    }
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// The capture that the stream's calls go into: 0 outside of captures.
int64_t capture_of(const Tensor& t) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (abi.capture_info(c10::hip::getCurrentHIPStream(t.device().index()).stream(), &status, &id) != hipSuccess)
        throw std::runtime_error("_seqops: the stream's capture is not valid");
    return status == hipStreamCaptureStatusNone ? 0 : static_cast<int64_t>(id);
}

template <typename T = void>
T* ptr(const Tensor& t) {
    return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr;
}
template <typename T = void>
T* ptr(const Optional& t) {
    return t ? ptr<T>(*t) : nullptr;
}

Tensor floats(const Tensor& like, at::IntArrayRef shape) { return at::empty(shape, like.options().dtype(at::kFloat)); }

// A call's own workspace.
Tensor workspace(const Tensor& like, int64_t words) {
    if (words < 0) throw std::runtime_error("_seqops: no workspace for these sizes");
    return words > 0 ? floats(like, {words}) : Tensor();
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const Optional& t) { return t && wants_grad(*t); }

bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool has_tangent(const Optional& t) { return t && has_tangent(*t); }

// Kernels write new tensors through their pointers, of which neither forward-mode differentiation nor a trace knows: the
// one would lose the derivative, the other would record an empty tensor.
template <typename... Ts>
void check_recorders(const char* what, const Ts&... operands) {
    if (torch::jit::tracer::isTracing())
        throw std::runtime_error(std::string(what) + " cannot be recorded by torch.jit.trace on the GPU");
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && (has_tangent(operands) || ...))
        throw std::invalid_argument(std::string(what) + " has no forward-mode derivative on the GPU: detach the dual tensor");
}

// t with its last dimension contiguous
Tensor rows(const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); }

// Gradients are new tensors that nothing recorded: where a graph of them is asked for, differentiating it is an error.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    for (auto& g : grads)
        if (g.defined()) g = g.detach().set_requires_grad(true);
    const auto error = std::make_shared<torch::autograd::DelayedError>(
        "the sequence-policy operators cannot be differentiated twice", static_cast<int>(grads.size()));
    return (*error)(std::move(grads));
}

// ---------------------------------------------------------------------------------- gated recurrence

struct Scan {
    Tensor h, last, tiles;
};

Scan scan_forward(const Tensor& gates, const Optional& state, const Optional& keep, const Optional& lengths, bool save) {
    const at::DeviceGuard guard(gates.device());
    const int64_t n = gates.size(0), T = gates.size(1), U = gates.size(2) / 3;
    Scan r{at::empty({n, T, U}, gates.options()), floats(gates, {n, U}),
           save ? floats(gates, {n, SWARM_GATED_TILES(T), U}) : Tensor()};
    const Tensor work = workspace(gates, abi.swarm_gated_scan_workspace(n, T, U));
    check(abi.swarm_gated_scan_forward(type_of(gates), n, T, U, ptr(gates), gates.stride(0), gates.stride(1),
                                       ptr<float>(state), ptr<float>(keep), ptr<int64_t>(lengths), ptr(r.h),
                                       ptr<float>(r.last), ptr<float>(r.tiles), ptr<float>(work), stream_of(gates)),
          "swarm_gated_scan_forward");
    return r;
}

// The backward pass forms the states again from one saved state per tile of steps, so nothing of the size of the
// sequence is kept but the inputs.
struct GatedScan : torch::autograd::Function<GatedScan> {
    static variable_list forward(AutogradContext* ctx, const Tensor& gates, const Optional& state, const Optional& keep,
                                 const Optional& lengths) {
        Scan r = scan_forward(gates, state, keep, lengths, true);
        ctx->save_for_backward({gates, keep.value_or(Tensor()), lengths.value_or(Tensor()), r.tiles});
        ctx->saved_data["state"] = wants_grad(state);
        ctx->set_materialize_grads(false);
        return {r.h, r.last};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &gates = saved[0], &keep = saved[1], &lengths = saved[2], &tiles = saved[3];
        const at::DeviceGuard guard(gates.device());
        const int64_t n = gates.size(0), T = gates.size(1), U = gates.size(2) / 3;
        const Tensor d_h = grads[0].defined() ? rows(grads[0]) : Tensor();
        const Tensor d_last = grads[1].defined() ? grads[1].contiguous() : Tensor();
        const Tensor d_gates = at::empty({n, T, 3 * U}, gates.options());
        const Tensor d_state = ctx->saved_data["state"].toBool() ? floats(gates, {n, U}) : Tensor();
        const Tensor work = workspace(gates, abi.swarm_gated_scan_workspace(n, T, U));
        check(abi.swarm_gated_scan_backward(type_of(gates), n, T, U, ptr(gates), gates.stride(0), gates.stride(1),
                                            ptr<float>(keep), ptr<int64_t>(lengths), ptr<float>(tiles), ptr(d_h),
                                            d_h.defined() ? d_h.stride(0) : 0, d_h.defined() ? d_h.stride(1) : 0,
                                            ptr<float>(d_last), ptr(d_gates), ptr<float>(d_state), ptr<float>(work),
                                            stream_of(gates)),
              "swarm_gated_scan_backward");
        return once({d_gates, d_state, Tensor(), Tensor()});
    }
};

std::tuple<Tensor, Tensor> gated_scan(const Tensor& gates, const Optional& state, const Optional& keep,
                                      const Optional& lengths) {
    check_recorders("gated_recurrence", gates, state, keep);
    if (at::GradMode::is_enabled() && (wants_grad(gates) || wants_grad(state))) {
        const auto r = GatedScan::apply(gates, state, keep, lengths);
        return {r[0], r[1]};
    }
    const Scan r = scan_forward(gates, state, keep, lengths, false);
    return {r.h, r.last};
}

std::tuple<Tensor, Tensor> gated_step(const Tensor& gates, const Tensor& state, const Optional& keep, bool inplace) {
    check_recorders("gated_recurrence_step", gates, state, keep);
    const at::DeviceGuard guard(gates.device());
    const int64_t rows = gates.size(0), U = gates.size(1) / 3;
    const Tensor h = at::empty({rows, U}, gates.options()), out = inplace ? state : at::empty_like(state);
    check(abi.swarm_gated_step(type_of(gates), rows, U, ptr(gates), gates.stride(0), ptr<float>(state), ptr<float>(keep),
                               ptr(h), ptr<float>(out), stream_of(gates)),
          "swarm_gated_step");
    // A backward pass that saved this state has to notice the write. Tensors of inference mode cannot be saved and have
    // no version.
    if (inplace && !state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
    return {h, out};
}

// --------------------------------------------------------------------------------- residual RMS norm

struct Norm {
    Tensor y, stream, rstd;
};

Norm norm_forward(const Tensor& x, const Optional& residual, const Optional& weight, double eps, bool save) {
    const at::DeviceGuard guard(x.device());
    const int64_t n = x.size(0), D = x.size(1);
    Norm r{at::empty({n, D}, x.options()), residual ? at::empty({n, D}, x.options()) : Tensor(),
           save ? floats(x, {n}) : Tensor()};
    check(abi.swarm_residual_norm_forward(type_of(x), n, D, ptr(x), x.stride(0), ptr(residual),
                                          residual ? residual->stride(0) : 0, ptr(weight), static_cast<float>(eps),
                                          ptr(r.y), ptr(r.stream), ptr<float>(r.rstd), stream_of(x)),
          "swarm_residual_norm_forward");
    return r;
}

// Saved are both addends: the stream that they gave is rounded to its type, and its gradients' sums would show it.
struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Optional& residual, const Optional& weight,
                                 double eps) {
        Norm r = norm_forward(x, residual, weight, eps, true);
        ctx->save_for_backward({x, residual.value_or(Tensor()), weight.value_or(Tensor()), r.rstd});
        ctx->saved_data["weight"] = wants_grad(weight);
        ctx->set_materialize_grads(false);
        return residual ? variable_list{r.y, r.stream} : variable_list{r.y};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &residual = saved[1], &weight = saved[2], &rstd = saved[3];
        const bool two = residual.defined(), with_w = ctx->saved_data["weight"].toBool();
        const at::DeviceGuard guard(x.device());
        const Tensor d_out = two && grads[1].defined() ? rows(grads[1]) : Tensor();
        if (!grads[0].defined())      // only the stream was used: the sum passes its gradient on
            return once({d_out, two ? d_out : Tensor(), with_w ? at::zeros_like(weight) : Tensor(), Tensor()});
        const int64_t n = x.size(0), D = x.size(1);
        const Tensor d_y = rows(grads[0]), d_x = at::empty({n, D}, x.options());
        Tensor d_w, work;
        if (with_w) {
            d_w = at::empty({D}, x.options());
            work = workspace(x, abi.swarm_residual_norm_workspace(n, D));
        }
        check(abi.swarm_residual_norm_backward(type_of(x), n, D, ptr(x), x.stride(0), ptr(residual),
                                               two ? residual.stride(0) : 0, ptr(weight), ptr<float>(rstd), ptr(d_y), d_y.stride(0),
                                               ptr(d_out), d_out.defined() ? d_out.stride(0) : 0, ptr(d_x), ptr(d_w),
                                               ptr<float>(work), stream_of(x)),
              "swarm_residual_norm_backward");
        return once({d_x, two ? d_x : Tensor(), d_w, Tensor()});
    }
};

std::tuple<Tensor, Optional> residual_norm(const Tensor& x, const Optional& residual, const Optional& weight, double eps) {
    check_recorders("residual_rms_norm", x, residual, weight);
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(residual) || wants_grad(weight))) {
        const auto r = ResidualNorm::apply(x, residual, weight, eps);
        return {r[0], residual ? Optional(r[1]) : std::nullopt};
    }
    const Norm r = norm_forward(x, residual, weight, eps, false);
    return {r.y, residual ? Optional(r.stream) : std::nullopt};
}

// --------------------------------------------------------------------------------------- policy loss

struct LossArgs {
    Tensor actions, old_lp, adv;
    Optional ref, mask, denom;
    double lo, hi, kl_coef, entropy_coef;
    Tensor flag;
};

struct Loss {
    Tensor loss, terms, used, work, unit;
};

float* row_stats(const Tensor& work) { return ptr<float>(work) + SWARM_POLICY_LOSS_PARTIALS; }

Loss loss_forward(const Tensor& logits, const LossArgs& a, bool save) {
    const at::DeviceGuard guard(logits.device());
    const int64_t M = logits.size(0), K = logits.size(1);
    // losses in float16 are scaled, so the gradient for an incoming gradient of 1 would not be the one asked for
    const bool unit = save && logits.scalar_type() != at::kHalf;
    Loss r{floats(logits, {}), floats(logits, {4}), floats(logits, {}), floats(logits, {SWARM_POLICY_LOSS_PARTIALS + 4 * M}),
           unit ? at::empty({M, K}, logits.options()) : Tensor()};
    check(abi.swarm_policy_loss_forward(
              type_of(logits), M, K, ptr(logits), logits.stride(0), ptr<int64_t>(a.actions), ptr<float>(a.old_lp),
              ptr<float>(a.ref), ptr<float>(a.adv), ptr<uint8_t>(a.mask), ptr<float>(a.denom), static_cast<float>(a.lo),
              static_cast<float>(a.hi), static_cast<float>(a.kl_coef), static_cast<float>(a.entropy_coef),
              ptr<float>(r.loss), ptr<float>(r.terms), ptr<float>(r.used), row_stats(r.work), ptr(r.unit),
              ptr<float>(r.work), ptr<int32_t>(a.flag), stream_of(logits)),
          "swarm_policy_loss_forward");
    return r;
}

// The forward call, which has the logits at hand, forms the gradient for an incoming gradient of 1 as well; the first
// backward call hands it out, written anew if the incoming gradient is another one, and later calls form their own.
// So does a backward call captured without its forward call: replays write the buffer again and again.
struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const LossArgs& a) {
        Loss r = loss_forward(logits, a, true);
        ctx->save_for_backward({logits, a.actions, r.work, r.used});
        ctx->saved_data["entropy_coef"] = a.entropy_coef;
        if (r.unit.defined()) {
            ctx->saved_data["unit"] = r.unit;
            ctx->saved_data["capture"] = capture_of(logits);
        }
        ctx->mark_non_differentiable({r.terms});
        return {r.loss, r.terms};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &actions = saved[1], &work = saved[2], &used = saved[3];
        const at::DeviceGuard guard(logits.device());
        const int64_t M = logits.size(0), K = logits.size(1);
        Tensor d;
        const auto unit = ctx->saved_data.find("unit");
        const bool have = unit != ctx->saved_data.end() && ctx->saved_data["capture"].toInt() == capture_of(logits);
        if (have) d = unit->second.toTensor();
        else d = at::empty({M, K}, logits.options());
        if (unit != ctx->saved_data.end()) ctx->saved_data.erase(unit);
        const Tensor g = grads[0].contiguous();
        check(abi.swarm_policy_loss_backward(type_of(logits), M, K, ptr(logits), logits.stride(0), ptr<int64_t>(actions),
                                             static_cast<float>(ctx->saved_data["entropy_coef"].toDouble()),
                                             row_stats(work), ptr<float>(used), ptr<float>(g), have, ptr(d),
                                             stream_of(logits)),
              "swarm_policy_loss_backward");
        return once({d, Tensor()});
    }
};

std::tuple<Tensor, Tensor> policy_loss(const Tensor& logits, const Tensor& actions, const Tensor& old_lp, const Tensor& adv,
                                       const Optional& ref, const Optional& mask, const Optional& denom, double lo,
                                       double hi, double kl_coef, double entropy_coef, const Tensor& flag) {
    check_recorders("categorical_policy_loss", logits, old_lp, adv, ref, denom);
    const LossArgs a{actions, old_lp, adv, ref, mask, denom, lo, hi, kl_coef, entropy_coef, flag};
    if (at::GradMode::is_enabled() && wants_grad(logits)) {
        const auto r = PolicyLoss::apply(logits, a);
        return {r[0], r[1]};
    }
    const Loss r = loss_forward(logits, a, false);
    return {r.loss, r.terms};
}

std::tuple<Tensor, Tensor> log_probs(const Tensor& logits, const Tensor& actions, const Tensor& flag) {
    check_recorders("categorical_log_probs", logits);
    const at::DeviceGuard guard(logits.device());
    const int64_t M = logits.size(0), K = logits.size(1);
    const Tensor lp = floats(logits, {M}), ent = floats(logits, {M});
    const Tensor work = workspace(logits, abi.swarm_log_probs_workspace(M, K));
    check(abi.swarm_log_probs(type_of(logits), M, K, ptr(logits), logits.stride(0), ptr<int64_t>(actions), ptr<float>(lp),
                              ptr<float>(ent), ptr<float>(work), ptr<int32_t>(flag), stream_of(logits)),
          "swarm_log_probs");
    return {lp, ent};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.attr("GATED_TILE") = SWARM_GATED_TILE;
    m.attr("POLICY_LOSS_PARTIALS") = SWARM_POLICY_LOSS_PARTIALS;
    m.def("bind", &bind);
    m.def("gated_scan", &gated_scan);
    m.def("gated_step", &gated_step);
    m.def("residual_norm", &residual_norm);
    m.def("policy_loss", &policy_loss);
    m.def("log_probs", &log_probs);
}
