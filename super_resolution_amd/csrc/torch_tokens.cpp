// The operators on rows of channels for PyTorch: argument checks, memory from PyTorch's allocator, the current stream and
// the autograd nodes, over the C ABI of libsr355.so (include/sr355.h).  In C++ because a backward pass in Python runs on the
// autograd engine's own thread, where it took longer than the kernels: 117 us a training call of layer norm on a slow host
// against the kernels' 19.
//
// The library's entry points are handed in by address (connect), so this module uses the library that the package loaded.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <array>
#include <climits>
#include <map>
#include <optional>
#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/sr355.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
    decltype(&sr355_last_error) last_error = nullptr;
    decltype(&sr355_layer_norm_fwd) layer_norm_fwd = nullptr;
    decltype(&sr355_layer_norm_bwd_workspace_bytes) layer_norm_bwd_workspace_bytes = nullptr;
    decltype(&sr355_layer_norm_bwd) layer_norm_bwd = nullptr;
    decltype(&sr355_dropout) dropout = nullptr;
    decltype(&sr355_gated_ffn_saved_bytes) gated_ffn_saved_bytes = nullptr;
    decltype(&sr355_gated_ffn_workspace_bytes) gated_ffn_workspace_bytes = nullptr;
    decltype(&sr355_gated_ffn_fwd) gated_ffn_fwd = nullptr;
    decltype(&sr355_gated_ffn_bwd) gated_ffn_bwd = nullptr;
} api;

void connect(const std::map<std::string, size_t> &address) {
    auto set = [&](auto &slot, const char *name) {
        slot = reinterpret_cast<std::decay_t<decltype(slot)>>(address.at(name));
    };
    set(api.last_error, "sr355_last_error");
    set(api.layer_norm_fwd, "sr355_layer_norm_fwd");
    set(api.layer_norm_bwd_workspace_bytes, "sr355_layer_norm_bwd_workspace_bytes");
    set(api.layer_norm_bwd, "sr355_layer_norm_bwd");
    set(api.dropout, "sr355_dropout");
    set(api.gated_ffn_saved_bytes, "sr355_gated_ffn_saved_bytes");
    set(api.gated_ffn_workspace_bytes, "sr355_gated_ffn_workspace_bytes");
    set(api.gated_ffn_fwd, "sr355_gated_ffn_fwd");
    set(api.gated_ffn_bwd, "sr355_gated_ffn_bwd");
}

void ok(int rc, const char *what) { TORCH_CHECK(rc == SR355_OK, what, " failed (", rc, "): ", api.last_error()); }

int code_of(at::ScalarType t) {
    return t == at::kBFloat16 ? SR355_DTYPE_BF16 : t == at::kHalf ? SR355_DTYPE_F16 : t == at::kFloat ? SR355_DTYPE_F32 : -1;
}

// (the kernels compute no tangents, so a dual tensor's derivative would be lost without a word)
void check_dual(const char *who, const Tensor &t) {
    TORCH_CHECK(!t._fw_grad(0).defined(), who, ": forward-mode derivatives are not supported (an input of shape ", t.sizes(), " carries a tangent)");
}

// x is a tensor of rows in one of the types
void check_rows(const char *who, const Tensor &x) {
    check_dual(who, x);
    TORCH_CHECK(x.is_cuda(), who, ": runs on ROCm devices only (got a tensor on ", x.device(), "); there is no CPU fallback");
    TORCH_CHECK(code_of(x.scalar_type()) >= 0, who, ": expected bfloat16, float16 or float32, got ", x.scalar_type());
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, who, ": expected rows of at least one channel, got shape ", x.sizes());
}
void check_device(const char *who, const Tensor &x, const Tensor &t) {
    check_dual(who, t);
    TORCH_CHECK(t.device() == x.device(), who, ": tensors on ", x.device(), " and ", t.device());
}

// x as rows with contiguous channels, and their stride in elements; a copy where x is not laid out so
struct Rows {
    Tensor t;
    int64_t ld;
    explicit Rows(const Tensor &x) {
        const int64_t c = x.size(-1);
        if (x.is_contiguous()) {
            t = x, ld = c;
            return;
        }
        t = x.reshape({-1, c});
        if ((t.size(0) > 1 && t.stride(0) < c) || (c > 1 && t.stride(1) != 1)) t = t.contiguous();
        ld = t.size(0) > 1 ? t.stride(0) : c;
    }
    const void *data() const { return t.const_data_ptr(); }
};

Tensor vector_of(const char *who, const char *name, const Tensor &x, const OptTensor &v, int64_t n, bool fp32_too) {
    if (!v.has_value() || !v->defined()) return Tensor();
    check_device(who, x, *v);
    TORCH_CHECK(v->dim() == 1 && v->size(0) == n && (v->scalar_type() == x.scalar_type() || (fp32_too && v->scalar_type() == at::kFloat)),
                who, ": ", name, " must have shape (", n, ",) and type ", x.scalar_type(), fp32_too ? " or Float" : "", ", got ",
                v->sizes(), " of ", v->scalar_type());
    return v->contiguous();
}

const void *ptr(const Tensor &t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void *out_ptr(const Tensor &t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

struct Launch {                       // the tensors' device is current and its stream taken
    c10::OptionalDeviceGuard guard;
    void *stream;
    explicit Launch(const Tensor &x) : guard(x.device()) {
        stream = static_cast<void *>(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.get_device()).stream());
    }
};

Tensor scratch(const Tensor &x, size_t bytes) { return at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte)); }

// A leaf's gradients are added up on the stream that was current when the oldest live graph of the leaf was recorded.  In a
// capture that must not be the default stream: the engine would make it wait for the captured one, which ends the process.  The
// leaves of a call are those among its inputs and those that the others were made from.
void check_capture(const std::vector<Tensor> &inputs) {
    std::vector<torch::autograd::Node *> ahead;
    std::vector<std::shared_ptr<torch::autograd::Node>> held;
    for (const Tensor &t : inputs) {
        if (!t.defined() || !t.is_cuda() || !t.requires_grad()) continue;
        const c10::OptionalDeviceGuard guard(t.device());
        if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
        held.push_back(t.is_leaf() ? torch::autograd::impl::try_get_grad_accumulator(t) : t.grad_fn());
        if (held.back()) ahead.push_back(held.back().get());
    }
    std::unordered_set<const torch::autograd::Node *> seen;
    while (!ahead.empty()) {
        const auto *node = ahead.back();
        ahead.pop_back();
        if (!seen.insert(node).second) continue;
        if (const auto *leaf = dynamic_cast<const torch::autograd::AccumulateGrad *>(node)) {
            const auto stream = const_cast<torch::autograd::AccumulateGrad *>(leaf)->stream();
            TORCH_CHECK(!stream || stream->id() != 0, "a graph is being captured, and a leaf of shape ", leaf->variable.sizes(),
                        " still belongs to one that was recorded on the default stream: drop that graph's outputs first");
        }
        for (const auto &edge : node->next_edges())
            if (edge.is_valid()) ahead.push_back(edge.function.get());
    }
}
// Whether somebody has to see the call as an operator and not as the work it does: a tensor subclass (a fake one has no memory) or
// a dispatch mode.  The public functions then return nothing, and their caller takes the registered op.  Functional transforms are
// refused: through a registered op a tangent would be lost.
template <typename... Ts>
bool interposed(const char *who, const Ts &...ts) {
    TORCH_CHECK(!c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode), who,
                ": functional transforms (torch.func, vmap) are not supported");
    constexpr c10::DispatchKeySet keys({c10::DispatchKey::Python, c10::DispatchKey::Functionalize});
    return c10::impl::TorchDispatchModeTLS::any_modes_set() || ((ts.defined() && ts.key_set().has_any(keys)) || ...);
}
// whether autograd records a call with these inputs
template <typename... Ts>
bool recorded(const Ts &...ts) {
    if (!at::GradMode::is_enabled() || !((ts.defined() && ts.requires_grad()) || ...)) return false;
    check_capture({ts...});
    return true;
}
Tensor defined(const OptTensor &t) { return t.has_value() ? *t : Tensor(); }

// Gradients of a backward pass that is itself being recorded: they raise when somebody differentiates them.
variable_list once(variable_list grads, const char *who) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list in;
    for (auto &g : grads)
        if (g.defined()) in.push_back(g.detach().requires_grad_(true));
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(who) + " is once differentiable", in.size());
    variable_list out = (*error)(std::move(in));
    size_t k = 0;
    for (auto &g : grads)
        if (g.defined()) g = out[k++];
    return grads;
}

// ---- layer norm ----------------------------------------------------------------------------------------------------
void check_channels(const char *who, const Tensor &x) {
    TORCH_CHECK(x.size(-1) <= INT_MAX - 255, who, ": ", x.size(-1), " channels; up to 2^31 - 256 are supported");
}
struct NormParams {
    Tensor w, b;
    at::ScalarType type;
    NormParams(const char *who, const Tensor &x, const OptTensor &weight, const OptTensor &bias) {
        w = vector_of(who, "weight", x, weight, x.size(-1), true);
        b = vector_of(who, "bias", x, bias, x.size(-1), true);
        TORCH_CHECK(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(), who, ": weight and bias are of types ",
                    w.scalar_type(), " and ", b.scalar_type());
        type = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat;
    }
};

std::tuple<Tensor, Tensor> layer_norm_fwd(const Tensor &x, const OptTensor &weight, const OptTensor &bias, double eps, bool want_stats) {
    check_rows("layer_norm", x);
    check_channels("layer_norm", x);
    const NormParams p("layer_norm", x, weight, bias);
    TORCH_CHECK(eps >= 0.0, "layer_norm: eps must not be negative, got ", eps);
    const Rows r(x);
    const int64_t c = x.size(-1), rows = x.numel() / c;
    Launch launch(x);
    Tensor y = at::empty(x.sizes(), x.options());
    Tensor stats = at::empty(want_stats ? std::vector<int64_t>{2, rows} : std::vector<int64_t>{0}, x.options().dtype(at::kFloat));
    float *s = want_stats && rows ? stats.mutable_data_ptr<float>() : nullptr;
    ok(api.layer_norm_fwd(r.data(), rows, static_cast<int>(c), r.ld, code_of(x.scalar_type()), ptr(p.w), ptr(p.b), code_of(p.type),
                          static_cast<float>(eps), y.mutable_data_ptr(), s, s ? s + rows : nullptr, launch.stream),
       "sr355_layer_norm_fwd");
    return {y, stats};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_bwd(const Tensor &dy, const Tensor &x, const OptTensor &weight, const Tensor &stats,
                                                  at::ScalarType param_type, const std::vector<bool> &need) {
    const char *who = "layer_norm backward";
    check_rows(who, x);
    check_channels(who, x);
    check_device(who, x, dy);
    check_device(who, x, stats);
    const int64_t c = x.size(-1), rows = x.numel() / c;
    TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && stats.dim() == 2 && stats.size(0) == 2 &&
                    stats.size(1) == rows && stats.scalar_type() == at::kFloat && stats.is_contiguous() && need.size() == 3 &&
                    (param_type == x.scalar_type() || param_type == at::kFloat),
                who, ": the gradient must have x's shape and type, the statistics be fp32 [2, rows]");
    const Tensor w = vector_of(who, "weight", x, weight, c, true);
    TORCH_CHECK(!w.defined() || w.scalar_type() == param_type, who, ": a weight of type ", w.scalar_type(), " for gradients of ", param_type);
    const Rows r(x), g(dy);
    Launch launch(x);
    Tensor dx = need[0] ? at::empty(x.sizes(), x.options()) : Tensor();
    Tensor dw, db, ws;
    size_t bytes = 0;
    if (need[1] || need[2]) {
        if (need[1]) dw = at::empty({c}, x.options().dtype(param_type));
        if (need[2]) db = at::empty({c}, x.options().dtype(param_type));
        bytes = api.layer_norm_bwd_workspace_bytes(static_cast<int>(c));
        ws = scratch(x, bytes);
    }
    const float *s = rows ? stats.const_data_ptr<float>() : nullptr;
    ok(api.layer_norm_bwd(g.data(), g.ld, r.data(), r.ld, rows, static_cast<int>(c), code_of(x.scalar_type()), ptr(w), code_of(param_type), s,
                          s ? s + rows : nullptr, out_ptr(dx), out_ptr(dw), out_ptr(db), out_ptr(ws), bytes, launch.stream),
       "sr355_layer_norm_bwd");
    return {dx, dw, db};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const OptTensor &weight, const OptTensor &bias, double eps) {
        auto [y, stats] = layer_norm_fwd(x, weight, bias, eps, true);
        const Tensor w = defined(weight), b = defined(bias);
        ctx->save_for_backward({x, w, stats});
        ctx->saved_data["w"] = w.defined();
        ctx->saved_data["b"] = b.defined();
        ctx->saved_data["type"] = static_cast<int64_t>(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat);
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list dy) {
        const auto saved = ctx->get_saved_variables();
        const bool has_w = ctx->saved_data["w"].toBool(), has_b = ctx->saved_data["b"].toBool();
        // (the edges count the tensors that were given)
        const std::vector<bool> need = {ctx->needs_input_grad(0), has_w && ctx->needs_input_grad(1),
                                        has_b && ctx->needs_input_grad(has_w ? 2 : 1)};
        auto [dx, dw, db] = layer_norm_bwd(dy[0], saved[0], has_w ? OptTensor(saved[1]) : OptTensor(), saved[2],
                                           static_cast<at::ScalarType>(ctx->saved_data["type"].toInt()), need);
        return once({dx, dw, db, Tensor()}, "layer_norm");
    }
};

Tensor layer_norm(const Tensor &x, const OptTensor &weight, const OptTensor &bias, double eps) {
    const Tensor w = defined(weight), b = defined(bias);
    if (interposed("layer_norm", x, w, b)) return Tensor();
    if (recorded(x, w, b)) return LayerNorm::apply(x, weight, bias, eps);
    return std::get<0>(layer_norm_fwd(x, weight, bias, eps, false));
}

// ---- dropout -------------------------------------------------------------------------------------------------------
Tensor dropout_fwd(const Tensor &x, const OptTensor &skip, double p, const Tensor &rng, int64_t site) {
    check_rows("dropout", x);
    check_device("dropout", x, rng);
    TORCH_CHECK(p >= 0.0 && p <= 1.0, "dropout: the probability must lie in [0, 1], got ", p);
    TORCH_CHECK(rng.scalar_type() == at::kLong && rng.dim() == 1 && rng.size(0) == 2 && rng.is_contiguous(),
                "dropout: the generator's state is a contiguous int64 tensor of two words (seed, step)");
    TORCH_CHECK(site >= 0 && site < (int64_t(1) << 32), "dropout: the site must lie in [0, 2^32), got ", site);
    Tensor s = defined(skip);
    if (s.defined()) {
        check_device("dropout", x, s);
        TORCH_CHECK(s.sizes() == x.sizes() && s.scalar_type() == x.scalar_type(), "dropout: the skip must have x's shape and type, got ",
                    s.sizes(), " of ", s.scalar_type());
        s = s.contiguous();
    }
    const Tensor r = x.contiguous();
    Launch launch(x);
    Tensor y = at::empty(x.sizes(), x.options());
    if (x.numel() == 0) return y;
    ok(api.dropout(r.const_data_ptr(), ptr(s), x.numel(), code_of(x.scalar_type()), p, reinterpret_cast<const long long *>(rng.const_data_ptr()),
                   static_cast<unsigned>(site), y.mutable_data_ptr(), launch.stream),
       "sr355_dropout");
    return y;
}

struct Dropout : torch::autograd::Function<Dropout> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, double p, const Tensor &rng, int64_t site, const OptTensor &residual) {
        ctx->save_for_backward({rng});
        ctx->saved_data["p"] = p;
        ctx->saved_data["site"] = site;
        ctx->saved_data["skip"] = residual.has_value() && residual->defined();
        return dropout_fwd(x, residual, p, rng, site);
    }
    static variable_list backward(AutogradContext *ctx, variable_list dy) {
        const auto saved = ctx->get_saved_variables();
        Tensor dx, ds;
        if (ctx->needs_input_grad(0))
            dx = dropout_fwd(dy[0], OptTensor(), ctx->saved_data["p"].toDouble(), saved[0], ctx->saved_data["site"].toInt());
        if (ctx->saved_data["skip"].toBool() && ctx->needs_input_grad(2)) ds = dy[0];
        return once({dx, Tensor(), Tensor(), Tensor(), ds}, "dropout");
    }
};

Tensor dropout(const Tensor &x, double p, const Tensor &rng, int64_t site, const OptTensor &residual) {
    const Tensor s = defined(residual);
    if (interposed("dropout", x, rng, s)) return Tensor();
    if (recorded(x, s)) return Dropout::apply(x, p, rng, site, residual);
    return dropout_fwd(x, residual, p, rng, site);
}

// ---- gated feed-forward --------------------------------------------------------------------------------------------
struct FfnCall {
    sr355_ffn_args a = {};
    std::vector<Tensor> keep;         // what has to outlive the call
    FfnCall(const char *who, const Tensor &x, const Tensor &w_gate, const Tensor &w_up, const Tensor &w_down, int64_t activation) {
        check_rows(who, x);
        const int64_t c = x.size(-1), f = w_gate.dim() == 2 ? w_gate.size(0) : 0;
        auto weight = [&](const char *name, const Tensor &w, int64_t n, int64_t k) {
            check_device(who, x, w);
            TORCH_CHECK(w.scalar_type() == x.scalar_type() && w.dim() == 2 && w.size(0) == n && w.size(1) == k && f >= 1, who, ": ", name,
                        " must have shape (", n, ", ", k, ") (at least one hidden channel) and x's type ", x.scalar_type(), ", got ",
                        w.sizes(), " of ", w.scalar_type());
            keep.push_back(w.contiguous());
            return keep.back().const_data_ptr();
        };
        a.w_gate_dev = weight("w_gate", w_gate, f, c);
        a.w_up_dev = weight("w_up", w_up, f, c);
        a.w_down_dev = weight("w_down", w_down, c, f);
        TORCH_CHECK(activation >= 0 && activation <= SR355_ACT_SIGMOID, who, ": unknown activation ", activation);
        TORCH_CHECK(c <= (1 << 20) && f <= (1 << 20), who, ": widths of ", c, " and ", f, "; up to 2^20 are supported");
        const Rows r(x);
        keep.push_back(r.t);
        a.dtype = code_of(x.scalar_type()), a.activation = static_cast<int>(activation);
        a.rows = x.numel() / c, a.channels = static_cast<int>(c), a.hidden = static_cast<int>(f);
        a.x_dev = r.data(), a.x_ld = r.ld;
    }
    void scratch_for(const Tensor &x, int backward) {
        const size_t bytes = api.gated_ffn_workspace_bytes(&a, backward);
        ok(bytes ? SR355_OK : SR355_ERR_INVALID, "sr355_gated_ffn_workspace_bytes");
        keep.push_back(scratch(x, bytes));
        a.workspace_dev = keep.back().mutable_data_ptr(), a.workspace_bytes = bytes;
    }
};

std::tuple<Tensor, Tensor> gated_ffn_fwd(const Tensor &x, const Tensor &w_gate, const Tensor &w_up, const Tensor &w_down,
                                         const OptTensor &b_gate, const OptTensor &b_up, const OptTensor &b_down, int64_t activation,
                                         bool want_saved) {
    FfnCall call("gated_ffn", x, w_gate, w_up, w_down, activation);
    sr355_ffn_args &a = call.a;
    auto bias = [&](const char *name, const OptTensor &b, int64_t n) -> const void * {
        const Tensor v = vector_of("gated_ffn", name, x, b, n, false);
        if (v.defined()) call.keep.push_back(v);
        return ptr(v);
    };
    a.b_gate_dev = bias("b_gate", b_gate, a.hidden);
    a.b_up_dev = bias("b_up", b_up, a.hidden);
    a.b_down_dev = bias("b_down", b_down, a.channels);
    Launch launch(x);
    Tensor y = at::empty(x.sizes(), x.options());
    Tensor saved = scratch(x, want_saved ? api.gated_ffn_saved_bytes(&a) : 0);
    a.y_dev = y.mutable_data_ptr();
    if (want_saved) a.saved_dev = saved.mutable_data_ptr(), a.saved_bytes = static_cast<size_t>(saved.numel());
    call.scratch_for(x, 0);
    ok(api.gated_ffn_fwd(&a, launch.stream), "sr355_gated_ffn_fwd");
    return {y, saved};
}

variable_list gated_ffn_bwd(const Tensor &dy, const Tensor &x, const Tensor &w_gate, const Tensor &w_up, const Tensor &w_down,
                            const Tensor &saved, int64_t activation, const std::vector<bool> &need) {
    const char *who = "gated_ffn backward";
    FfnCall call(who, x, w_gate, w_up, w_down, activation);
    sr355_ffn_args &a = call.a;
    check_device(who, x, dy);
    check_device(who, x, saved);
    TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && need.size() == 7,
                who, ": the gradient must have x's shape and type");
    TORCH_CHECK(saved.scalar_type() == at::kByte && saved.is_contiguous(), who, ": what the forward pass saved is a contiguous tensor of bytes");
    const Rows g(dy);
    a.dy_dev = g.data(), a.dy_ld = g.ld;
    a.saved_dev = a.rows ? const_cast<void *>(saved.const_data_ptr()) : nullptr, a.saved_bytes = static_cast<size_t>(saved.numel());
    Launch launch(x);
    variable_list out(7);
    const std::array<std::vector<int64_t>, 6> shapes = {w_gate.sizes().vec(), w_up.sizes().vec(), w_down.sizes().vec(),
                                                        {a.hidden}, {a.hidden}, {a.channels}};
    if (need[0]) out[0] = at::empty(x.sizes(), x.options());
    for (size_t i = 0; i < 6; ++i)
        if (need[i + 1]) out[i + 1] = at::empty(shapes[i], x.options());
    a.dx_dev = a.rows ? out_ptr(out[0]) : nullptr;
    a.dw_gate_dev = out_ptr(out[1]), a.dw_up_dev = out_ptr(out[2]), a.dw_down_dev = out_ptr(out[3]);
    a.db_gate_dev = out_ptr(out[4]), a.db_up_dev = out_ptr(out[5]), a.db_down_dev = out_ptr(out[6]);
    call.scratch_for(x, 1);
    ok(api.gated_ffn_bwd(&a, launch.stream), "sr355_gated_ffn_bwd");
    return out;
}

struct GatedFfn : torch::autograd::Function<GatedFfn> {
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w_gate, const Tensor &w_up, const Tensor &w_down,
                          const OptTensor &b_gate, const OptTensor &b_up, const OptTensor &b_down, int64_t activation) {
        auto [y, saved] = gated_ffn_fwd(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, true);
        ctx->save_for_backward({x, w_gate, w_up, w_down, saved});
        ctx->saved_data["activation"] = activation;
        ctx->saved_data["biases"] = static_cast<int64_t>(defined(b_gate).defined() | defined(b_up).defined() << 1 | defined(b_down).defined() << 2);
        return y;
    }
    static variable_list backward(AutogradContext *ctx, variable_list dy) {
        const auto s = ctx->get_saved_variables();
        std::vector<bool> need(7, false);
        const int64_t biases = ctx->saved_data["biases"].toInt();
        for (size_t i = 0, edge = 0; i < 7; ++i)
            if (i < 4 || (biases >> (i - 4) & 1)) need[i] = ctx->needs_input_grad(edge++);
        variable_list g = gated_ffn_bwd(dy[0], s[0], s[1], s[2], s[3], s[4], ctx->saved_data["activation"].toInt(), need);
        g.emplace_back();
        return once(std::move(g), "gated_ffn");
    }
};

Tensor gated_ffn(const Tensor &x, const Tensor &w_gate, const Tensor &w_up, const Tensor &w_down, const OptTensor &b_gate,
                 const OptTensor &b_up, const OptTensor &b_down, int64_t activation) {
    const Tensor bg = defined(b_gate), bu = defined(b_up), bd = defined(b_down);
    if (interposed("gated_ffn", x, w_gate, w_up, w_down, bg, bu, bd)) return Tensor();
    if (recorded(x, w_gate, w_up, w_down, bg, bu, bd))
        return GatedFfn::apply(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation);
    return std::get<0>(gated_ffn_fwd(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, false));
}

}  // namespace

PYBIND11_MODULE(_torch_tokens, m) {
    namespace py = pybind11;
    typedef py::call_guard<py::gil_scoped_release> free;
    m.def("connect", &connect);
    m.def("layer_norm", &layer_norm, free());
    m.def("dropout", &dropout, free());
    m.def("gated_ffn", &gated_ffn, free());
    m.def("layer_norm_fwd", &layer_norm_fwd, free());
    m.def("layer_norm_bwd", &layer_norm_bwd, free());
    m.def("dropout_fwd", &dropout_fwd, free());
    m.def("gated_ffn_fwd", &gated_ffn_fwd, free());
    m.def("gated_ffn_bwd", &gated_ffn_bwd, free());
}
