// row_autograd.cpp — the row operators' calls and their autograd nodes (layer norm, log probabilities of score rows, distillation).
//
// The kernels and the C entries are layer_norm.hip's and score_rows.hip's; here is what a call on torch tensors does around them:
// rows by strides, outputs, workspaces, the current stream, and the backward as a node of the graph.  It is C++ because of the
// backward: that runs on the engine's own thread, and for a small batch a Python backward costs more there than both kernels (a
// 64 x 5382 distillation step, whose kernels take 9 us: 97 us with the nodes in Python, 50 with these).  The entries are bound by
// address from the library that the Python package has loaded, so there is one copy of the kernels and one place that decides
// which library that is.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include "../../include/armnet_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

struct Calls {
    decltype(&armnet_strerror) strerror;
    decltype(&armnet_last_hip_error) last_hip_error;
    decltype(&armnet_layer_norm_fwd) layer_norm_fwd;
    decltype(&armnet_layer_norm_bwd_ws_bytes) layer_norm_bwd_ws_bytes;
    decltype(&armnet_layer_norm_bwd) layer_norm_bwd;
    decltype(&armnet_score_ws_bytes) score_ws_bytes;
    decltype(&armnet_score_logprobs_fwd) score_logprobs_fwd;
    decltype(&armnet_score_logprobs_bwd) score_logprobs_bwd;
    decltype(&armnet_distill_fwd) distill_fwd;
    decltype(&armnet_distill_bwd) distill_bwd;
};
Calls lib = {};

struct ArmnetError : std::runtime_error {
    using std::runtime_error::runtime_error;
};
PyObject* error_type = nullptr;      // armnet_hip.native.ArmnetNativeError

void check(int rc) {
    if (rc == ARMNET_OK) return;
    std::string what = "armnet_hip call failed (" + std::to_string(rc) + "): " + lib.strerror(rc);
    if (rc == ARMNET_ERR_HIP) what += std::string(": ") + lib.last_hip_error();
    throw ArmnetError(what);
}

int float_type(const Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kFloat: return ARMNET_F32;
        case at::kBFloat16: return ARMNET_BF16;
        case at::kHalf: return ARMNET_F16;
        default: throw ArmnetError(std::string(name) + ": expected float32, bfloat16 or float16, got " + c10::toString(t.scalar_type()));
    }
}

int id_type(const Tensor& t) {
    if (t.scalar_type() == at::kLong) return ARMNET_ID_I64;
    if (t.scalar_type() == at::kInt) return ARMNET_ID_I32;
    throw ArmnetError("ids must be int64 or int32");
}

void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor or_none(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }
// what memory holds is what the tensor says (a view that is negated on reading is copied)
Tensor as_stored(const Tensor& t) { return t.defined() ? t.resolve_neg() : t; }
MaybeTensor as_stored(const MaybeTensor& t) { return t.has_value() ? MaybeTensor(as_stored(*t)) : t; }
Tensor dense(const Tensor& t) { return t.defined() ? as_stored(t).contiguous() : t; }

// The rows of a tensor as the C entries take them: row r begins (r / inner) * outer + (r % inner) * stride elements behind x
// (inner = 0: r * stride).  Leading dimensions that two strides describe need no copy: slices, transposed batches, expanded rows.
struct Rows {
    Tensor x;                        // the tensor itself, or a dense copy
    int64_t n, inner = 0, outer = 0, stride, d;
};

Rows rows_of(const Tensor& x) {
    Rows o;
    const Tensor t = o.x = as_stored(x);
    o.d = t.size(-1);
    o.n = t.numel() / o.d;
    o.stride = o.d;
    if (t.is_contiguous()) return o;
    if (o.d == 1 || t.stride(-1) == 1) {
        int64_t size[2], step[2];
        int dims = 0;
        bool fits = true;
        for (int64_t i = 0; i + 1 < t.dim() && fits; ++i) {
            const int64_t n = t.size(i), s = t.stride(i);
            if (n == 1) continue;
            if (dims && step[dims - 1] == s * n) {         // adjacent to the dimension before: one
                size[dims - 1] *= n;
                step[dims - 1] = s;
            } else if (dims < 2) {
                size[dims] = n;
                step[dims++] = s;
            } else {
                fits = false;
            }
        }
        if (fits) {
            if (dims == 1) o.stride = step[0];
            if (dims == 2) {
                o.inner = size[1];
                o.outer = step[0];
                o.stride = step[1];
            }
            return o;
        }
    }
    o.x = t.contiguous();
    return o;
}

// x's device is the current one during a call: the library asks it for its size, and its stream is the current one
struct OnDevice {
    c10::DeviceGuard guard;
    void* stream;
    explicit OnDevice(const Tensor& x) : guard(device_of(x)) {
        stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream();
    }
    static c10::Device device_of(const Tensor& x) {
        if (!x.is_cuda()) throw ArmnetError("expected a tensor on the HIP device (no CPU fallback)");
        return x.device();
    }
};

void same_device(const Tensor& x, const Tensor& t, const char* name) {
    if (t.defined() && t.device() != x.device())
        throw ArmnetError(std::string(name) + " is on " + t.device().str() + ", the rows are on " + x.device().str());
}

Tensor fresh(const Tensor& like, at::IntArrayRef shape, at::ScalarType type) { return at::empty(shape, like.options().dtype(type)); }

std::vector<int64_t> lead(const Tensor& x, int64_t last = 0) {
    std::vector<int64_t> s(x.sizes().begin(), x.sizes().end() - 1);
    if (last) s.push_back(last);
    return s;
}

// Gradients of a backward that was asked for a graph of its own: they are right, but differentiating them raises.
variable_list once(variable_list grads, const char* name) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list in;
    for (auto& g : grads)
        if (g.defined()) in.push_back(g.detach().set_requires_grad(true));
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string("trying to differentiate twice the gradient of ") + name + ", which is differentiable once", (int64_t)in.size());
    variable_list out = (*error)(std::move(in));
    size_t k = 0;
    for (auto& g : grads)
        if (g.defined()) g = out[k++];
    return grads;
}

// What a call cannot do.  A tangent (forward-mode derivative) cannot pass the kernels; a result without one would be taken for a
// constant.  A trace records the outputs' allocation and not the kernels; what it replays would be memory that nothing wrote.
// A tensor without memory (a fake one, or one whose storage was freed) has its offset for an address.
void refuse(const char* name, std::initializer_list<const Tensor*> inputs) {
    using c10::impl::TorchDispatchModeTLS;
    if (torch::jit::tracer::isTracing() || TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value())
        throw ArmnetError(std::string(name) + ": a trace cannot record the kernels (call it outside of the traced part)");
    for (const Tensor* t : inputs) {
        if (!t->defined()) continue;
        if (t->_fw_grad(0).defined())
            throw ArmnetError(std::string(name) + ": forward-mode derivatives are not supported (use the backward pass)");
        if (t->numel() && !t->storage().data()) throw ArmnetError(std::string(name) + ": a tensor without memory (fake, or its storage was freed)");
    }
}

bool wants_graph(const Tensor& t) { return t.defined() && t.requires_grad() && at::GradMode::is_enabled(); }

// ---- layer norm ----------------------------------------------------------------------------------------------------------

std::pair<Tensor, Tensor> norm_forward(const Tensor& x_, const Tensor& weight, const Tensor& bias, double eps, bool stats) {
    OnDevice on(x_);
    const Rows x = rows_of(x_);
    same_device(x.x, weight, "weight");
    same_device(x.x, bias, "bias");
    Tensor y = fresh(x.x, x.x.sizes(), x.x.scalar_type());
    Tensor st = stats ? fresh(x.x, {2, x.n}, at::kFloat) : Tensor();           // mean, 1 / standard deviation
    float* mean = stats ? st.data_ptr<float>() : nullptr;
    const Tensor& p = weight.defined() ? weight : bias;
    if (x.n)
        check(lib.layer_norm_fwd(x.n, x.inner, x.outer, x.stride, x.d, float_type(x.x, "x"), x.x.data_ptr(),
                                 p.defined() ? float_type(p, "weight") : ARMNET_F32, address(weight), address(bias), (float)eps,
                                 y.data_ptr(), mean, stats ? mean + x.n : nullptr, on.stream));
    return {y, st};
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps) {
        const Tensor w = or_none(weight), b = or_none(bias);
        auto [y, st] = norm_forward(x, w, b, eps, true);
        ctx->save_for_backward({x, w, st});
        ctx->saved_data["type"] = (int64_t)(w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : at::kFloat);
        ctx->saved_data["need"] = (int64_t)(x.requires_grad() | (w.defined() && w.requires_grad()) << 1 | (b.defined() && b.requires_grad()) << 2);
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x_ = saved[0], &weight = saved[1], &st = saved[2];
        const int64_t need = ctx->saved_data["need"].toInt();
        const auto type = (at::ScalarType)ctx->saved_data["type"].toInt();
        refuse("layer_norm's backward", {&x_, &weight, &st, &grads[0]});
        OnDevice on(x_);
        const Rows x = rows_of(x_);
        const Tensor dy = dense(grads[0]);
        Tensor dx, dw, db, ws;
        if (need & 1) dx = fresh(x.x, x.x.sizes(), x.x.scalar_type());
        if (need & 2) dw = fresh(x.x, {x.d}, type);
        if (need & 4) db = fresh(x.x, {x.d}, type);
        const int64_t bytes = need & 6 ? lib.layer_norm_bwd_ws_bytes(x.n, x.d) : 0;
        if (bytes) ws = fresh(x.x, {bytes}, at::kByte);
        const float* mean = st.data_ptr<float>();
        check(lib.layer_norm_bwd(x.n, x.inner, x.outer, x.stride, x.d, float_type(x.x, "x"), x.x.data_ptr(), dy.data_ptr(),
                                 type == at::kFloat ? ARMNET_F32 : type == at::kBFloat16 ? ARMNET_BF16 : ARMNET_F16, address(weight), mean,
                                 mean + x.n, address(dx), address(dw), address(db), address(ws), bytes, on.stream));
        return once({dx, dw, db, Tensor()}, "layer_norm");
    }
};

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight_, const MaybeTensor& bias_, double eps) {
    const MaybeTensor weight = as_stored(weight_), bias = as_stored(bias_);
    const Tensor w = or_none(weight), b = or_none(bias);
    refuse("layer_norm", {&x, &w, &b});
    if (wants_graph(x) || wants_graph(w) || wants_graph(b)) return LayerNorm::apply(x, weight, bias, eps);
    return norm_forward(x, w, b, eps, false).first;
}

// ---- log probabilities ---------------------------------------------------------------------------------------------------

struct Answer {
    Tensor logp, entropy, top_logp, top_ids, stats;
};

// ids [.., n] dense beside the rows of X, or undefined
Answer scores_forward(const Tensor& X_, const Tensor& ids, double temperature, int64_t top, bool entropy, bool stats, const Tensor& word) {
    OnDevice on(X_);
    const Rows X = rows_of(X_);
    same_device(X.x, ids, "ids");
    const int64_t n_ids = ids.defined() ? ids.size(-1) : 0;
    if (ids.defined() && (ids.numel() != X.n * n_ids || !ids.is_contiguous())) throw ArmnetError("ids: expected a dense list for each row");
    Answer o;
    if (ids.defined()) o.logp = fresh(X.x, ids.sizes(), at::kFloat);
    if (entropy) o.entropy = fresh(X.x, lead(X.x), at::kFloat);
    if (top) {
        o.top_logp = fresh(X.x, lead(X.x, top), at::kFloat);
        o.top_ids = fresh(X.x, lead(X.x, top), at::kLong);
    }
    if (stats) o.stats = fresh(X.x, {X.n, 2}, at::kFloat);
    const int64_t bytes = lib.score_ws_bytes(X.n, X.d, (int)top);
    const Tensor ws = bytes > 0 ? fresh(X.x, {bytes}, at::kByte) : Tensor();
    if (X.n)
        check(lib.score_logprobs_fwd(X.n, X.inner, X.outer, X.stride, X.d, float_type(X.x, "X"), X.x.data_ptr(), (float)temperature, n_ids,
                                     address(ids), ids.defined() ? id_type(ids) : ARMNET_ID_I64, (int)top, (float*)address(o.logp),
                                     (float*)address(o.entropy), (float*)address(o.top_logp), (int64_t*)address(o.top_ids),
                                     (float*)address(o.stats), address(ws), bytes, (int32_t*)address(word), on.stream));
    return o;
}

struct ScoreLogprobs : torch::autograd::Function<ScoreLogprobs> {
    // outputs: those of logp, entropy, top_logp, top_ids that there are
    static variable_list forward(AutogradContext* ctx, const Tensor& X, const MaybeTensor& ids_, double temperature, int64_t top, bool entropy,
                                 const MaybeTensor& word) {
        const Tensor ids = or_none(ids_);
        const Answer o = scores_forward(X, ids, temperature, top, entropy, true, or_none(word));
        ctx->save_for_backward({X, ids, o.stats, o.entropy});
        ctx->saved_data["t"] = temperature;
        ctx->saved_data["has"] = (int64_t)(ids.defined() | entropy << 1);
        ctx->set_materialize_grads(false);
        variable_list out;
        if (ids.defined()) out.push_back(o.logp);
        if (entropy) out.push_back(o.entropy);
        if (top) {
            out.push_back(o.top_logp);
            out.push_back(o.top_ids);
            ctx->mark_non_differentiable({o.top_logp, o.top_ids});
        }
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &X_ = saved[0], &ids = saved[1], &stats = saved[2], &entropy = saved[3];
        const int64_t has = ctx->saved_data["has"].toInt();
        Tensor g_logp, g_entropy, dx;
        if (has & 1) g_logp = grads[0];
        if (has & 2) g_entropy = grads[has & 1];
        refuse("score_logprobs' backward", {&X_, &ids, &stats, &entropy, &g_logp, &g_entropy});
        g_logp = dense(g_logp);
        g_entropy = dense(g_entropy);
        if (g_logp.defined() || g_entropy.defined()) {
            OnDevice on(X_);
            const Rows X = rows_of(X_);
            dx = fresh(X.x, X.x.sizes(), X.x.scalar_type());
            if (X.n)
                check(lib.score_logprobs_bwd(X.n, X.inner, X.outer, X.stride, X.d, float_type(X.x, "X"), X.x.data_ptr(),
                                             (float)ctx->saved_data["t"].toDouble(), ids.defined() ? ids.size(-1) : 0, address(ids),
                                             ids.defined() ? id_type(ids) : ARMNET_ID_I64, stats.data_ptr<float>(),
                                             (float*)address(entropy), (float*)address(g_logp), (float*)address(g_entropy), dx.data_ptr(),
                                             on.stream));
        }
        return once({dx, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, "score_logprobs");
    }
};

std::tuple<MaybeTensor, MaybeTensor, MaybeTensor, MaybeTensor> score_logprobs(const Tensor& X, const MaybeTensor& ids_, double temperature,
                                                                              int64_t top, bool entropy, const MaybeTensor& word) {
    const MaybeTensor ids = as_stored(ids_);
    const Tensor list = or_none(ids);
    refuse("score_logprobs", {&X, &list});
    auto some = [](const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); };
    if (wants_graph(X) && (ids.has_value() || entropy || top)) {
        const variable_list out = ScoreLogprobs::apply(X, ids, temperature, top, entropy, word);
        size_t k = 0;
        auto next = [&](bool there) { return there ? MaybeTensor(out[k++]) : MaybeTensor(); };
        MaybeTensor logp = next(ids.has_value()), ent = next(entropy), tl = next(top), ti = next(top);
        return {logp, ent, tl, ti};
    }
    const Answer o = scores_forward(X, list, temperature, top, entropy, false, or_none(word));
    return {some(o.logp), some(o.entropy), some(o.top_logp), some(o.top_ids)};
}

// ---- distillation --------------------------------------------------------------------------------------------------------

std::pair<Tensor, Tensor> distill_forward(const Tensor& X_, const Tensor& ids, const Tensor& teacher, double temperature, bool stats,
                                          const Tensor& word) {
    OnDevice on(X_);
    const Rows X = rows_of(X_);
    same_device(X.x, ids, "top_ids");
    same_device(X.x, teacher, "top_scores");
    const int64_t k = ids.size(-1);
    if (ids.numel() != X.n * k || teacher.numel() != X.n * k || !ids.is_contiguous() || !teacher.is_contiguous())
        throw ArmnetError("top_ids, top_scores: expected a dense list for each row");
    Tensor loss = fresh(X.x, lead(X.x), at::kFloat);
    Tensor st = stats ? fresh(X.x, {X.n, 4}, at::kFloat) : Tensor();
    const int64_t bytes = lib.score_ws_bytes(X.n, X.d, 0);
    const Tensor ws = bytes > 0 ? fresh(X.x, {bytes}, at::kByte) : Tensor();
    if (X.n)
        check(lib.distill_fwd(X.n, X.inner, X.outer, X.stride, X.d, float_type(X.x, "X"), X.x.data_ptr(), (float)temperature, k, ids.data_ptr(),
                              id_type(ids), float_type(teacher, "top_scores"), teacher.data_ptr(), loss.data_ptr<float>(), (float*)address(st),
                              address(ws), bytes, (int32_t*)address(word), on.stream));
    return {loss, st};
}

struct Distill : torch::autograd::Function<Distill> {
    static Tensor forward(AutogradContext* ctx, const Tensor& X, const Tensor& ids, const Tensor& teacher, double temperature,
                          const MaybeTensor& word) {
        auto [loss, st] = distill_forward(X, ids, teacher, temperature, true, or_none(word));
        ctx->save_for_backward({X, ids, teacher, st});
        ctx->saved_data["t"] = temperature;
        return loss;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &X_ = saved[0], &ids = saved[1], &teacher = saved[2], &st = saved[3];
        refuse("distill_loss' backward", {&X_, &ids, &teacher, &st, &grads[0]});
        OnDevice on(X_);
        const Rows X = rows_of(X_);
        const Tensor g = dense(grads[0]);
        Tensor dx = fresh(X.x, X.x.sizes(), X.x.scalar_type());
        if (X.n)
            check(lib.distill_bwd(X.n, X.inner, X.outer, X.stride, X.d, float_type(X.x, "X"), X.x.data_ptr(),
                                  (float)ctx->saved_data["t"].toDouble(), ids.size(-1), ids.data_ptr(), id_type(ids),
                                  float_type(teacher, "top_scores"), teacher.data_ptr(), st.data_ptr<float>(), g.data_ptr<float>(),
                                  dx.data_ptr(), on.stream));
        return once({dx, Tensor(), Tensor(), Tensor(), Tensor()}, "distill_loss");
    }
};

Tensor distill_loss(const Tensor& X, const Tensor& ids_, const Tensor& teacher_, double temperature, const MaybeTensor& word) {
    const Tensor ids = as_stored(ids_), teacher = as_stored(teacher_);
    refuse("distill_loss", {&X, &ids, &teacher});
    if (wants_graph(X)) return Distill::apply(X, ids, teacher, temperature, word);
    return distill_forward(X, ids, teacher, temperature, false, or_none(word)).first;
}

void bind(const std::map<std::string, uintptr_t>& at, py::object error) {
    Calls c;
#define ARMNET_BIND(name) c.name = (decltype(c.name))at.at("armnet_" #name)
    ARMNET_BIND(strerror);
    ARMNET_BIND(last_hip_error);
    ARMNET_BIND(layer_norm_fwd);
    ARMNET_BIND(layer_norm_bwd_ws_bytes);
    ARMNET_BIND(layer_norm_bwd);
    ARMNET_BIND(score_ws_bytes);
    ARMNET_BIND(score_logprobs_fwd);
    ARMNET_BIND(score_logprobs_bwd);
    ARMNET_BIND(distill_fwd);
    ARMNET_BIND(distill_bwd);
#undef ARMNET_BIND
    lib = c;
    error_type = error.release().ptr();
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const ArmnetError& e) {
            PyErr_SetString(error_type ? error_type : PyExc_RuntimeError, e.what());
        }
    });
    m.attr("abi_version") = ARMNET_ABI_VERSION;      // of the entries' signatures, which are compiled in
    m.def("bind", &bind);
    m.def("layer_norm", &layer_norm, py::call_guard<py::gil_scoped_release>());
    m.def("score_logprobs", &score_logprobs, py::call_guard<py::gil_scoped_release>());
    m.def("distill_loss", &distill_loss, py::call_guard<py::gil_scoped_release>());
    m.def("rows_of", [](const Tensor& t) {
        const Rows o = rows_of(t);
        return std::make_tuple(o.x, o.n, o.inner, o.outer, o.stride);
    });
}
