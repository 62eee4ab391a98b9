// Torch side of the row operators (rms_norm.hip, token_logprobs.hip, grad_norm.hip): argument checks, outputs and workspaces from torch's
// allocator, autograd nodes, and the list of gradients.  Host code only; the kernels are reached through the C ABI (include/i2p_ops.h), whose
// addresses i2pnet_amd/ops.py hands over, so that one loaded library serves both.
//
// Why not Python over ctypes, as for the other operators: these calls are short (2 .. 20 us on the device).  A backward pass in Python costs
// about 90 us for the hand-over of the interpreter to autograd's device thread alone, and a list of 254 gradients 100 us of attribute reads.
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>
#include <ATen/ATen.h>

#include "../../include/i2p_ops.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// ---- the C ABI -------------------------------------------------------------------------------------------------------------------
struct {
#define I2P_ENTRY(name) decltype(&::i2p_##name) name = nullptr;
#define I2P_ENTRIES                                                                                                                   \
    I2P_ENTRY(rms_norm_fwd) I2P_ENTRY(rms_norm_q8) I2P_ENTRY(rms_norm_bwd) I2P_ENTRY(rms_norm_bwd_scratch) I2P_ENTRY(token_logprobs_fwd) \
    I2P_ENTRY(token_logprobs_bwd) I2P_ENTRY(token_logprobs_scratch) I2P_ENTRY(clip_grad_norm) I2P_ENTRY(grad_norm_scratch)
    I2P_ENTRIES
#undef I2P_ENTRY
} abi;

void bind(const std::map<std::string, uintptr_t> &entries) {
    auto find = [&](const char *name) {
        const auto it = entries.find(name);
        TORCH_CHECK(it != entries.end() && it->second, name, " is not in the loaded library");
        return it->second;
    };
#define I2P_ENTRY(name) abi.name = reinterpret_cast<decltype(abi.name)>(find("i2p_" #name));
    I2P_ENTRIES
#undef I2P_ENTRY
}

// `device` current for a launch, and its current stream
struct On {
    c10::DeviceIndex before, device;
    explicit On(const c10::Device &d) : before(c10::hip::current_device()), device(d.index()) {
        if (device != before) c10::hip::set_device(device);
    }
    ~On() {
        if (device != before) c10::hip::set_device(before);
    }
    void *stream() const { return (void *)c10::hip::getCurrentHIPStream(device).stream(); }
};

void check(int rc, const char *name) {
    TORCH_CHECK(rc == 0, name, " failed: ", rc == I2P_ERR_BAD_ARG ? "bad argument" : rc == I2P_ERR_OVERLAP ? "tensors of the list share memory"
                : "hipError_t ", rc > 0 ? std::to_string(rc) : "");
}

int type_of(const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return I2P_F32;
        case at::kBFloat16: return I2P_BF16;
        case at::kHalf: return I2P_F16;
        default: return -1;
    }
}

void *ptr(const OptTensor &t) { return t ? t->data_ptr() : nullptr; }

// The kernels are launched by address, which nothing that records torch's operators sees: a trace would hold the allocation of the outputs
// alone and return what memory held when it is replayed
void eager(const char *name) {
    using c10::impl::TorchDispatchModeTLS;
    TORCH_CHECK(!torch::jit::tracer::isTracing() && !TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value() &&
                    !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch),
                name, " cannot be traced (torch.jit.trace, make_fx, torch.export): the trace would not hold its kernels");
}

// A forward-mode tangent would be lost without a word: the outputs come from the kernels and carry none
void primal(const Tensor &t, const char *what) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), what, " has a forward-mode tangent: the row operators have no forward-mode derivative");
}
void primal(const OptTensor &t, const char *what) {
    if (t) primal(*t, what);
}

// the values that a tensor stands for, in memory: torch may keep a sign beside it as a flag (the imaginary part of a conjugate)
Tensor plain(const Tensor &t) { return t.is_neg() ? t.resolve_neg() : t; }
OptTensor plain(const OptTensor &t) { return t ? OptTensor(plain(*t)) : std::nullopt; }

// a tensor [..., d] as rows of pitch ld; a copy only where the columns are not next to each other or rows overlap
struct Rows {
    Tensor t;
    int64_t n, d, ld;
    int type;
    Rows(const Tensor &x, const char *what, const Tensor *like = nullptr) {
        primal(x, what);
        TORCH_CHECK(x.is_cuda(), what, " must be a cuda tensor (got ", x.device(), ")");
        type = type_of(x);
        TORCH_CHECK(type >= 0, what, " must be float32, bfloat16 or float16 (got ", x.scalar_type(), ")");
        if (like)
            TORCH_CHECK(x.sizes() == like->sizes() && x.scalar_type() == like->scalar_type() && x.device() == like->device(), what, " must be ",
                        like->scalar_type(), " ", like->sizes(), " on ", like->device(), " (got ", x.scalar_type(), " ", x.sizes(), " on ",
                        x.device(), ")");
        TORCH_CHECK(x.dim() > 0 && x.size(-1) > 0, what, " must have rows of at least one element (got ", x.sizes(), ")");
        d = x.size(-1);
        TORCH_CHECK(d <= I2P_MAX_ROW, what, ": rows of ", d, " elements are too long");
        n = x.numel() / d;
        ld = d;
        t = plain(x);
        if (t.is_contiguous()) return;
        if (x.dim() != 2) t = t.reshape({n, d});
        if ((d > 1 && t.stride(1) != 1) || (n > 1 && t.stride(0) < d)) t = t.contiguous();
        if (n > 1) ld = t.stride(0);
    }
};

// Gradients of a backward pass that cannot be differentiated again.  They get a history that says so when it is walked: an error node above all
// that they depend on, the operator's inputs and the gradients `from` that came in, so that no way to a second derivative takes it for zero
variable_list once(variable_list g, const variable_list &from) {
    if (!at::GradMode::is_enabled()) return g;
    torch::autograd::edge_list above = torch::autograd::collect_next_edges(from);
    if (const auto node = torch::autograd::get_current_node()) above.insert(above.end(), node->next_edges().begin(), node->next_edges().end());
    const auto error = std::make_shared<torch::autograd::Error>("trying to differentiate twice a function marked once_differentiable", std::move(above));
    for (auto &t : g)
        if (t.defined()) {
            t = t.detach();
            torch::autograd::set_history(t, error);
        }
    return g;
}

// ---- RMS norm --------------------------------------------------------------------------------------------------------------------
int weight_type(const OptTensor &w, const Tensor &x, int64_t d) {
    if (!w) return I2P_F32;
    TORCH_CHECK(w->device() == x.device() && w->dim() == 1 && w->size(0) == d && (w->scalar_type() == at::kFloat || w->scalar_type() == x.scalar_type()) &&
                    w->is_contiguous(),
                "weight must be a contiguous float32 or ", x.scalar_type(), " [", d, "] on ", x.device(), " (got ", w->scalar_type(), " ", w->sizes(),
                " on ", w->device(), ")");
    return type_of(*w);
}

// -> y, the stream (x itself, as rows, without a residual), rstd (undefined unless wanted)
std::tuple<Tensor, Tensor, Tensor> rms_norm_forward(const Tensor &x, const OptTensor &weight, const OptTensor &residual, double eps, bool want_rstd) {
    eager("rms_norm");
    primal(residual, "residual");
    primal(weight, "weight");
    const Rows a(x, "x");
    std::optional<Rows> r;
    if (residual) r.emplace(*residual, "residual", &x);
    const int wt = weight_type(weight, x, a.d);
    const OptTensor w = plain(weight);
    Tensor y = at::empty(x.sizes(), x.options()), s = r ? at::empty(x.sizes(), x.options()) : a.t, rstd;
    if (want_rstd) rstd = at::empty({a.n}, x.options().dtype(at::kFloat));
    const On on(x.device());
    check(abi.rms_norm_fwd(a.n, (int)a.d, a.type, wt, a.t.data_ptr(), a.ld, r ? r->t.data_ptr() : nullptr, r ? r->ld : 0, ptr(w), (float)eps,
                           r ? s.data_ptr() : nullptr, y.data_ptr(), want_rstd ? rstd.data_ptr<float>() : nullptr, on.stream()),
          "i2p_rms_norm_fwd");
    return {y, s, rstd};
}

std::tuple<Tensor, Tensor, OptTensor> rms_norm_q8(const Tensor &x, const OptTensor &weight, const OptTensor &residual, double eps, int64_t group) {
    eager("rms_norm_q8");
    TORCH_CHECK(!at::GradMode::is_enabled() || !(x.requires_grad() || (weight && weight->requires_grad()) || (residual && residual->requires_grad())),
                "rms_norm_q8 has no gradient: call it under torch.no_grad() or on detached tensors");
    primal(residual, "residual");
    primal(weight, "weight");
    TORCH_CHECK_VALUE(group == 0 || (group >= 32 && group <= 512 && (group & (group - 1)) == 0),
                      "rms_norm_q8: group must be 0 (the whole row) or a power of two from 32 to 512 (got ", group, ")");
    const Rows a(x, "x");
    std::optional<Rows> r;
    if (residual) r.emplace(*residual, "residual", &x);
    const int wt = weight_type(weight, x, a.d);
    const OptTensor w = plain(weight);
    std::vector<int64_t> groups = x.sizes().vec();
    groups.back() = group ? (a.d + group - 1) / group : 1;
    Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn)), scale = at::empty(groups, x.options().dtype(at::kFloat));
    OptTensor s;
    if (r) s = at::empty(x.sizes(), x.options());
    const On on(x.device());
    check(abi.rms_norm_q8(a.n, (int)a.d, a.type, wt, a.t.data_ptr(), a.ld, r ? r->t.data_ptr() : nullptr, r ? r->ld : 0, ptr(w), (float)eps,
                          (int)group, ptr(s), (unsigned char *)q.data_ptr(), scale.data_ptr<float>(), on.stream()),
          "i2p_rms_norm_q8");
    return {q, scale, s};
}

// gs: the stream's gradient or none; s may be given as rows -> dx like gy, dw like weight
std::tuple<Tensor, OptTensor> rms_norm_backward(const Tensor &s, const OptTensor &weight, const Tensor &rstd, const Tensor &gy, const OptTensor &gs,
                                                bool need_dw) {
    eager("rms_norm");
    primal(s, "s");
    primal(gs, "gs");
    const Rows g(gy, "gy"), a(s, "s");
    TORCH_CHECK(a.n == g.n && a.d == g.d && a.type == g.type && s.device() == gy.device(), "gy must be ", s.scalar_type(), " with the rows of s");
    std::optional<Rows> e;
    if (gs) e.emplace(*gs, "gs", &gy);
    const int wt = weight_type(weight, s, a.d);
    const OptTensor w = plain(weight);
    TORCH_CHECK(rstd.is_contiguous() && rstd.scalar_type() == at::kFloat && rstd.numel() == a.n && rstd.device() == s.device(), "rstd must be float32 [", a.n, "]");
    Tensor dx = at::empty(gy.sizes(), gy.options());
    OptTensor dw, scratch;
    TORCH_CHECK(!need_dw || weight, "rms_norm_backward: the weight's gradient is wanted, but there is no weight");
    if (need_dw) dw = a.n ? at::empty(weight->sizes(), weight->options()) : at::zeros(weight->sizes(), weight->options());
    if (a.n == 0) return {dx, dw};
    if (need_dw) scratch = at::empty({abi.rms_norm_bwd_scratch(a.n, (int)a.d)}, gy.options().dtype(at::kByte));
    const On on(gy.device());
    check(abi.rms_norm_bwd(a.n, (int)a.d, a.type, wt, a.t.data_ptr(), a.ld, g.t.data_ptr(), g.ld, e ? e->t.data_ptr() : nullptr, e ? e->ld : 0, ptr(w),
                           rstd.data_ptr<float>(), dx.data_ptr(), ptr(dw), ptr(scratch), on.stream()),
          "i2p_rms_norm_bwd");
    return {dx, dw};
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const OptTensor &residual, const OptTensor &weight, double eps) {
        auto [y, s, rstd] = rms_norm_forward(x, weight, residual, eps, true);
        ctx->set_materialize_grads(false);
        variable_list saved{s, rstd};
        if (weight) saved.push_back(*weight);
        ctx->save_for_backward(std::move(saved));
        ctx->saved_data["residual"] = residual.has_value();
        return residual ? variable_list{y, s} : variable_list{y};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        const variable_list saved = ctx->get_saved_variables();
        const bool residual = ctx->saved_data["residual"].toBool();
        OptTensor weight, gs;
        if (saved.size() > 2) weight = saved[2];
        if (residual && g[1].defined()) gs = g[1];
        if (!g[0].defined()) return once({gs.value_or(Tensor()), residual ? gs.value_or(Tensor()) : Tensor(), Tensor(), Tensor()}, g);
        auto [dx, dw] = rms_norm_backward(saved[0], weight, saved[1], g[0], gs, weight && ctx->needs_input_grad(residual ? 2 : 1));
        return once({dx, residual ? dx : Tensor(), dw.value_or(Tensor()), Tensor()}, g);
    }
};

bool wants_grad(const Tensor &x, const OptTensor &a, const OptTensor &b) {
    return at::GradMode::is_enabled() && (x.requires_grad() || (a && a->requires_grad()) || (b && b->requires_grad()));
}

Tensor rms_norm(const Tensor &x, const OptTensor &weight, double eps) {
    if (!wants_grad(x, weight, std::nullopt)) return std::get<0>(rms_norm_forward(x, weight, std::nullopt, eps, false));
    return RmsNorm::apply(x, OptTensor(), weight, eps)[0];
}

std::tuple<Tensor, Tensor> rms_norm_residual(const Tensor &x, const OptTensor &weight, const Tensor &residual, double eps) {
    if (!wants_grad(x, weight, residual)) {
        auto [y, s, rstd] = rms_norm_forward(x, weight, residual, eps, false);
        return {y, s};
    }
    const variable_list out = RmsNorm::apply(x, OptTensor(residual), weight, eps);
    return {out[0], out[1]};
}

// ---- log probabilities -----------------------------------------------------------------------------------------------------------
// -> logp, entropy, top_logp, top_ids, the scores as rows, ids (contiguous), stat
using Logprobs = std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor>;
Logprobs token_logprobs_forward(const Tensor &logits, const Tensor &ids, int64_t top, int64_t ignore_index, bool want_stat) {
    eager("token_logprobs");
    const Rows a(logits, "logits");
    TORCH_CHECK(ids.scalar_type() == at::kLong && ids.device() == logits.device() && ids.sizes() == logits.sizes().slice(0, logits.dim() - 1),
                "ids must be int64 ", logits.sizes().slice(0, logits.dim() - 1), " on ", logits.device(), " (got ", ids.scalar_type(), " ", ids.sizes(),
                " on ", ids.device(), ")");
    TORCH_CHECK_VALUE(a.d <= I2P_MAX_CANDIDATES, "token_logprobs: rows of at most ", I2P_MAX_CANDIDATES, " candidates (got ", a.d, ")");
    TORCH_CHECK_VALUE(top >= 0 && top <= a.d && top <= I2P_MAX_TOP, "token_logprobs: top must be between 0 and ", std::min<int64_t>(a.d, I2P_MAX_TOP),
                      " (got ", top, ")");
    const Tensor id = plain(ids).contiguous();
    const auto f32 = logits.options().dtype(at::kFloat);
    std::vector<int64_t> list = ids.sizes().vec();
    list.push_back(top);
    Tensor logp = at::empty(ids.sizes(), f32), entropy = at::empty(ids.sizes(), f32), stat, top_logp = at::empty(list, f32),
           top_ids = at::empty(list, id.options());
    if (want_stat) stat = at::empty({a.n, 2}, f32);
    OptTensor scratch;
    if (const int64_t bytes = abi.token_logprobs_scratch(a.n, (int)a.d, a.type, (int)top)) scratch = at::empty({bytes}, f32.dtype(at::kByte));
    const On on(logits.device());
    check(abi.token_logprobs_fwd(a.n, (int)a.d, a.type, a.t.data_ptr(), a.ld, id.data_ptr<int64_t>(), ignore_index, (int)top, logp.data_ptr<float>(),
                                 entropy.data_ptr<float>(), want_stat ? stat.data_ptr<float>() : nullptr, top_logp.data_ptr<float>(), top_ids.data_ptr<int64_t>(), ptr(scratch),
                                 on.stream()),
          "i2p_token_logprobs_fwd");
    return {logp, entropy, top_logp, top_ids, a.t, id, stat};
}

// x2, ids, stat, entropy as the forward left them -> the gradient, dense, like x2
Tensor token_logprobs_backward(const Tensor &x2, const Tensor &ids, int64_t ignore_index, const Tensor &stat, const Tensor &entropy, const OptTensor &g_logp,
                               const OptTensor &g_entropy) {
    eager("token_logprobs");
    primal(g_logp, "g_logp");
    primal(g_entropy, "g_entropy");
    const Rows a(x2, "logits");
    auto dense = [&](const OptTensor &g, const char *what) -> OptTensor {
        if (!g) return std::nullopt;
        TORCH_CHECK(g->scalar_type() == at::kFloat && g->device() == x2.device() && g->numel() == a.n, what, " must be float32 with ", a.n, " elements");
        return plain(*g).contiguous();
    };
    TORCH_CHECK(ids.is_contiguous() && ids.numel() == a.n && stat.is_contiguous() && stat.numel() == 2 * a.n && entropy.is_contiguous() &&
                    entropy.numel() == a.n, "token_logprobs: ids, stat and entropy must be the forward's");
    const OptTensor gl = dense(g_logp, "g_logp"), gh = dense(g_entropy, "g_entropy");
    Tensor dx = at::empty(x2.sizes(), x2.options());
    const On on(x2.device());
    check(abi.token_logprobs_bwd(a.n, (int)a.d, a.type, a.t.data_ptr(), a.ld, ids.data_ptr<int64_t>(), ignore_index, stat.data_ptr<float>(),
                                 entropy.data_ptr<float>(), (const float *)ptr(gl), (const float *)ptr(gh), dx.data_ptr(), on.stream()),
          "i2p_token_logprobs_bwd");
    return dx;
}

struct TokenLogprobs : torch::autograd::Function<TokenLogprobs> {
    static variable_list forward(AutogradContext *ctx, const Tensor &logits, const Tensor &ids, int64_t top, int64_t ignore_index) {
        auto [logp, entropy, top_logp, top_ids, x2, id, stat] = token_logprobs_forward(logits, ids, top, ignore_index, true);
        ctx->set_materialize_grads(false);
        ctx->mark_non_differentiable({top_logp, top_ids});
        ctx->save_for_backward({x2, id, stat, entropy});
        ctx->saved_data["ignore"] = ignore_index;
        ctx->saved_data["shape"] = logits.sizes().vec();
        return {logp, entropy, top_logp, top_ids};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        if (!g[0].defined() && !g[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
        const variable_list s = ctx->get_saved_variables();
        const Tensor dx = token_logprobs_backward(s[0], s[1], ctx->saved_data["ignore"].toInt(), s[2], s[3], g[0].defined() ? OptTensor(g[0]) : OptTensor(),
                                                  g[1].defined() ? OptTensor(g[1]) : OptTensor());
        return once({dx.view(ctx->saved_data["shape"].toIntVector()), Tensor(), Tensor(), Tensor()}, g);
    }
};

std::tuple<Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor &logits, const Tensor &ids, int64_t top, int64_t ignore_index) {
    if (!wants_grad(logits, std::nullopt, std::nullopt)) {
        auto [logp, entropy, top_logp, top_ids, x2, id, stat] = token_logprobs_forward(logits, ids, top, ignore_index, false);
        return {logp, entropy, top_logp, top_ids};
    }
    const variable_list o = TokenLogprobs::apply(logits, ids, top, ignore_index);
    return {o[0], o[1], o[2], o[3]};
}

// ---- gradient norm ---------------------------------------------------------------------------------------------------------------
// the gradients meant by one tensor or an iterable of them: a parameter's .grad (where it has one), or the gradient tensor itself; `device`:
// of the first of them
std::vector<Tensor> grad_list(const py::object &parameters, std::optional<c10::Device> *device = nullptr) {
    std::vector<Tensor> grads;
    auto add = [&](PyObject *o) {
        if (Py_TYPE(o) == (PyTypeObject *)THPVariableClass) {
            const Tensor &t = THPVariable_Unpack(o);
            if (!t.requires_grad()) { grads.push_back(t); return; }
        }
        TORCH_CHECK(THPVariable_Check(o), "parameters (leaves) or gradient tensors are wanted (got ", Py_TYPE(o)->tp_name, ")");
        const Tensor &t = THPVariable_Unpack(o);
        TORCH_CHECK(t.requires_grad() || !ParameterClass || PyObject_IsInstance(o, ParameterClass) == 1,
                    "parameters (leaves) or gradient tensors are wanted (got ", Py_TYPE(o)->tp_name, " without a gradient)");
        TORCH_CHECK(t.is_leaf(), "parameters (leaves) or gradient tensors are wanted (got a tensor that an operation made and that requires a gradient)");
        if (t.grad().defined()) grads.push_back(t.grad());
        else if (device && !*device) *device = t.device();
    };
    if (THPVariable_Check(parameters.ptr())) { add(parameters.ptr()); return grads; }
    const auto list = py::reinterpret_steal<py::object>(PySequence_Fast(parameters.ptr(), "parameters, gradient tensors or one of them are wanted"));
    if (!list) throw py::error_already_set();
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(list.ptr());
    grads.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) add(PySequence_Fast_GET_ITEM(list.ptr(), i));
    return grads;
}

// total norm f32 0-d of a list that is not empty; no max_norm: nothing is clipped
Tensor clip_grad_norm(const std::vector<Tensor> &grads, int64_t kind, std::optional<double> max_norm, const OptTensor &out) {
    eager("clip_grad_norm");
    TORCH_CHECK(!grads.empty(), "clip_grad_norm: no gradients");
    primal(out, "out");
    const auto device = grads[0].device();
    const int n = (int)grads.size();
    std::vector<const void *> ptrs(n);
    std::vector<long long> sizes(n);
    std::vector<int> types(n);
    const bool forward_mode = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;       // (asking 254 tensors takes 1 .. 3 us)
    std::vector<Tensor> copies;                 // (in place a flagged sign changes nothing: what is scaled is its negative)
    long long total = 0;
    for (int i = 0; i < n; ++i) {
        const Tensor &g = grads[i];
        if (forward_mode) primal(g, "a gradient");
        types[i] = type_of(g);
        TORCH_CHECK(types[i] >= 0, "gradients must be float32, bfloat16 or float16 (got ", g.scalar_type(), ")");
        TORCH_CHECK(g.is_cuda() && g.device() == device, "gradients must be cuda tensors on one device (got ", g.device(), ")");
        TORCH_CHECK(g.layout() == at::kStrided && g.is_non_overlapping_and_dense(), "gradients must be dense (got sizes ", g.sizes(), ", strides ",
                    g.layout() == at::kStrided ? g.strides() : at::IntArrayRef(), ")");
        if (out && g.is_neg()) copies.push_back(g.resolve_neg());
        ptrs[i] = out && g.is_neg() ? copies.back().data_ptr() : g.data_ptr();
        total += sizes[i] = g.numel();
    }
    if (out)
        TORCH_CHECK(out->device() == device && out->scalar_type() == at::kFloat && out->dim() == 1 && out->is_contiguous() && out->numel() == total &&
                        !out->is_neg() && !(out->requires_grad() && out->is_leaf()),
                    "out must be a contiguous float32 [", total, "] on ", device, " (got ", out->scalar_type(), " ", out->sizes(), " on ", out->device(), ")");
    const auto f32 = grads[0].options().dtype(at::kFloat).memory_format(std::nullopt);
    const Tensor scratch = at::empty({abi.grad_norm_scratch(n, sizes.data())}, f32.dtype(at::kByte)), norm = at::empty({}, f32);
    if (max_norm) {                             // what autograd saved of them is stale from here on
        if (out) out->unsafeGetTensorImpl()->bump_version();
        else
            for (const Tensor &g : grads) g.unsafeGetTensorImpl()->bump_version();
    }
    const On on(device);
    check(abi.clip_grad_norm(n, ptrs.data(), sizes.data(), types.data(), (int)kind, max_norm.has_value(), (float)max_norm.value_or(0.0),
                             out ? out->data_ptr<float>() : nullptr, scratch.data_ptr(), norm.data_ptr<float>(), on.stream()),
          "i2p_clip_grad_norm");
    return norm;
}

// the same on parameters or gradients.  Parameters without gradients have a norm of 0 on their device; no parameter at all: on the current one
Tensor clip_parameters(const py::object &parameters, int64_t kind, std::optional<double> max_norm, const OptTensor &out) {
    std::optional<c10::Device> device;
    const std::vector<Tensor> grads = grad_list(parameters, &device);
    if (grads.empty()) {
        TORCH_CHECK(!max_norm || !out || out->numel() == 0, "out must be empty: there is no gradient");
        return at::zeros({}, at::TensorOptions().dtype(at::kFloat).device(device.value_or(c10::Device(c10::kCUDA))));
    }
    return clip_grad_norm(grads, kind, max_norm, out);
}

}  // namespace

PYBIND11_MODULE(_torch_rows, m) {
    using torch::wrap_pybind_function;
    using torch::wrap_pybind_function_no_gil;
    m.def("bind", wrap_pybind_function(bind));
    m.def("rms_norm", wrap_pybind_function_no_gil(rms_norm));
    m.def("rms_norm_residual", wrap_pybind_function_no_gil(rms_norm_residual));
    m.def("rms_norm_q8", wrap_pybind_function_no_gil(rms_norm_q8));
    m.def("rms_norm_forward", wrap_pybind_function_no_gil(rms_norm_forward));
    m.def("rms_norm_backward", wrap_pybind_function_no_gil(rms_norm_backward));
    m.def("token_logprobs", wrap_pybind_function_no_gil(token_logprobs));
    m.def("token_logprobs_forward", wrap_pybind_function_no_gil(token_logprobs_forward));
    m.def("token_logprobs_backward", wrap_pybind_function_no_gil(token_logprobs_backward));
    m.def("grad_list", wrap_pybind_function([](const py::object &parameters) { return grad_list(parameters); }));
    m.def("clip_grad_norm", wrap_pybind_function(clip_grad_norm));
    m.def("clip_parameters", wrap_pybind_function(clip_parameters));
}
