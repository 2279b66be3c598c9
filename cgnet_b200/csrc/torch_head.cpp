// PyTorch side of the operators behind the invariant embedding (cgnet_b200/head.py): argument checks, output and workspace
// allocation, and the autograd nodes, around the C entry points of include/cgnet_b200.h.  In C++ because a training step of a
// small head is bound by this host code: with the nodes in Python a forward and backward took 105 us of host time, of which the
// kernels needed 10.
//
// Module functions (positional arguments, None where a tensor is optional):
//     layer_norm(x, weight, bias, eps)
//     gated_feed_forward(x, w_gate, w_up, activation)        activation: "silu", "gelu", "relu"
//     log_probs(logits, targets, top) -> (log_prob, entropy, top_log_probs, top_ids)
//     distillation_loss(logits, teacher_ids, teacher_scores, temperature)
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cmath>
#include <stdexcept>
#include <string>

#include "../../include/cgnet_b200.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

[[noreturn]] void fail(const std::string& msg) { throw std::runtime_error(msg); }

// ---- checks (before any pointer reaches the library) --------------------------------------------------------------------
int type_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return CGB200_F32;
        case at::kBFloat16: return CGB200_BF16;
        case at::kHalf: return CGB200_F16;
        default: return -1;
    }
}
std::string type_name(const Tensor& t) {
    const int c = type_code(t);
    return c == CGB200_F32 ? "torch.float32" : c == CGB200_BF16 ? "torch.bfloat16" : c == CGB200_F16 ? "torch.float16" : c10::toString(t.scalar_type());
}
std::string shape_of(at::IntArrayRef s) {
    std::string o = "(";
    for (size_t i = 0; i < s.size(); ++i) o += (i ? ", " : "") + std::to_string(s[i]);
    return o + (s.size() == 1 ? ",)" : ")");
}
const Tensor& tensor_of(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) fail(std::string(name) + " must be a tensor, got " + Py_TYPE(o)->tp_name);
    return THPVariable_Unpack(o);
}
void check_device(const Tensor& t, const char* name, const Tensor& like) {
    if (t.device() != like.device()) fail(std::string(name) + " lives on " + t.device().str() + ", expected " + like.device().str());
}
const Tensor& values_of(PyObject* o, const char* name, const Tensor* like = nullptr) {
    const Tensor& t = tensor_of(o, name);
    if (type_code(t) < 0) fail(std::string(name) + " must be float32, bfloat16 or float16, got " + type_name(t));
    if (like != nullptr) check_device(t, name, *like);
    // a trace would hold the allocation of the results and not the kernel that writes them
    if (torch::jit::tracer::isTracing()) fail("the operators of cgnet_b200.head cannot be recorded by torch.jit.trace");
    if (t._fw_grad(0).defined()) fail(std::string(name) + " has a forward-mode derivative, which the operators of cgnet_b200.head do not pass on");
    return t;
}
void check_shape(const Tensor& t, const char* name, at::IntArrayRef want) {
    if (t.sizes() != want) fail(std::string(name) + " has shape " + shape_of(t.sizes()) + ", expected " + shape_of(want));
}
void check_rows(const Tensor& t, const char* name) {
    if (t.dim() == 0 || t.size(-1) == 0)
        fail(std::string(name) + " must have at least one value in its last dimension, got shape " + shape_of(t.sizes()));
}
void check_cuda(const Tensor& t, const char* name) {
    if (!t.is_cuda()) fail(std::string(name) + " must be a CUDA tensor (cgnet_b200 has no CPU path)");
}
// int64 (or int32) class indices; their values are the kernels' business
Tensor classes_of(PyObject* o, const char* name, at::IntArrayRef want, const Tensor& like) {
    if (!THPVariable_Check(o) || (THPVariable_Unpack(o).scalar_type() != at::kLong && THPVariable_Unpack(o).scalar_type() != at::kInt))
        fail(std::string(name) + " must be an int64 or int32 tensor");
    const Tensor& t = THPVariable_Unpack(o);
    check_device(t, name, like);
    check_shape(t, name, want);
    return t.to(at::kLong).resolve_neg().contiguous();
}
// (rows, columns) whose columns are neighbours in memory; rows may be any distance apart
// (a lazily negated view, such as the imaginary part of a conjugate, is negated first)
Tensor rows_of(const Tensor& given) {
    const Tensor t = given.is_neg() ? given.resolve_neg() : given;
    const Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
    return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}
void once() {
    // autograd enables gradients in a backward only where its result is to be differentiated again
    if (at::GradMode::is_enabled()) fail("the operators of cgnet_b200.head are differentiable once only");
}

// ---- calls ---------------------------------------------------------------------------------------------------------------
void check(int rc, const char* what) {
    if (rc != CGB200_OK) {
        const char* msg = cgb200_last_error();
        fail(std::string(what) + " failed with status " + std::to_string(rc) + ": " + (msg != nullptr ? msg : "?"));
    }
}
// The tensor's device made current, and torch's current stream on it
struct Launch {
    c10::cuda::CUDAGuard guard;
    void* stream;
    explicit Launch(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const optional<Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }
float* fptr(const Tensor& t) { return t.defined() ? (float*)t.data_ptr() : nullptr; }
Tensor empty(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options().requires_grad(false)); }
Tensor empty_as(at::IntArrayRef shape, const Tensor& like, at::ScalarType type) { return at::empty(shape, like.options().dtype(type).requires_grad(false)); }
// Scratch of one call, from torch's allocator, which keeps it apart from other streams' and graphs' calls
Tensor workspace(int64_t bytes, const Tensor& like) {
    if (bytes < 0) check(CGB200_ERR_ARGUMENT, "workspace size");
    return bytes > 0 ? empty_as({bytes}, like, at::kByte) : Tensor();
}

// ---- layer norm ------------------------------------------------------------------------------------------------------------
std::pair<Tensor, Tensor> norm_fwd(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps, bool keep) {
    const int64_t rows = x.size(0), dim = x.size(1);
    Tensor y = empty({rows, dim}, x), stats;
    if (keep) stats = empty_as({rows, 2}, x, at::kFloat);
    const int type = type_code(x), param = w.has_value() ? type_code(*w) : b.has_value() ? type_code(*b) : type;
    const Launch l(x);
    check(cgb200_layer_norm_fwd(x.data_ptr(), x.stride(0), ptr(w), ptr(b), (float)eps, y.data_ptr(), fptr(stats), rows, dim, type, param, l.stream),
          "cgb200_layer_norm_fwd");
    return {y, stats};
}
struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps) {
        auto [y, stats] = norm_fwd(x, w, b, eps, true);
        ctx->save_for_backward({x, w.has_value() ? *w : Tensor(), stats});
        ctx->saved_data["w"] = w.has_value();
        ctx->saved_data["b"] = b.has_value();
        ctx->saved_data["param"] = (int64_t)(w.has_value() ? w->scalar_type() : b.has_value() ? b->scalar_type() : x.scalar_type());
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once();
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
        const bool has_w = ctx->saved_data["w"].toBool(), has_b = ctx->saved_data["b"].toBool();
        const auto param = (at::ScalarType)ctx->saved_data["param"].toInt();
        const int64_t rows = x.size(0), dim = x.size(1);
        const Tensor dy = rows_of(grads[0]);
        const bool need_x = ctx->needs_input_grad(0), need_w = has_w && ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(1 + has_w);
        Tensor dx, dw, db;
        if (need_x) dx = empty({rows, dim}, x);
        if (need_w) dw = empty_as({dim}, x, param);
        if (need_b) db = empty_as({dim}, x, param);
        const int type = type_code(x), ptype = param == x.scalar_type() ? type : CGB200_F32;
        const int64_t n = need_w || need_b ? cgb200_layer_norm_bwd_workspace_bytes(rows, dim, type) : 0;
        const Tensor ws = workspace(n, x);
        const Launch l(x);
        check(cgb200_layer_norm_bwd(x.data_ptr(), x.stride(0), dy.data_ptr(), dy.stride(0), ptr(w), fptr(stats), ptr(dx), ptr(dw), ptr(db), rows, dim, type,
                                    ptype, ptr(ws), n, l.stream),
              "cgb200_layer_norm_bwd");
        return {dx, dw, db, Tensor()};
    }
};
Tensor layer_norm(PyObject* const* a) {
    const Tensor& x = values_of(a[0], "x");
    const double eps = PyFloat_AsDouble(a[3]);
    if (eps == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        fail("eps must be a number");
    }
    if (!(eps >= 0.0 && std::isfinite(eps))) fail("eps must be finite and not negative, got " + std::to_string(eps));
    check_rows(x, "x");
    optional<Tensor> p[2];
    const char* names[2] = {"weight", "bias"};
    for (int i = 0; i < 2; ++i) {
        if (a[1 + i] == Py_None) continue;
        const Tensor& t = values_of(a[1 + i], names[i], &x);
        check_shape(t, names[i], {x.size(-1)});
        if (t.scalar_type() != x.scalar_type() && t.scalar_type() != at::kFloat)
            fail(std::string(names[i]) + " must be " + type_name(x) + " or float32, got " + type_name(t));
        p[i] = t.resolve_neg().contiguous();
    }
    if (p[0].has_value() && p[1].has_value() && p[0]->scalar_type() != p[1]->scalar_type())
        fail("weight and bias must have one type, got " + type_name(*p[0]) + " and " + type_name(*p[1]));
    check_cuda(x, "x");
    const Tensor x2 = rows_of(x);
    const bool grad = at::GradMode::is_enabled() &&
                      (x.requires_grad() || (p[0].has_value() && p[0]->requires_grad()) || (p[1].has_value() && p[1]->requires_grad()));
    const Tensor y = grad ? LayerNorm::apply(x2, p[0], p[1], eps) : norm_fwd(x2, p[0], p[1], eps, false).first;
    return x.dim() == 2 ? y : y.view(x.sizes());
}

// ---- gated feed-forward block ------------------------------------------------------------------------------------------------
std::pair<Tensor, Tensor> ff_fwd(const Tensor& x, const Tensor& wg, const Tensor& wu, int64_t act, bool keep) {
    const int64_t rows = x.size(0), dim = x.size(1), hidden = wg.size(0);
    Tensor h = empty({rows, hidden}, x), gate_up;
    if (keep) gate_up = empty_as({2, rows, (hidden + 3) / 4 * 4}, x, at::kFloat);
    const int type = type_code(x);
    const int64_t n = cgb200_gated_ff_workspace_bytes(x.data_ptr(), x.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0), rows, dim,
                                                      hidden, type, 0);
    const Tensor ws = workspace(n, x);
    const Launch l(x);
    check(cgb200_gated_ff_fwd(x.data_ptr(), x.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0), (int)act, h.data_ptr(),
                              fptr(gate_up), rows, dim, hidden, type, ptr(ws), n, l.stream),
          "cgb200_gated_ff_fwd");
    return {h, gate_up};
}
struct GatedFeedForward : torch::autograd::Function<GatedFeedForward> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, int64_t act) {
        auto [h, gate_up] = ff_fwd(x, wg, wu, act, true);
        ctx->save_for_backward({x, wg, wu, gate_up});
        ctx->saved_data["act"] = act;
        return h;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once();
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &wg = saved[1], &wu = saved[2], &gate_up = saved[3];
        const int64_t rows = x.size(0), dim = x.size(1), hidden = wg.size(0);
        const Tensor dh = rows_of(grads[0]);
        Tensor dx, dwg, dwu;
        if (ctx->needs_input_grad(0)) dx = empty({rows, dim}, x);
        if (ctx->needs_input_grad(1)) dwg = empty({hidden, dim}, x);
        if (ctx->needs_input_grad(2)) dwu = empty({hidden, dim}, x);
        const int type = type_code(x);
        const int64_t n = cgb200_gated_ff_workspace_bytes(x.data_ptr(), x.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0), rows, dim,
                                                          hidden, type, (dx.defined() ? 1 : 0) + (dwg.defined() ? 2 : 0) + (dwu.defined() ? 4 : 0));
        const Tensor ws = workspace(n, x);
        const Launch l(x);
        check(cgb200_gated_ff_bwd(x.data_ptr(), x.stride(0), wg.data_ptr(), wg.stride(0), wu.data_ptr(), wu.stride(0),
                                  (int)ctx->saved_data["act"].toInt(), fptr(gate_up), dh.data_ptr(), dh.stride(0), ptr(dx), ptr(dwg), ptr(dwu), rows, dim,
                                  hidden, type, ptr(ws), n, l.stream),
              "cgb200_gated_ff_bwd");
        return {dx, dwg, dwu, Tensor()};
    }
};
int activation_of(PyObject* o) {
    const char* s = PyUnicode_Check(o) ? PyUnicode_AsUTF8(o) : nullptr;
    if (s != nullptr) {
        if (std::string(s) == "silu") return CGB200_ACT_SILU;
        if (std::string(s) == "gelu") return CGB200_ACT_GELU;
        if (std::string(s) == "relu") return CGB200_ACT_RELU;
    }
    PyErr_Clear();
    fail(std::string("activation must be one of gelu, relu, silu, got ") + (s != nullptr ? s : Py_TYPE(o)->tp_name));
}
Tensor gated_feed_forward(PyObject* const* a) {
    const int act = activation_of(a[3]);
    const Tensor& x = values_of(a[0], "x");
    check_rows(x, "x");
    const Tensor* w[2];
    const char* names[2] = {"w_gate", "w_up"};
    for (int i = 0; i < 2; ++i) {
        w[i] = &values_of(a[1 + i], names[i], &x);
        if (w[i]->scalar_type() != x.scalar_type()) fail(std::string(names[i]) + " must be " + type_name(x) + ", got " + type_name(*w[i]));
        if (w[i]->dim() != 2 || w[i]->size(1) != x.size(-1) || w[i]->size(0) == 0)
            fail(std::string(names[i]) + " has shape " + shape_of(w[i]->sizes()) + ", expected (hidden, " + std::to_string(x.size(-1)) + ")");
    }
    check_shape(*w[1], "w_up", w[0]->sizes());
    check_cuda(x, "x");
    const Tensor x2 = rows_of(x), wg = rows_of(*w[0]), wu = rows_of(*w[1]);
    const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || w[0]->requires_grad() || w[1]->requires_grad());
    const Tensor h = grad ? GatedFeedForward::apply(x2, wg, wu, (int64_t)act) : ff_fwd(x2, wg, wu, act, false).first;
    if (x.dim() == 2) return h;
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end() - 1);
    shape.push_back(h.size(1));
    return h.view(shape);
}

// ---- log probabilities -------------------------------------------------------------------------------------------------------
variable_list logp_fwd(const Tensor& z, const optional<Tensor>& targets, int64_t top, Tensor* stats) {
    const int64_t rows = z.size(0), classes = z.size(1);
    const Tensor lp = empty_as({rows}, z, at::kFloat), ent = empty_as({rows}, z, at::kFloat), top_lp = empty_as({rows, top}, z, at::kFloat),
                 top_ids = empty_as({rows, top}, z, at::kLong);
    if (stats != nullptr) *stats = empty_as({rows, 2}, z, at::kFloat);
    const Launch l(z);
    check(cgb200_log_probs_fwd(z.data_ptr(), z.stride(0), (const int64_t*)ptr(targets), (int)top, fptr(lp), fptr(ent), fptr(top_lp),
                               (int64_t*)top_ids.data_ptr(), stats != nullptr ? fptr(*stats) : nullptr, rows, classes, type_code(z), l.stream),
          "cgb200_log_probs_fwd");
    return {lp, ent, top_lp, top_ids};
}
struct LogProbs : torch::autograd::Function<LogProbs> {
    static variable_list forward(AutogradContext* ctx, const Tensor& z, const optional<Tensor>& targets, int64_t top) {
        Tensor stats;
        const variable_list out = logp_fwd(z, targets, top, &stats);
        ctx->save_for_backward({z, targets.has_value() ? *targets : Tensor(), out[1], stats});
        ctx->mark_non_differentiable({out[2], out[3]});
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once();
        const auto saved = ctx->get_saved_variables();
        const Tensor &z = saved[0], &targets = saved[1], &ent = saved[2], &stats = saved[3];
        const Tensor g_lp = targets.defined() && grads[0].defined() ? grads[0].resolve_neg().contiguous() : Tensor();
        const Tensor g_ent = grads[1].defined() ? grads[1].resolve_neg().contiguous() : Tensor();
        if (!ctx->needs_input_grad(0) || (!g_lp.defined() && !g_ent.defined())) return {Tensor(), Tensor(), Tensor()};
        const int64_t rows = z.size(0), classes = z.size(1);
        const Tensor dz = empty({rows, classes}, z);
        const Launch l(z);
        check(cgb200_log_probs_bwd(z.data_ptr(), z.stride(0), (const int64_t*)ptr(targets), fptr(ent), fptr(stats), fptr(g_lp), fptr(g_ent), dz.data_ptr(),
                                   rows, classes, type_code(z), l.stream),
              "cgb200_log_probs_bwd");
        return {dz, Tensor(), Tensor()};
    }
};
PyObject* log_probs(PyObject* const* a) {
    const Tensor& z = values_of(a[0], "logits");
    check_rows(z, "logits");
    const at::IntArrayRef lead = z.sizes().slice(0, z.dim() - 1);
    const int64_t most = std::min<int64_t>(128, z.size(-1));
    const long top = PyLong_Check(a[2]) && !PyBool_Check(a[2]) ? PyLong_AsLong(a[2]) : -1;
    if (top < 0 || top > most) {
        PyErr_Clear();
        fail("top must be an integer from 0 to " + std::to_string(most));
    }
    optional<Tensor> targets;
    if (a[1] != Py_None) {
        targets = classes_of(a[1], "targets", lead, z);
        if (targets->dim() != 1) targets = targets->reshape({-1});
    }
    check_cuda(z, "logits");
    const Tensor z2 = rows_of(z);
    variable_list out = at::GradMode::is_enabled() && z.requires_grad() ? LogProbs::apply(z2, targets, (int64_t)top) : logp_fwd(z2, targets, top, nullptr);
    if (lead.size() != 1) {
        std::vector<int64_t> wide(lead.begin(), lead.end());
        wide.push_back(top);
        out[0] = out[0].view(lead), out[1] = out[1].view(lead), out[2] = out[2].view(wide), out[3] = out[3].view(wide);
    }
    PyObject* r = PyTuple_New(4);
    for (int i = 0; i < 4; ++i) {
        PyObject* o = i == 0 && !targets.has_value() ? Py_NewRef(Py_None) : THPVariable_Wrap(out[i]);
        PyTuple_SET_ITEM(r, i, o);
    }
    return r;
}

// ---- distillation --------------------------------------------------------------------------------------------------------------
std::pair<Tensor, Tensor> distill_fwd(const Tensor& z, const Tensor& ids, const Tensor& scores, double temperature, bool keep) {
    const int64_t rows = z.size(0), classes = z.size(1);
    Tensor loss = empty_as({rows}, z, at::kFloat), stats;
    if (keep) stats = empty_as({rows, 4}, z, at::kFloat);
    const Launch l(z);
    check(cgb200_distill_fwd(z.data_ptr(), z.stride(0), (const int64_t*)ids.data_ptr(), scores.data_ptr(), (int)ids.size(1), type_code(scores),
                             (float)temperature, fptr(loss), fptr(stats), rows, classes, type_code(z), l.stream),
          "cgb200_distill_fwd");
    return {loss, stats};
}
struct Distill : torch::autograd::Function<Distill> {
    static Tensor forward(AutogradContext* ctx, const Tensor& z, const Tensor& ids, const Tensor& scores, double temperature) {
        auto [loss, stats] = distill_fwd(z, ids, scores, temperature, true);
        ctx->save_for_backward({z, ids, scores, stats});
        ctx->saved_data["temperature"] = temperature;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        once();
        const auto saved = ctx->get_saved_variables();
        const Tensor &z = saved[0], &ids = saved[1], &scores = saved[2], &stats = saved[3];
        const Tensor g = grads[0].resolve_neg().contiguous();
        const int64_t rows = z.size(0), classes = z.size(1);
        const Tensor dz = empty({rows, classes}, z);
        const Launch l(z);
        check(cgb200_distill_bwd(z.data_ptr(), z.stride(0), (const int64_t*)ids.data_ptr(), scores.data_ptr(), (int)ids.size(1), type_code(scores),
                                 (float)ctx->saved_data["temperature"].toDouble(), fptr(stats), fptr(g), dz.data_ptr(), rows, classes, type_code(z),
                                 l.stream),
              "cgb200_distill_bwd");
        return {dz, Tensor(), Tensor(), Tensor()};
    }
};
Tensor distillation_loss(PyObject* const* a) {
    const Tensor& z = values_of(a[0], "logits");
    check_rows(z, "logits");
    const at::IntArrayRef lead = z.sizes().slice(0, z.dim() - 1);
    const Tensor& given = values_of(a[2], "teacher_scores", &z);
    const int64_t k = given.dim() > 0 ? given.size(-1) : 0;
    if (k < 1 || k > CGB200_MAX_TEACHER)
        fail("teacher_scores must name 1 to " + std::to_string(CGB200_MAX_TEACHER) + " classes a row, got shape " + shape_of(given.sizes()));
    std::vector<int64_t> want(lead.begin(), lead.end());
    want.push_back(k);
    check_shape(given, "teacher_scores", want);
    const Tensor ids = classes_of(a[1], "teacher_ids", want, z).reshape({-1, k});
    const double temperature = PyFloat_AsDouble(a[3]);
    if (!(temperature >= 1e-3 && temperature <= 1e3)) {
        PyErr_Clear();
        fail("temperature must be between 0.001 and 1000, got " + std::to_string(temperature));
    }
    check_cuda(z, "logits");
    const Tensor z2 = rows_of(z), scores = given.detach().resolve_neg().reshape({-1, k}).contiguous();
    const Tensor loss = at::GradMode::is_enabled() && z.requires_grad() ? Distill::apply(z2, ids, scores, temperature)
                                                                        : distill_fwd(z2, ids, scores, temperature, false).first;
    return lead.size() == 1 ? loss : loss.view(lead);
}

// ---- module --------------------------------------------------------------------------------------------------------------------
// Errors keep their type: one that Python code raised below this call (saved-tensor hooks, such as the one by which activation
// checkpointing ends its recomputation) goes on as it is, and an allocation that failed is torch.OutOfMemoryError.
template <typename F>
PyObject* guarded(const char* name, Py_ssize_t given, Py_ssize_t want, F f) {
    if (given != want) return PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, want, given);
    HANDLE_TH_ERRORS
    return f();
    END_HANDLE_TH_ERRORS
}
PyObject* py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("layer_norm", n, 4, [&] { return THPVariable_Wrap(layer_norm(a)); });
}
PyObject* py_gated_feed_forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("gated_feed_forward", n, 4, [&] { return THPVariable_Wrap(gated_feed_forward(a)); });
}
PyObject* py_log_probs(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("log_probs", n, 3, [&] { return log_probs(a); });
}
PyObject* py_distillation_loss(PyObject*, PyObject* const* a, Py_ssize_t n) {
    return guarded("distillation_loss", n, 4, [&] { return THPVariable_Wrap(distillation_loss(a)); });
}
PyMethodDef kMethods[] = {{"layer_norm", (PyCFunction)(void (*)())py_layer_norm, METH_FASTCALL, nullptr},
                          {"gated_feed_forward", (PyCFunction)(void (*)())py_gated_feed_forward, METH_FASTCALL, nullptr},
                          {"log_probs", (PyCFunction)(void (*)())py_log_probs, METH_FASTCALL, nullptr},
                          {"distillation_loss", (PyCFunction)(void (*)())py_distillation_loss, METH_FASTCALL, nullptr},
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_head", "Operators behind the invariant embedding, for torch tensors.", -1, kMethods,
                       nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_head(void) { return PyModule_Create(&kModule); }
