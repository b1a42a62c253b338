// block_autograd.cpp -- the operators of an attention block as autograd nodes over the C ABI (host code only).
//
// Nodes in C++, not Python: autograd runs a backward on a thread of its own, and a Python node pays there for the
// interpreter's lock and its cold state: a training step of a small layer norm takes 144 us with Python nodes, most of it
// behind the kernels (a trivial torch operation, forward and backward: 43 us).  Argument checks, allocations and launches
// of one call are one trip through the binding; the documentation is in block_ops.py.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include "../../include/tsdiff_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using Opt = std::optional<Tensor>;

struct Failure : std::runtime_error {  // tsdiff_amd._lib.TsdError
    using std::runtime_error::runtime_error;
};
struct Unsupported : std::runtime_error {  // NotImplementedError
    using std::runtime_error::runtime_error;
};

template <class... A> [[noreturn]] void refuse(const A&... a) { throw py::value_error(c10::str(a...)); }

void check(int rc) {
    if (rc == TSD_OK) return;
    const char* msg = tsd_last_error();
    if (rc == TSD_ERR_INVALID) throw py::value_error(msg);
    if (rc == TSD_ERR_UNSUPPORTED) throw Unsupported(msg);
    throw Failure(msg);
}

int dtype_of(at::ScalarType t) {
    return t == at::kFloat ? TSD_F32 : t == at::kBFloat16 ? TSD_BF16 : t == at::kHalf ? TSD_F16 : -1;
}
// type and device of a call's tensors
void same(const char* name, const Tensor& x, std::initializer_list<const Tensor*> others) {
    if (!x.is_cuda()) throw Failure("tsdiff_amd runs on the GPU only (no CPU fallback)");
    if (dtype_of(x.scalar_type()) < 0) refuse(name, ": float32, bfloat16 or float16 expected, got ", x.scalar_type());
    for (const Tensor* t : others)
        if (t->defined() && (t->scalar_type() != x.scalar_type() || t->device() != x.device()))
            refuse(name, ": ", t->scalar_type(), " on ", t->device(), " beside ", x.scalar_type(), " on ", x.device());
}
void* stream_of(const Tensor& x) { return c10::hip::getCurrentHIPStream(x.get_device()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor dense(const Opt& t) { return t.has_value() && t->defined() ? t->contiguous() : Tensor(); }
// t as [rows, features] with contiguous features, copied only where its strides ask for it
Tensor rows_of(const Tensor& x) {
    const Tensor t = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    return (t.size(0) > 1 && t.stride(0) < t.size(1)) || (t.size(1) > 1 && t.stride(1) != 1) ? t.contiguous() : t;
}
int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
int32_t count(const char* name, int64_t n) {
    if (n > 0x7fffffff) throw Unsupported(c10::str(name, ": size ", n, " does not fit 32 bits"));
    return (int32_t)n;
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}
// A tangent (forward-mode differentiation, which works under no_grad too) would be lost where raw pointers are handed on, and
// a lost tangent counts as zero
void no_tangents(const char* name, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t->defined() && t->_fw_grad(/*level=*/0).defined()) throw Unsupported(c10::str(name, " has no forward-mode derivative"));
}
// A missing argument is no edge of the graph: the edge of argument `k` is the number of tensors in front of it
Opt maybe(const Tensor& t) { return t.defined() ? Opt(t) : std::nullopt; }
Tensor given(const Opt& t) { return t.has_value() ? *t : Tensor(); }
bool needs(AutogradContext* ctx, const variable_list& args, size_t k) {
    if (!args[k].defined()) return false;
    size_t edge = 0;
    for (size_t i = 0; i < k; ++i) edge += args[i].defined();
    return ctx->needs_input_grad(edge);
}
// Gradients as they leave a node: what is differentiated once more (create_graph) raises there
variable_list once(const char* name, variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list some;
    for (Tensor& g : grads)
        if (g.defined()) some.push_back(g.detach().requires_grad_());
    auto node = std::make_shared<torch::autograd::DelayedError>(c10::str(name, " has first derivatives only"), (int)some.size());
    variable_list out = (*node)(std::move(some));
    size_t k = 0;
    for (Tensor& g : grads)
        if (g.defined()) g = out[k++];
    return grads;
}

// ---- layer norm -----------------------------------------------------------------------------------------------
Tensor norm_fwd(const Tensor& x, const Tensor& w, const Tensor& b, double eps, Tensor* stats) {
    c10::DeviceGuard guard(x.device());
    const int32_t rows = count("layer_norm", x.size(0)), dim = count("layer_norm", x.size(1));
    Tensor y = at::empty({rows, dim}, x.options());
    float* mean = nullptr;
    if (stats != nullptr) {
        *stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
        mean = stats->data_ptr<float>();
    }
    check(tsd_layer_norm_fwd(dtype_of(x.scalar_type()), rows, dim, ptr(x), ld(x), ptr(w), ptr(b), (float)eps, ptr(y), mean,
                             mean != nullptr ? mean + rows : nullptr, stream_of(x)));
    return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Opt& w, const Opt& b, double eps) {
        Tensor stats, y = norm_fwd(x, given(w), given(b), eps, &stats);
        ctx->save_for_backward({x, given(w), given(b), stats});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &stats = saved[3];
        if (!grads[0].defined()) return variable_list(4);
        no_tangents("layer_norm", {&grads[0]});
        c10::DeviceGuard guard(x.device());
        const Tensor dy = rows_of(grads[0].detach());
        const int32_t rows = (int32_t)x.size(0), dim = (int32_t)x.size(1);
        const bool nw = needs(ctx, saved, 1), nb = needs(ctx, saved, 2);
        Tensor dx, dw, db, scratch;
        if (needs(ctx, saved, 0)) dx = at::empty({rows, dim}, x.options());
        if (nw) dw = at::empty({dim}, x.options());
        if (nb) db = at::empty({dim}, x.options());
        const size_t n = nw || nb ? tsd_layer_norm_scratch_floats(rows, dim) : 0;
        if (n > 0) scratch = at::empty({(int64_t)n}, stats.options());
        const float* mean = stats.data_ptr<float>();
        check(tsd_layer_norm_bwd(dtype_of(x.scalar_type()), rows, dim, ptr(x), ld(x), ptr(w), ptr(dy), ld(dy), mean, mean + rows,
                                 ptr(dx), ptr(dw), ptr(db), (float*)ptr(scratch), n, stream_of(x)));
        return once("layer_norm", {dx, dw, db, Tensor()});
    }
};

Tensor layer_norm(const Tensor& x, const Opt& weight, const Opt& bias, double eps) {
    const Tensor w0 = given(weight), b0 = given(bias);
    no_tangents("layer_norm", {&x, &w0, &b0});
    if (x.dim() < 1 || x.size(-1) < 1) refuse("layer_norm: x has shape ", x.sizes());
    const Tensor w = dense(weight), b = dense(bias);
    for (const Tensor* t : {&w, &b})
        if (t->defined() && (t->dim() != 1 || t->size(0) != x.size(-1)))
            refuse("layer_norm: weight or bias has shape ", t->sizes(), ", [", x.size(-1), "] expected");
    same("layer_norm", x, {&w, &b});
    const Tensor r = rows_of(x), y = wants_grad({&r, &w, &b}) ? LayerNorm::apply(r, maybe(w), maybe(b), eps) : norm_fwd(r, w, b, eps, nullptr);
    return x.dim() == 2 ? y : y.view(x.sizes());
}

// ---- gated linear layer ---------------------------------------------------------------------------------------
Tensor gated_fwd(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& bg, const Tensor& bu, int64_t act) {
    c10::DeviceGuard guard(x.device());
    const int32_t rows = count("gated_linear", x.size(0)), in = count("gated_linear", x.size(1)),
                  out = count("gated_linear", wg.size(0));
    const int dtype = dtype_of(x.scalar_type());
    Tensor h = at::empty({rows, out}, x.options()), scratch;
    const size_t n = tsd_gated_linear_scratch_floats(dtype, rows, in, out, ptr(x), ld(x), ptr(wg), ptr(wu), 0);
    if (n > 0) scratch = at::empty({(int64_t)n}, x.options().dtype(at::kFloat));
    check(tsd_gated_linear_fwd(dtype, (int32_t)act, rows, in, out, ptr(x), ld(x), ptr(wg), ptr(wu), ptr(bg), ptr(bu), ptr(h),
                               (float*)ptr(scratch), n, stream_of(x)));
    return h;
}

struct GatedLinear : torch::autograd::Function<GatedLinear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu, const Opt& bg, const Opt& bu,
                          int64_t act) {
        Tensor h = gated_fwd(x, wg, wu, given(bg), given(bu), act);
        ctx->save_for_backward({x, wg, wu, given(bg), given(bu)});
        ctx->saved_data["act"] = act;
        return h;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &x = s[0], &wg = s[1], &wu = s[2], &bg = s[3], &bu = s[4];
        if (!grads[0].defined()) return variable_list(6);
        no_tangents("gated_linear", {&grads[0]});
        c10::DeviceGuard guard(x.device());
        const Tensor dh = rows_of(grads[0].detach());
        const int dtype = dtype_of(x.scalar_type());
        const int32_t rows = (int32_t)x.size(0), in = (int32_t)x.size(1), out = (int32_t)wg.size(0);
        variable_list g(6);
        const Tensor* like[5] = {&x, &wg, &wu, &bg, &bu};
        for (int k = 0; k < 5; ++k)
            if (needs(ctx, s, k)) g[k] = at::empty(like[k]->sizes(), x.options());
        const size_t n = tsd_gated_linear_scratch_floats(dtype, rows, in, out, ptr(x), ld(x), ptr(wg), ptr(wu), 1);
        Tensor scratch;
        if (n > 0) scratch = at::empty({(int64_t)n}, x.options().dtype(at::kFloat));
        check(tsd_gated_linear_bwd(dtype, (int32_t)ctx->saved_data["act"].toInt(), rows, in, out, ptr(x), ld(x), ptr(wg), ptr(wu),
                                   ptr(bg), ptr(bu), ptr(dh), ld(dh), ptr(g[0]), ptr(g[1]), ptr(g[2]), ptr(g[3]), ptr(g[4]),
                                   (float*)ptr(scratch), n, stream_of(x)));
        return once("gated_linear", std::move(g));
    }
};

Tensor gated_linear(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Opt& b_gate, const Opt& b_up,
                    const std::string& act) {
    const Tensor bg0 = given(b_gate), bu0 = given(b_up);
    no_tangents("gated_linear", {&x, &w_gate, &w_up, &bg0, &bu0});
    const int64_t kind = act == "swish" ? 0 : act == "ssp" ? 1 : act == "ReLU" ? 2 : act == "Softplus" ? 3 : -1;  // tsd_act_fwd's
    if (kind < 0) throw Unsupported("gated_linear: activation '" + act + "'");
    if (w_gate.dim() != 2 || w_gate.sizes() != w_up.sizes() || w_gate.numel() == 0 || x.dim() < 1 || x.size(-1) != w_gate.size(1))
        refuse("gated_linear: x ", x.sizes(), ", w_gate ", w_gate.sizes(), ", w_up ", w_up.sizes());
    const Tensor bg = dense(b_gate), bu = dense(b_up);
    for (const Tensor* t : {&bg, &bu})
        if (t->defined() && (t->dim() != 1 || t->size(0) != w_gate.size(0)))
            refuse("gated_linear: a bias has shape ", t->sizes(), ", [", w_gate.size(0), "] expected");
    same("gated_linear", x, {&w_gate, &w_up, &bg, &bu});
    const Tensor r = rows_of(x), wg = w_gate.contiguous(), wu = w_up.contiguous();
    const Tensor h = wants_grad({&r, &wg, &wu, &bg, &bu}) ? GatedLinear::apply(r, wg, wu, maybe(bg), maybe(bu), kind)
                                                          : gated_fwd(r, wg, wu, bg, bu, kind);
    if (x.dim() == 2) return h;
    std::vector<int64_t> shape = x.sizes().vec();
    shape.back() = w_gate.size(0);
    return h.view(shape);
}

// ---- attention ------------------------------------------------------------------------------------------------
Tensor heads_of(const Tensor& t) { return t.size(2) == 1 || t.stride(2) == 1 ? t : t.contiguous(); }

tsd_attention attention_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& q_ptr, const Tensor& k_ptr,
                             const Tensor& mask, double scale) {
    const char* name = "graph_attention";
    tsd_attention a = {};
    a.dtype = dtype_of(q.scalar_type());
    a.num_graphs = count(name, q_ptr.size(0) - 1);
    a.num_queries = count(name, q.size(0));
    a.num_keys = count(name, k.size(0));
    a.heads = count(name, q.size(1));
    a.kv_heads = count(name, k.size(1));
    a.dim = count(name, q.size(2));
    a.scale = (float)scale;
    a.q = ptr(q);
    a.k = ptr(k);
    a.v = ptr(v);
    a.q_row = q.stride(0);
    a.q_head = q.stride(1);
    a.k_row = k.stride(0);
    a.k_head = k.stride(1);
    a.v_row = v.stride(0);
    a.v_head = v.stride(1);
    a.q_ptr = q_ptr.data_ptr<int32_t>();
    a.k_ptr = k_ptr.data_ptr<int32_t>();
    a.key_mask = (const uint8_t*)ptr(mask);
    return a;
}
Tensor attention_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& q_ptr, const Tensor& k_ptr,
                     const Tensor& mask, double scale, Tensor* rest, Tensor* lse) {
    c10::DeviceGuard guard(q.device());
    const tsd_attention a = attention_args(q, k, v, q_ptr, k_ptr, mask, scale);
    Tensor out = at::empty(q.sizes(), q.options()), scratch;
    if (lse != nullptr) *lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
    if (rest != nullptr && q.scalar_type() != at::kFloat) *rest = at::empty(q.sizes(), q.options());
    const size_t n = tsd_graph_attention_scratch_floats(&a, 0);
    if (n > 0) scratch = at::empty({(int64_t)n}, q.options().dtype(at::kFloat));
    check(tsd_graph_attention_fwd(&a, ptr(out), rest != nullptr ? ptr(*rest) : nullptr, lse != nullptr ? (float*)ptr(*lse) : nullptr,
                                  (float*)ptr(scratch), n, stream_of(q)));
    return out;
}

struct GraphAttention : torch::autograd::Function<GraphAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& q_ptr,
                          const Tensor& k_ptr, const Opt& mask, double scale) {
        Tensor lse, rest, out = attention_fwd(q, k, v, q_ptr, k_ptr, given(mask), scale, &rest, &lse);
        ctx->save_for_backward({q, k, v, q_ptr, k_ptr, given(mask), out, lse, rest});
        ctx->saved_data["scale"] = scale;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        const Tensor &q = s[0], &k = s[1], &v = s[2], &out = s[6], &lse = s[7];
        if (!grads[0].defined()) return variable_list(7);
        no_tangents("graph_attention", {&grads[0]});
        c10::DeviceGuard guard(q.device());
        const Tensor dout = heads_of(grads[0].detach());
        const tsd_attention a = attention_args(q, k, v, s[3], s[4], s[5], ctx->saved_data["scale"].toDouble());
        Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), q.options()), dv = at::empty(v.sizes(), q.options());
        const size_t n = tsd_graph_attention_scratch_floats(&a, 1);
        Tensor scratch;
        if (n > 0) scratch = at::empty({(int64_t)n}, lse.options());
        check(tsd_graph_attention_bwd(&a, ptr(out), ptr(s[8]), (const float*)ptr(lse), ptr(dout), dout.stride(0), dout.stride(1), ptr(dq),
                                      ptr(dk), ptr(dv), (float*)ptr(scratch), n, stream_of(q)));
        return once("graph_attention", {dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor()});
    }
};

Tensor graph_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& graph_ptr, const Opt& key_ptr,
                       const Opt& key_mask, std::optional<double> scale) {
    const char* name = "graph_attention";
    no_tangents(name, {&q, &k, &v});
    for (const Tensor* t : {&q, &k, &v})
        if (t->dim() != 3) refuse(name, ": shape ", t->sizes(), ", [nodes, heads, dim] expected");
    if (k.sizes() != v.sizes() || q.size(2) != k.size(2) || q.size(1) < 1 || q.size(2) < 1 || k.size(1) < 1 ||
        q.size(1) % k.size(1) != 0)
        refuse(name, ": q ", q.sizes(), ", k ", k.sizes(), ", v ", v.sizes());
    same(name, q, {&k, &v});
    if (!key_ptr.has_value() && k.size(0) != q.size(0))
        refuse(name, ": ", q.size(0), " queries and ", k.size(0), " keys need a key_ptr");
    const Tensor kp = key_ptr.has_value() ? *key_ptr : graph_ptr;
    for (const Tensor* t : {&graph_ptr, &kp})
        if (t->dim() != 1 || t->size(0) < 1 || (t->scalar_type() != at::kInt && t->scalar_type() != at::kLong) ||
            t->device() != q.device())
            refuse(name, ": offsets are ", t->scalar_type(), " ", t->sizes(), " on ", t->device(), ", integers [graphs + 1] on ",
                   q.device(), " expected");
    if (graph_ptr.size(0) != kp.size(0))
        refuse(name, ": ", graph_ptr.size(0) - 1, " graphs of queries, ", kp.size(0) - 1, " of keys");
    Tensor mask;
    if (key_mask.has_value()) {
        if (key_mask->dim() != 1 || key_mask->size(0) != k.size(0) || key_mask->device() != q.device() ||
            (key_mask->scalar_type() != at::kBool && key_mask->scalar_type() != at::kByte))
            refuse(name, ": key_mask is ", key_mask->scalar_type(), " ", key_mask->sizes(), " on ", key_mask->device(), ", bool [",
                   k.size(0), "] on ", q.device(), " expected");
        mask = key_mask->contiguous();
    }
    c10::DeviceGuard guard(q.device());
    const Tensor qp = graph_ptr.to(at::kInt).contiguous(), kpi = key_ptr.has_value() ? kp.to(at::kInt).contiguous() : qp;
    const double s = scale.has_value() ? *scale : 1.0 / std::sqrt((double)q.size(2));
    const Tensor qh = heads_of(q), kh = heads_of(k), vh = heads_of(v);
    return wants_grad({&qh, &kh, &vh}) ? GraphAttention::apply(qh, kh, vh, qp, kpi, maybe(mask), s)
                                       : attention_fwd(qh, kh, vh, qp, kpi, mask, s, nullptr, nullptr);
}

}  // namespace

PYBIND11_MODULE(_block_ops, m) {
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const Failure& e) {
            PyErr_SetString(py::module_::import("tsdiff_amd._lib").attr("TsdError").ptr(), e.what());
        } catch (const Unsupported& e) {
            PyErr_SetString(PyExc_NotImplementedError, e.what());
        }
    });
    using release = py::call_guard<py::gil_scoped_release>;
    m.def("layer_norm", &layer_norm, release());
    m.def("gated_linear", &gated_linear, release());
    m.def("graph_attention", &graph_attention, release());
}
