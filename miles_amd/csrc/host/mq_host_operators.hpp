// The norms, linear layers and 8-bit activation checkpoints in native code: outputs, workspaces, graph nodes and their backward passes.
// Written in Python a training step of one norm costs some 100 us of host time, several times what its kernels take.  Included by
// mq_host.cpp, whose rules hold: ordinary tensors only (here also one run of memory each, on the current device), None for
// everything else, which goes on in Python, where every argument is checked and every refusal is worded.
#include <c10/hip/HIPFunctions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

namespace {

// ---- what the native form takes ------------------------------------------------------------------------------------------
bool simple(const at::Tensor* t) {
    return t && t->is_contiguous() && t->numel() > 0 && !t->_fw_grad(0).defined() && t->device().index() == c10::hip::current_device();
}
// the tensor of an argument that may be None: false if it is one that goes to Python
bool optional_simple(PyObject* o, const at::Tensor*& t) {
    t = nullptr;
    if (o == Py_None) return true;
    t = ordinary(o);
    return simple(t);
}
bool truth(PyObject* o, bool& v) {
    v = o == Py_True;
    return v || o == Py_False;
}
bool wants_graph(std::initializer_list<const at::Tensor*> inputs) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor* t : inputs)
        if (t && t->requires_grad()) return true;
    return false;
}
at::Tensor maybe(const at::Tensor* t) { return t ? *t : at::Tensor(); }
// an argument of a graph node that may be missing; a missing one has no edge, and those behind it move up
using Input = std::optional<at::Tensor>;
Input input(const at::Tensor* t) { return t ? Input(*t) : Input(); }
at::Tensor maybe(const Input& t) { return t.has_value() ? *t : at::Tensor(); }
void* pointer(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
// what the library refuses, on its way through torch's functions to the caller, who is given a MilesQuantError
struct Refusal : std::runtime_error {
    using std::runtime_error::runtime_error;
};
void checked(int rc) {
    if (rc != MQ_OK) throw Refusal(mq_last_error());
}
template <class F>
PyObject* or_refused(F&& call) {
    try {
        return call();
    } catch (const Refusal& why) {
        PyErr_SetString(g_error ? g_error : PyExc_RuntimeError, why.what());
        return nullptr;
    }
}
// t as one run of memory that begins at a multiple of 16 bytes
at::Tensor one_run(const at::Tensor& t) {
    const at::Tensor c = t.contiguous();
    return (uintptr_t)c.data_ptr() % 16 == 0 ? c : c.clone();
}
// A tensor that was saved, as the kernels read it: hooks on saved tensors may give back anything, and a kernel has no way to see it.
at::Tensor unpacked(const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& like, const char* what) {
    if (!t.defined()) return t;
    TORCH_CHECK(t.sizes() == sizes && t.scalar_type() == dtype && t.device() == like.device() && t.layout() == at::kStrided, what,
                ": a saved tensor came back as ", t.toString(), t.sizes(), " on ", t.device(), ", not of the type, shape and device that it was saved with");
    return t.contiguous();
}
at::Tensor scratch(int64_t bytes, const at::Tensor& like) { return bytes > 0 ? make({bytes}, at::kByte, like) : at::Tensor(); }
// Gradients are taken once: where a graph of the backward pass itself is asked for, those that the node now running has made are part of
// one that refuses to be gone through, and as constants would leave what depends on them out of a second derivative.  Its edges are the
// node's own and those of the incoming gradients, so that every way to an input that a gradient depends on meets the refusal, also where a
// caller names the inputs whose gradients it wants.
void once(torch::autograd::variable_list& made, const torch::autograd::variable_list& incoming, const char* what) {
    const auto node = torch::autograd::get_current_node();
    TORCH_CHECK(node, what, ": no backward pass is running");
    torch::autograd::edge_list edges = node->next_edges();
    for (const at::Tensor& g : incoming)
        if (g.defined() && g.requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(g));
    const auto refuse = std::make_shared<torch::autograd::Error>(std::string(what) + ": gradients of gradients are not supported", std::move(edges));
    for (at::Tensor& g : made) {
        if (!g.defined()) continue;
        g = g.detach();
        torch::autograd::create_gradient_edge(g, refuse);
    }
}
// once(list of gradients, list of incoming gradients, name of the operator) -> list of gradients
PyObject* once_of(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 3 || !PyList_Check(a[0]) || !PyList_Check(a[1]) || !PyUnicode_Check(a[2])) return PyErr_Format(PyExc_TypeError, "once: (list, list, str)");
    torch::autograd::variable_list lists[2];
    for (int which = 0; which < 2; which++)
        for (Py_ssize_t i = 0; i < PyList_GET_SIZE(a[which]); i++) {
            PyObject* t = PyList_GET_ITEM(a[which], i);
            if (!THPVariable_Check(t)) return PyErr_Format(PyExc_TypeError, "once: lists of tensors");
            lists[which].push_back(THPVariable_Unpack(t));
        }
    once(lists[0], lists[1], PyUnicode_AsUTF8(a[2]));
    Owned out = owned(PyList_New((Py_ssize_t)lists[0].size()));
    if (!out) return nullptr;
    for (size_t i = 0; i < lists[0].size(); i++) PyList_SET_ITEM(out.ptr(), (Py_ssize_t)i, THPVariable_Wrap(lists[0][i]));
    return out.release().ptr();
    END_HANDLE_TH_ERRORS
}

// ---- norms -----------------------------------------------------------------------------------------------------------------
struct NormCall {
    double eps;
    bool rms, keep, copy;
    at::Tensor yq, ys;         // the copy of the result
};
struct NormKept {
    at::Tensor xq, xs, mean, rstd;
};
at::Tensor norm_forward(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b, NormCall& call, bool graph, NormKept& kept) {
    const int64_t n = x.size(-1), m = x.numel() / n;
    at::Tensor y = make(x.sizes(), x.scalar_type(), x);
    if (graph) {
        kept.rstd = make({m}, at::kFloat, x);
        if (call.keep) {
            kept.xq = make({m, n}, at::kFloat8_e4m3fn, x);
            kept.xs = make({m, n / 32}, at::kByte, x);
        } else if (!call.rms) {
            kept.mean = make({m}, at::kFloat, x);
        }
    }
    if (call.copy) {
        c10::SmallVector<int64_t, 4> sizes(x.sizes().begin(), x.sizes().end());
        call.yq = make(sizes, at::kFloat8_e4m3fn, x);
        sizes.back() /= 32;
        call.ys = make(sizes, at::kByte, x);
    }
    const at::ScalarType vector = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type();
    checked(mq_norm_forward(x.data_ptr(), dtype_code(x.scalar_type()), n, pointer(w), pointer(b), dtype_code(vector), y.data_ptr(), pointer(kept.xq),
                            (uint8_t*)pointer(kept.xs), pointer(call.yq), (uint8_t*)pointer(call.ys), (float*)pointer(kept.mean),
                            (float*)pointer(kept.rstd), m, n, (float)call.eps, call.rms, stream_of(x)));
    return y;
}
struct Norm : torch::autograd::Function<Norm> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const Input& weight, const Input& bias, NormCall* call) {
        NormKept kept;
        const at::Tensor w = maybe(weight), b = maybe(bias);
        at::Tensor y = norm_forward(x, w, b, *call, true, kept);
        ctx->save_for_backward({call->keep ? kept.xq : x, kept.xs, kept.mean, kept.rstd, w});
        ctx->saved_data["rms"] = call->rms;
        ctx->saved_data["bias"] = b.defined() ? (int64_t)b.scalar_type() : (int64_t)-1;
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const bool again = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        const auto saved = ctx->get_saved_variables();
        const at::Tensor dy = one_run(grads[0]);
        const int64_t bias = ctx->saved_data["bias"].toInt(), n = dy.size(-1), m = dy.numel() / n;
        const bool kept8 = saved[1].defined(), weight = saved[4].defined();
        const at::ScalarType vector = weight ? saved[4].scalar_type() : bias >= 0 ? (at::ScalarType)bias : dy.scalar_type();
        const at::Tensor x = one_run(kept8 ? unpacked(saved[0], {m, n}, at::kFloat8_e4m3fn, dy, "norm") : unpacked(saved[0], dy.sizes(), dy.scalar_type(), dy, "norm"));
        const at::Tensor xs = unpacked(saved[1], {m, n / 32}, at::kByte, dy, "norm"), mean = unpacked(saved[2], {m}, at::kFloat, dy, "norm"),
                         rstd = unpacked(saved[3], {m}, at::kFloat, dy, "norm"), w = unpacked(saved[4], {n}, vector, dy, "norm");
        const bool rms = ctx->saved_data["rms"].toBool(), want_x = ctx->needs_input_grad(0), want_w = weight && ctx->needs_input_grad(1);
        const bool want_b = bias >= 0 && ctx->needs_input_grad(weight ? 2 : 1);
        at::Tensor dx, dw, db;
        if (want_x) dx = make(dy.sizes(), dy.scalar_type(), dy);
        if (want_w) dw = make({n}, vector, dy);
        if (want_b) db = make({n}, vector, dy);
        const at::Tensor ws = scratch((want_w + want_b) * (int64_t)mq_norm_backward_parts(m, n) * n * 4, dy);
        checked(mq_norm_backward(dy.data_ptr(), dtype_code(dy.scalar_type()), n, x.data_ptr(), n, (const uint8_t*)pointer(xs), (const float*)pointer(mean),
                                 (const float*)pointer(rstd), pointer(w), dtype_code(vector), pointer(dx), pointer(dw), pointer(db),
                                 (float*)pointer(ws), m, n, rms, stream_of(dy)));
        torch::autograd::variable_list out{dx, dw, db};
        if (again) once(out, grads, "norm");
        out.resize(4);
        return out;
    }
};
// norm(x, weight | None, bias | None, eps, rms, keep in 8 bits, copy of the result) -> y, (y, codes, scales) or None
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    return or_refused([&]() -> PyObject* {
        if (n != 7) return PyErr_Format(PyExc_TypeError, "norm: 7 arguments");
        const at::Tensor *x = ordinary(a[0]), *w, *b;
        NormCall call;
        if (listing() || !ordinary_moment() || !simple(x) || x->dim() == 0 || dtype_code(x->scalar_type()) < 0 || (uintptr_t)x->data_ptr() % 16) Py_RETURN_NONE;
        if (!optional_simple(a[1], w) || !optional_simple(a[2], b) || !truth(a[4], call.rms) || !truth(a[5], call.keep) || !truth(a[6], call.copy)) Py_RETURN_NONE;
        if (!PyFloat_Check(a[3])) Py_RETURN_NONE;
        call.eps = PyFloat_AS_DOUBLE(a[3]);
        const int64_t columns = x->size(-1);
        if ((call.keep || call.copy) && columns % 32 != 0) Py_RETURN_NONE;
        for (const at::Tensor* v : {w, b})
            if (v && (v->dim() != 1 || v->size(0) != columns || v->device() != x->device() ||
                      (v->scalar_type() != x->scalar_type() && v->scalar_type() != at::kFloat)))
                Py_RETURN_NONE;
        if (w && b && w->scalar_type() != b->scalar_type()) Py_RETURN_NONE;
        at::Tensor y;
        {
            pybind11::gil_scoped_release no_gil;
            if (wants_graph({x, w, b})) {
                y = Norm::apply(*x, input(w), input(b), &call);
            } else {
                at::NoGradGuard no_grad;
                NormKept none;
                y = norm_forward(*x, maybe(w), maybe(b), call, false, none);
            }
        }
        if (!call.copy) return THPVariable_Wrap(std::move(y));
        return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(y)), THPVariable_Wrap(std::move(call.yq)), THPVariable_Wrap(std::move(call.ys)));
    });
    END_HANDLE_TH_ERRORS
}

// ---- 8-bit activation checkpoints --------------------------------------------------------------------------------------------
void keep_into(const at::Tensor& x, at::Tensor& codes, at::Tensor& scales) {
    c10::SmallVector<int64_t, 4> sizes(x.sizes().begin(), x.sizes().end());
    codes = make(sizes, at::kFloat8_e4m3fn, x);
    const int64_t k = sizes.back();
    sizes.back() /= 32;
    scales = make(sizes, at::kByte, x);
    checked(mq_mxfp8_quant(x.data_ptr(), dtype_code(x.scalar_type()), codes.data_ptr(), (uint8_t*)scales.data_ptr(), x.numel() / k, k, stream_of(x)));
}
// keep8(x) -> (codes, scales) or None
PyObject* keep8(PyObject*, PyObject* o) {
    HANDLE_TH_ERRORS
    return or_refused([&]() -> PyObject* {
        const at::Tensor* x = ordinary(o);
        if (listing() || !ordinary_moment() || !simple(x) || x->dim() == 0 || dtype_code(x->scalar_type()) < 0 || x->size(-1) % 32 != 0) Py_RETURN_NONE;
        at::Tensor codes, scales;
        {
            pybind11::gil_scoped_release no_gil;
            at::NoGradGuard no_grad;
            keep_into(*x, codes, scales);
        }
        return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(codes)), THPVariable_Wrap(std::move(scales)));
    });
    END_HANDLE_TH_ERRORS
}
// mxfp8_dequant(codes, scales, dtype) -> values or None
PyObject* mxfp8_dequant(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    return or_refused([&]() -> PyObject* {
        if (n != 3) return PyErr_Format(PyExc_TypeError, "mxfp8_dequant: 3 arguments");
        const at::Tensor *q = ordinary(a[0]), *s = ordinary(a[1]);
        if (listing() || !ordinary_moment() || !simple(q) || !simple(s) || q->scalar_type() != at::kFloat8_e4m3fn || s->scalar_type() != at::kByte) Py_RETURN_NONE;
        if (!THPDtype_Check(a[2]) || dtype_code(((THPDtype*)a[2])->scalar_type) < 0) Py_RETURN_NONE;
        const at::ScalarType out = ((THPDtype*)a[2])->scalar_type;
        if (q->dim() == 0 || s->dim() != q->dim() || q->device() != s->device() || q->size(-1) != s->size(-1) * 32) Py_RETURN_NONE;
        for (int64_t i = 0; i + 1 < q->dim(); i++)
            if (q->size(i) != s->size(i)) Py_RETURN_NONE;
        at::Tensor y;
        {
            pybind11::gil_scoped_release no_gil;
            at::NoGradGuard no_grad;
            y = make(q->sizes(), out, *q);
            checked(mq_mxfp8_dequant(q->data_ptr(), (const uint8_t*)s->data_ptr(), y.data_ptr(), dtype_code(out), q->numel() / q->size(-1), q->size(-1),
                                     stream_of(*q)));
        }
        return THPVariable_Wrap(std::move(y));
    });
    END_HANDLE_TH_ERRORS
}

// ---- linear layers ---------------------------------------------------------------------------------------------------------------
struct LinearCall {
    int act;
    bool keep;
    at::Tensor codes, scales;  // a copy of x that exists already
};
at::Tensor product_scratch(int product, const void* a, int64_t lda, const void* b, int64_t ldb, bool kept8, int64_t m, int64_t n, int64_t k, const at::Tensor& like) {
    int64_t bytes = 0;
    checked(mq_linear_workspace(product, a, lda, b, ldb, kept8, m, n, k, &bytes));
    return scratch(bytes, like);
}
at::Tensor linear_forward(const at::Tensor& x, const at::Tensor& w, const at::Tensor& b, const at::Tensor& r, const LinearCall& call, bool keep_z,
                          at::Tensor& z, at::Tensor& zs) {
    const int64_t n = w.size(0), k = w.size(1), m = x.numel() / k;
    c10::SmallVector<int64_t, 4> sizes(x.sizes().begin(), x.sizes().end());
    sizes.back() = n;
    at::Tensor y = make(sizes, x.scalar_type(), x);
    if (keep_z) {
        z = make({m, n}, call.keep ? at::kFloat8_e4m3fn : x.scalar_type(), x);
        if (call.keep) zs = make({m, n / 32}, at::kByte, x);
    }
    const bool z8 = keep_z && call.keep;
    const at::Tensor ws = product_scratch(MQ_LINEAR_FORWARD, x.data_ptr(), k, w.data_ptr(), k, z8, m, n, k, x);
    checked(mq_linear_forward(x.data_ptr(), dtype_code(x.scalar_type()), k, w.data_ptr(), k, pointer(b), call.act, pointer(r), n, y.data_ptr(),
                              z8 ? nullptr : pointer(z), z8 ? pointer(z) : nullptr, (uint8_t*)pointer(zs), m, n, k, pointer(ws), stream_of(x)));
    return y;
}
struct Linear : torch::autograd::Function<Linear> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const Input& b, const Input& r,
                              LinearCall* call, bool need_x, bool need_w, bool need_b) {
        at::Tensor z, zs, kept, scales;
        at::Tensor y = linear_forward(x, w, maybe(b), maybe(r), *call, call->act != MQ_ACT_NONE && (need_x || need_w || need_b), z, zs);
        if (need_w && call->keep && call->codes.defined()) kept = call->codes, scales = call->scales;
        else if (need_w && call->keep) keep_into(x, kept, scales);
        else if (need_w) kept = x;
        ctx->save_for_backward({kept, scales, z, zs, need_x ? w : at::Tensor()});
        ctx->saved_data["act"] = (int64_t)call->act;
        ctx->saved_data["sizes"] = x.sizes().vec();
        ctx->saved_data["bias"] = b.has_value();
        ctx->saved_data["residual"] = r.has_value();
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const bool again = at::GradMode::is_enabled();
        at::NoGradGuard no_grad;
        const auto saved = ctx->get_saved_variables();
        const int act = (int)ctx->saved_data["act"].toInt();
        const std::vector<int64_t> sizes = ctx->saved_data["sizes"].toIntVector();
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
        const bool has_b = ctx->saved_data["bias"].toBool(), need_b = has_b && ctx->needs_input_grad(2);
        const bool need_r = ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(has_b ? 3 : 2);
        at::Tensor dx, dw, db;
        if (need_x || need_w || need_b) {
            const at::Tensor dy = grads[0].contiguous();
            const int64_t n = dy.size(-1), k = sizes.back(), m = dy.numel() / n;
            const int dtype = dtype_code(dy.scalar_type());
            const hipStream_t stream = stream_of(dy);
            std::vector<int64_t> groups = sizes;
            groups.back() /= 32;
            auto values = [&](const at::Tensor& t, bool codes, at::IntArrayRef shape) {        // 16-bit ones begin anywhere
                return codes ? one_run(unpacked(t, shape, at::kFloat8_e4m3fn, dy, "linear")) : unpacked(t, shape, dy.scalar_type(), dy, "linear");
            };
            const at::Tensor kept = values(saved[0], saved[1].defined(), sizes), scales = unpacked(saved[1], groups, at::kByte, dy, "linear"),
                             z = values(saved[2], saved[3].defined(), {m, n}), zs = unpacked(saved[3], {m, n / 32}, at::kByte, dy, "linear"),
                             w = values(saved[4], false, {n, k});
            at::Tensor dz = dy;
            if (need_b || act != MQ_ACT_NONE) {
                if (act != MQ_ACT_NONE) dz = make({m, n}, dy.scalar_type(), dy);
                if (need_b) db = make({n}, dy.scalar_type(), dy);
                const at::Tensor ws = scratch(need_b ? (int64_t)mq_activation_backward_parts(m, n) * n * 4 : 0, dy);
                checked(mq_activation_backward(dy.data_ptr(), dtype, n, pointer(z), (const uint8_t*)pointer(zs), act, act != MQ_ACT_NONE ? dz.data_ptr() : nullptr,
                                               pointer(db), (float*)pointer(ws), m, n, stream));
            }
            if (need_x) {
                dx = make(sizes, dy.scalar_type(), dy);
                const at::Tensor ws = product_scratch(MQ_LINEAR_INPUT_GRAD, dz.data_ptr(), n, w.data_ptr(), k, false, m, n, k, dy);
                checked(mq_linear_input_grad(dz.data_ptr(), dtype, n, w.data_ptr(), k, dx.data_ptr(), m, n, k, pointer(ws), stream));
            }
            if (need_w) {
                dw = make({n, k}, dy.scalar_type(), dy);
                const at::Tensor ws = product_scratch(MQ_LINEAR_WEIGHT_GRAD, dz.data_ptr(), n, kept.data_ptr(), k, scales.defined(), m, n, k, dy);
                checked(mq_linear_weight_grad(dz.data_ptr(), dtype, n, kept.data_ptr(), k, (const uint8_t*)pointer(scales), dw.data_ptr(), m, n, k,
                                              pointer(ws), stream));
            }
        }
        torch::autograd::variable_list out{dx, dw, db};
        if (again) once(out, grads, "linear");
        out.push_back(need_r ? grads[0] : at::Tensor());    // (handed on as it is)
        out.resize(8);
        return out;
    }
};
// linear(x, weight, bias | None, activation code, residual | None, keep in 8 bits, codes | None, scales | None) -> y or None
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t count) {
    HANDLE_TH_ERRORS
    return or_refused([&]() -> PyObject* {
        if (count != 8) return PyErr_Format(PyExc_TypeError, "linear: 8 arguments");
        const at::Tensor *x = ordinary(a[0]), *w = ordinary(a[1]), *b, *r, *codes, *scales;
        if (listing() || !ordinary_moment() || !simple(x) || !simple(w) || !optional_simple(a[2], b) || !optional_simple(a[4], r)) Py_RETURN_NONE;
        if (x->scalar_type() != at::kBFloat16 && x->scalar_type() != at::kHalf) Py_RETURN_NONE;
        int64_t act;
        LinearCall call;
        if (!integer(a[3], act) || act < 0 || act > MQ_ACT_GELU_TANH || !truth(a[5], call.keep)) Py_RETURN_NONE;
        if (!optional_simple(a[6], codes) || !optional_simple(a[7], scales) || !codes != !scales) Py_RETURN_NONE;
        call.act = (int)act;
        if (x->dim() == 0 || w->dim() != 2 || w->size(1) != x->size(-1)) Py_RETURN_NONE;
        const int64_t n = w->size(0), k = w->size(1);
        if (b && (b->dim() != 1 || b->size(0) != n)) Py_RETURN_NONE;
        if (r) {
            if (r->dim() != x->dim() || r->size(-1) != n) Py_RETURN_NONE;
            for (int64_t i = 0; i + 1 < x->dim(); i++)
                if (r->size(i) != x->size(i)) Py_RETURN_NONE;
        }
        for (const at::Tensor* t : {w, b, r})
            if (t && (t->scalar_type() != x->scalar_type() || t->device() != x->device())) Py_RETURN_NONE;
        if (call.keep && (k % 32 != 0 || (act != MQ_ACT_NONE && n % 32 != 0))) Py_RETURN_NONE;
        if (codes) {
            if (!call.keep || codes->sizes() != x->sizes() || codes->scalar_type() != at::kFloat8_e4m3fn || codes->device() != x->device()) Py_RETURN_NONE;
            if (scales->scalar_type() != at::kByte || scales->dim() != codes->dim() || scales->size(-1) * 32 != k || scales->device() != x->device() ||
                (uintptr_t)codes->data_ptr() % 16)
                Py_RETURN_NONE;
            for (int64_t i = 0; i + 1 < codes->dim(); i++)
                if (scales->size(i) != codes->size(i)) Py_RETURN_NONE;
            call.codes = *codes, call.scales = *scales;
        }
        at::Tensor y;
        {
            pybind11::gil_scoped_release no_gil;
            if (wants_graph({x, w, b, r})) {
                y = Linear::apply(*x, *w, input(b), input(r), &call, x->requires_grad(), w->requires_grad(), b && b->requires_grad());
            } else {
                at::NoGradGuard no_grad;
                at::Tensor z, zs;
                y = linear_forward(*x, *w, maybe(b), maybe(r), call, false, z, zs);
            }
        }
        return THPVariable_Wrap(std::move(y));
    });
    END_HANDLE_TH_ERRORS
}

}  // namespace
