// Rotary positions, the paged cache and the attention over it in native code, for the same reason: the single token of a decode step costs its
// kernels a few us, and as much again for every check, allocation and graph node that is written in Python.  Included by mq_host.cpp.
namespace {

// a tensor whose vectors (its last dimension) are one run of memory each; the other dimensions may have any strides
bool vectors(const at::Tensor* t) {
    return t && t->numel() > 0 && t->dim() >= 1 && (t->stride(-1) == 1 || t->size(-1) == 1) && !t->_fw_grad(0).defined() &&
           t->device().index() == c10::hip::current_device();
}
bool whole_numbers(const at::Tensor* t) { return simple(t) && (t->scalar_type() == at::kLong || t->scalar_type() == at::kInt); }
bool frequencies(const at::Tensor* t) {
    return simple(t) && t->dim() == 1 && (t->scalar_type() == at::kDouble || t->scalar_type() == at::kFloat) && !t->requires_grad();
}
bool number(PyObject* o, double& v) {
    if (!PyFloat_Check(o)) return false;
    v = PyFloat_AS_DOUBLE(o);
    return true;
}

// ---- rotary positions --------------------------------------------------------------------------------------------------------
struct RotaryCall {
    at::Tensor positions, inv_freq;
    double scale;
    bool interleaved, back;
};
mq_heads heads_of(const at::Tensor& t, void* out) {
    const int64_t n = t.dim();
    return mq_heads{t.data_ptr(), out, t.size(n - 2), n > 3 ? t.stride(n - 4) : 0, t.stride(n - 3), t.stride(n - 2)};
}
torch::autograd::variable_list rotary_run(const at::Tensor& q, const at::Tensor& k, const RotaryCall& call) {
    const at::Tensor x = q.stride(-1) == 1 || q.size(-1) == 1 ? q : q.contiguous();
    const int64_t n = x.dim(), tokens = x.size(n - 3), batch = n > 3 ? x.size(0) : 1;
    torch::autograd::variable_list out{make(x.sizes(), x.scalar_type(), x)};
    mq_heads heads[2] = {heads_of(x, out[0].data_ptr()), mq_heads{}};
    at::Tensor y;
    if (k.defined()) {
        y = k.stride(-1) == 1 || k.size(-1) == 1 ? k : k.contiguous();
        out.push_back(make(y.sizes(), y.scalar_type(), y));
        heads[1] = heads_of(y, out[1].data_ptr());
    }
    checked(mq_rotary(heads, (int)out.size(), dtype_code(x.scalar_type()), batch, tokens, x.size(-1), call.positions.data_ptr(), call.positions.scalar_type() == at::kLong,
                      call.positions.dim() == n - 2 ? tokens : 0, call.inv_freq.data_ptr(), call.inv_freq.scalar_type() == at::kDouble, call.inv_freq.numel(),
                      call.interleaved, call.scale, call.back, stream_of(x)));
    return out;
}
torch::autograd::variable_list rotary_of(const at::Tensor& q, const at::Tensor& k, RotaryCall& call);
struct Rotary : torch::autograd::Function<Rotary> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const Input& k, RotaryCall* call) {
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({call->positions, call->inv_freq});
        ctx->saved_data["scale"] = call->scale;
        ctx->saved_data["interleaved"] = call->interleaved;
        ctx->saved_data["back"] = call->back;
        ctx->saved_data["positions"] = call->positions.sizes().vec();
        ctx->saved_data["types"] = std::vector<int64_t>{(int64_t)call->positions.scalar_type(), (int64_t)call->inv_freq.scalar_type(), call->inv_freq.numel()};
        return rotary_run(q, maybe(k), *call);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        torch::autograd::variable_list wanted;
        for (size_t i = 0; i < grads.size(); i++)
            if (grads[i].defined() && ctx->needs_input_grad(i)) wanted.push_back(grads[i]);
        torch::autograd::variable_list out(3);
        if (wanted.empty()) return out;
        const auto saved = ctx->get_saved_variables();
        const std::vector<int64_t> types = ctx->saved_data["types"].toIntVector();
        RotaryCall call;
        call.positions = unpacked(saved[0], ctx->saved_data["positions"].toIntVector(), (at::ScalarType)types[0], wanted[0], "rotary");
        call.inv_freq = unpacked(saved[1], {types[2]}, (at::ScalarType)types[1], wanted[0], "rotary");
        call.scale = ctx->saved_data["scale"].toDouble();
        call.interleaved = ctx->saved_data["interleaved"].toBool();
        call.back = !ctx->saved_data["back"].toBool();
        const torch::autograd::variable_list made = rotary_of(wanted[0], wanted.size() > 1 ? wanted[1] : at::Tensor(), call);
        size_t next = 0;
        for (size_t i = 0; i < grads.size(); i++)
            if (grads[i].defined() && ctx->needs_input_grad(i)) out[i] = made[next++];
        return out;
    }
};
// a graph of its own where one is asked for: turning is linear, and its gradient is turning back
torch::autograd::variable_list rotary_of(const at::Tensor& q, const at::Tensor& k, RotaryCall& call) {
    if (wants_graph({&q, k.defined() ? &k : nullptr})) return Rotary::apply(q, k.defined() ? Input(k) : Input(), &call);
    at::NoGradGuard no_grad;
    return rotary_run(q, k, call);
}
// rotary(q, k | None, positions, inv_freq, interleaved, scale, inverse) -> q, (q, k) or None
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    return or_refused([&]() -> PyObject* {
        if (n != 7) return PyErr_Format(PyExc_TypeError, "rotary: 7 arguments");
        const at::Tensor *q = ordinary(a[0]), *k = nullptr, *positions = ordinary(a[2]), *inv_freq = ordinary(a[3]);
        RotaryCall call;
        if (listing() || !ordinary_moment() || !vectors(q) || (q->dim() != 3 && q->dim() != 4) || dtype_code(q->scalar_type()) < 0) Py_RETURN_NONE;
        if (a[1] != Py_None) {
            k = ordinary(a[1]);
            if (!vectors(k) || k->dim() != q->dim() || k->size(-1) != q->size(-1) || k->scalar_type() != q->scalar_type() || k->device() != q->device()) Py_RETURN_NONE;
            for (int64_t i = 0; i + 2 < q->dim(); i++)
                if (k->size(i) != q->size(i)) Py_RETURN_NONE;
        }
        if (!whole_numbers(positions) || !frequencies(inv_freq) || !truth(a[4], call.interleaved) || !number(a[5], call.scale) || !truth(a[6], call.back)) Py_RETURN_NONE;
        if (positions->device() != q->device() || inv_freq->device() != q->device() || 2 * inv_freq->numel() > q->size(-1)) Py_RETURN_NONE;
        const int64_t lead = q->dim() - 2;
        const bool all = positions->dim() == lead && positions->sizes() == q->sizes().slice(0, lead);
        if (!all && !(positions->dim() == 1 && positions->size(0) == q->size(lead - 1))) Py_RETURN_NONE;
        call.positions = *positions, call.inv_freq = *inv_freq;
        torch::autograd::variable_list out;
        {
            pybind11::gil_scoped_release no_gil;
            out = rotary_of(*q, maybe(k), call);
        }
        if (!k) return THPVariable_Wrap(std::move(out[0]));
        return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(out[0])), THPVariable_Wrap(std::move(out[1])));
    });
    END_HANDLE_TH_ERRORS
}

// ---- the paged cache -----------------------------------------------------------------------------------------------------------
// false: a cache that Python has to look at (it says what is wrong with it)
bool cache_of(PyObject* const* a, at::ScalarType dtype, mq_paged_cache& c) {
    const at::Tensor *keys = ordinary(a[0]), *values = ordinary(a[1]), *key_scales, *value_scales;
    if (!simple(keys) || !simple(values) || !optional_simple(a[2], key_scales) || !optional_simple(a[3], value_scales) || !key_scales != !value_scales) return false;
    const bool kept = key_scales;
    if (keys->dim() != 5 || values->dim() != 4 || keys->size(0) != values->size(0) || keys->size(1) != values->size(1) || keys->size(3) != values->size(2) ||
        keys->size(4) != (kept ? 16 : 8))
        return false;
    if ((dtype != at::kBFloat16 && dtype != at::kHalf) || keys->scalar_type() != (kept ? at::kFloat8_e4m3fn : dtype) || values->scalar_type() != keys->scalar_type()) return false;
    c = mq_paged_cache{keys->data_ptr(), values->data_ptr(), nullptr, nullptr, keys->size(0), keys->size(3), keys->size(1), keys->size(2) * keys->size(4),
                       values->size(3), dtype_code(dtype)};
    for (const at::Tensor* t : {keys, values, key_scales, value_scales})
        if (t && (t->device() != keys->device() || t->requires_grad())) return false;
    if (kept) {
        if (c.key_dim % 32 || c.value_dim % 32) return false;
        const int64_t shape[2][4] = {{c.pages, c.kv_heads, c.key_dim / 32, c.page_size}, {c.pages, c.kv_heads, c.value_dim / 32, c.page_size}};
        if (key_scales->scalar_type() != at::kByte || value_scales->scalar_type() != at::kByte || key_scales->sizes() != at::IntArrayRef(shape[0], 4) ||
            value_scales->sizes() != at::IntArrayRef(shape[1], 4))
            return false;
        c.key_scales = (uint8_t*)key_scales->data_ptr();
        c.value_scales = (uint8_t*)value_scales->data_ptr();
    }
    return true;
}
// [tokens, heads, dim] whose vectors begin at multiples of 16 bytes, without a gradient that would have to go on
bool cached_vectors(const at::Tensor* t, at::ScalarType dtype) {
    return vectors(t) && t->dim() == 3 && t->scalar_type() == dtype && (uintptr_t)t->data_ptr() % 16 == 0 && (t->size(0) == 1 || t->stride(0) % 8 == 0) &&
           (t->size(1) == 1 || t->stride(1) % 8 == 0) && !wants_graph({t});
}
// append(keys, values, key scales | None, value scales | None, k, v, slots, positions | None, inv_freq | None, interleaved, scale, q | None) ->
// the turned queries, True (there are none) or None
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    return or_refused([&]() -> PyObject* {
        if (n != 12) return PyErr_Format(PyExc_TypeError, "append: 12 arguments");
        const at::Tensor *k = ordinary(a[4]), *v = ordinary(a[5]), *slots = ordinary(a[6]), *positions = nullptr, *inv_freq = nullptr, *q = nullptr;
        mq_paged_cache c;
        if (listing() || !ordinary_moment() || !k || !cache_of(a, k->scalar_type(), c)) Py_RETURN_NONE;
        const at::ScalarType dtype = k->scalar_type();
        const at::Device device = THPVariable_Unpack(a[0]).device();
        if (!cached_vectors(k, dtype) || !cached_vectors(v, dtype) || k->size(1) != c.kv_heads || k->size(2) != c.key_dim || v->size(1) != c.kv_heads ||
            v->size(2) != c.value_dim || v->size(0) != k->size(0))
            Py_RETURN_NONE;
        const int64_t tokens = k->size(0);
        bool interleaved;
        double scale;
        if (!whole_numbers(slots) || slots->dim() != 1 || slots->size(0) != tokens || !truth(a[9], interleaved) || !number(a[10], scale)) Py_RETURN_NONE;
        if ((a[7] == Py_None) != (a[8] == Py_None)) Py_RETURN_NONE;
        if (a[7] != Py_None) {
            positions = ordinary(a[7]), inv_freq = ordinary(a[8]);
            if (!whole_numbers(positions) || positions->dim() != 1 || positions->size(0) != tokens || !frequencies(inv_freq) || 2 * inv_freq->numel() > c.key_dim ||
                inv_freq->numel() % 8)
                Py_RETURN_NONE;
        }
        if (a[11] != Py_None) {
            q = ordinary(a[11]);
            if (!inv_freq || !cached_vectors(q, dtype) || q->size(0) != tokens || q->size(2) != c.key_dim) Py_RETURN_NONE;
        }
        for (const at::Tensor* t : {k, v, slots, positions, inv_freq, q})
            if (t && t->device() != device) Py_RETURN_NONE;
        at::Tensor turned;
        for (int i = 0; i < 4; i++)                           // written in place: a graph that saved them before says so
            if (a[i] != Py_None && !THPVariable_Unpack(a[i]).is_inference()) THPVariable_Unpack(a[i]).unsafeGetTensorImpl()->bump_version();
        {
            pybind11::gil_scoped_release no_gil;
            at::NoGradGuard no_grad;
            if (q) turned = make(q->sizes(), dtype, *q);
            auto heads = [](const at::Tensor& t, void* out) { return mq_heads{t.data_ptr(), out, t.size(1), 0, t.stride(0), t.stride(1)}; };
            const mq_heads hk = heads(*k, nullptr), hv = heads(*v, nullptr), hq = q ? heads(*q, turned.data_ptr()) : mq_heads{};
            checked(mq_cache_append(&c, &hk, &hv, q ? &hq : nullptr, tokens, slots->data_ptr(), slots->scalar_type() == at::kLong,
                                    positions ? positions->data_ptr() : nullptr, positions && positions->scalar_type() == at::kLong,
                                    inv_freq ? inv_freq->data_ptr() : nullptr, inv_freq && inv_freq->scalar_type() == at::kDouble, inv_freq ? inv_freq->numel() : 0,
                                    interleaved, scale, stream_of(*k)));
        }
        if (!q) Py_RETURN_TRUE;
        return THPVariable_Wrap(std::move(turned));
    });
    END_HANDLE_TH_ERRORS
}
// attend(q, keys, values, key scales | None, value scales | None, pages, lengths, scale | None, window | None, sinks | None) -> out or None
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    return or_refused([&]() -> PyObject* {
        if (n != 10) return PyErr_Format(PyExc_TypeError, "attend: 10 arguments");
        const at::Tensor *q = ordinary(a[0]), *pages = ordinary(a[5]), *lengths = ordinary(a[6]), *sinks;
        mq_paged_cache c;
        if (listing() || !ordinary_moment() || !q || !cache_of(a + 1, q->scalar_type(), c) || !cached_vectors(q, q->scalar_type())) Py_RETURN_NONE;
        const at::Device device = THPVariable_Unpack(a[1]).device();
        if (q->size(2) != c.key_dim || q->size(1) % c.kv_heads) Py_RETURN_NONE;
        const int64_t batch = q->size(0), heads = q->size(1);
        if (!vectors(pages) || pages->scalar_type() != at::kInt || pages->dim() != 2 || pages->size(0) != batch) Py_RETURN_NONE;
        if (!simple(lengths) || lengths->scalar_type() != at::kInt || lengths->dim() != 1 || lengths->size(0) != batch) Py_RETURN_NONE;
        if (!optional_simple(a[9], sinks)) Py_RETURN_NONE;
        if (sinks && (sinks->scalar_type() != at::kFloat || sinks->dim() != 1 || sinks->size(0) != heads || wants_graph({sinks}))) Py_RETURN_NONE;
        for (const at::Tensor* t : {q, pages, lengths, sinks})
            if (t && t->device() != device) Py_RETURN_NONE;
        double scale = 1.0 / std::sqrt((double)c.key_dim);
        int64_t window = 0;
        if (a[7] != Py_None && !number(a[7], scale)) Py_RETURN_NONE;
        if (a[8] != Py_None && (!integer(a[8], window) || window < 1)) Py_RETURN_NONE;
        at::Tensor out;
        {
            pybind11::gil_scoped_release no_gil;
            at::NoGradGuard no_grad;
            const int64_t sizes[3] = {batch, heads, c.value_dim}, width = pages->size(1);
            out = make(at::IntArrayRef(sizes, 3), q->scalar_type(), *q);
            int64_t bytes = 0;
            checked(mq_paged_attention_workspace(&c, batch, heads, width, window, &bytes));
            const at::Tensor ws = scratch(bytes, *q);
            checked(mq_paged_attention(&c, q->data_ptr(), q->stride(0), q->stride(1), (const int32_t*)pages->data_ptr(), pages->stride(0), width,
                                       (const int32_t*)lengths->data_ptr(), sinks ? (const float*)sinks->data_ptr() : nullptr, scale, window, out.data_ptr(), batch,
                                       heads, pointer(ws), stream_of(*q)));
        }
        return THPVariable_Wrap(std::move(out));
    });
    END_HANDLE_TH_ERRORS
}

}  // namespace
